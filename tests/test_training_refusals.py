"""What the training operators' entry points refuse on the host, before any launch."""

import ctypes as C
import random

import pytest
import torch

from tileccl_amd import _lib, ops_training


def refused(rc, text, code=None):
    assert rc == (_lib.ERR_INVALID if code is None else code)
    assert text in _lib.last_error()


def test_two_outputs_in_one_place(lib):
    d = _lib.NormDesc(x=0x1000, residual=0x2000, summed=0x3000, out=0x3000, mean=0x4000, rstd=0x5000, ld_x=64, ld_residual=64, ld_summed=64, ld_out=64,
                      rows=4, cols=64, dtype=_lib.BF16, affine_dtype=_lib.BF16)
    refused(lib.tccl_layer_norm(C.byref(d), None), "out and summed are the same memory")


def test_results_and_operands_that_share_bytes():
    """Against the sets of bytes, over random places of a matrix and a vector in one allocation."""
    rng = random.Random(1)
    memory = torch.zeros(400, dtype=torch.int16)
    met = 0
    for _ in range(3000):
        rows, cols, n = rng.randint(1, 6), rng.randint(1, 9), rng.randint(1, 30)
        pitch = cols + rng.choice((0, 1, 7, 30))
        first = rng.randint(0, 400 - (rows - 1) * pitch - cols)
        out, start = memory[first:].as_strided((rows, cols), (pitch, 1)), rng.randint(0, 400 - n)
        written = {first + r * pitch + c for r in range(rows) for c in range(cols)}
        try:
            ops_training._clear(out, "op", weight=memory[start: start + n])
            assert not written & set(range(start, start + n))
        except ValueError as e:
            assert "op: out overlaps weight" in str(e) and written & set(range(start, start + n))
            met += 1
    assert 300 < met < 2700


LIMIT = (1 << 31) - (1 << 16) - 1


@pytest.mark.parametrize("rows", [LIMIT + 1, (1 << 31) - 8, (1 << 31) - 1])
def test_rows_whose_indexes_would_pass_32_bits(lib, rows):
    """A grid's last turns count up to (workgroups of a turn) x (groups of rows of one) past the last row."""
    assert LIMIT == _lib.TRAINING_MAX_ROWS
    text, code = f"rows={rows}, at most {LIMIT}", _lib.ERR_UNSUPPORTED
    h = _lib.HeldDesc(0x1000, 0x2000, 0x3000, 1, rows, 1, _lib.F16)
    for entry in (lib.tccl_hold, lib.tccl_restore):
        refused(entry(C.byref(h), None), text, code)
    n = _lib.NormDesc(x=0x1000, out=0x2000, mean=0x3000, rstd=0x4000, ld_x=1, ld_out=1, rows=rows, cols=1, dtype=_lib.F32, affine_dtype=_lib.F32)
    refused(lib.tccl_layer_norm(C.byref(n), None), text, code)
    g = _lib.NormGradDesc(grad=0x1000, x=0x5000, dx=0x2000, mean=0x3000, rstd=0x4000, ld_grad=1, ld_x=1, ld_dx=1, rows=rows, cols=1, dtype=_lib.F32, affine_dtype=_lib.F32)
    refused(lib.tccl_layer_norm_grad(C.byref(g), None), text, code)
    assert lib.tccl_layer_norm_grad_workspace(rows, 1, _lib.F32, 0) == -1 and text in _lib.last_error()
    w = _lib.WeightGradientDesc(values=0x1000, scales=0x2000, grad=0x3000, out=0x4000, ld_grad=8, ld_out=8, rows=rows, cols=1, outputs=8, dtype=_lib.BF16, out_dtype=_lib.F32)
    refused(lib.tccl_weight_gradient(C.byref(w), None), text, code)
    assert lib.tccl_weight_gradient_workspace(rows, 1, 8) == -1 and text in _lib.last_error()


def test_weight_gradient_workspace_of_sizes_that_the_operator_refuses(lib):
    for cols, outputs in (((1 << 24) + 1, 8), (8, (1 << 31) - 1)):
        assert lib.tccl_weight_gradient_workspace(64, cols, outputs) == -1 and f"at most {1 << 24}" in _lib.last_error()


def test_the_limit_is_the_headers(tmp_path):
    from tests.test_cabi_from_c import build_and_run

    assert int(build_and_run(tmp_path, '  printf("%d\\n", TCCL_TRAINING_MAX_ROWS);\n')) == LIMIT


def test_python_refuses_such_checkpoints():
    for rows, columns in ((LIMIT + 1, 1), (-1, 8), (8, 0)):
        with pytest.raises(ValueError, match="a checkpoint of"):
            ops_training._held(ops_training.ActivationCheckpoint(torch.zeros(0), torch.zeros(0), rows, columns, torch.float16), "op")
