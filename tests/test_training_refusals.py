"""What the training operators' entry points refuse on the host, before any launch."""

import ctypes as C
import random

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
