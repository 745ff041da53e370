"""The training operators without a GPU: what they refuse, and the descriptors as a C compiler lays them out."""

import ctypes as C
import shutil

import pytest
import torch

from tileccl_amd import _lib, ops
from tests.test_cabi_from_c import build_and_run


def test_entry_points_are_public():
    for name in ("layer_norm", "layer_norm_backward", "checkpoint_activation", "restore_activation", "weight_gradient", "ActivationCheckpoint"):
        assert name in ops.__all__ and hasattr(ops, name)


def test_operands_must_be_matrices_on_the_gpu():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="x must be a 2-D tensor"):
        ops.layer_norm(torch.zeros(8))
    with pytest.raises(ValueError, match="x must reside on the GPU"):
        ops.layer_norm(x)
    with pytest.raises(ValueError, match="grad must reside on the GPU"):
        ops.layer_norm_backward(x, x, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="x must reside on the GPU"):
        ops.checkpoint_activation(x.half())
    with pytest.raises(ValueError, match="expected an ActivationCheckpoint, got Tensor"):
        ops.restore_activation(x)
    held = ops.ActivationCheckpoint.empty(4, 8, torch.float16, "cpu")
    with pytest.raises(ValueError, match="must reside on the GPU"):
        ops.restore_activation(held)
    with pytest.raises(ValueError, match="grad must reside on the GPU"):
        ops.weight_gradient(held, x.half())
    with pytest.raises(ValueError, match="layout must be"):
        ops.weight_gradient(held, x.half(), layout="km")


@pytest.mark.parametrize("rows, cols, values, scales", [(1, 1, (1, 128, 8), (1, 16)), (8, 128, (1, 128, 8), (1, 16)), (129, 129, (17, 256, 8), (2, 32)), (0, 5, (0, 128, 8), (1, 0))])
def test_checkpoint_shapes(rows, cols, values, scales):
    held = ops.ActivationCheckpoint.empty(rows, cols, torch.bfloat16, "cpu")
    assert tuple(held.values.shape) == values and tuple(held.scales.shape) == scales
    assert held.nbytes == held.values.numel() + held.scales.numel()


def refused(rc, text, code=None):
    assert rc == (_lib.ERR_INVALID if code is None else code)
    assert text in _lib.last_error()


def test_bad_descriptors_are_refused_on_the_host(lib):
    for entry in (lib.tccl_hold, lib.tccl_restore, lib.tccl_layer_norm, lib.tccl_layer_norm_grad, lib.tccl_weight_gradient):
        refused(entry(None, None), "the descriptor is NULL")
    h = _lib.HeldDesc(0x1000, 0x2000, 0x3000, 128, 8, 0, _lib.F16)
    refused(lib.tccl_hold(C.byref(h), None), "cols must be positive")
    h.cols, h.rows = 128, -1
    refused(lib.tccl_hold(C.byref(h), None), "rows must not be negative")
    h.rows, h.ld = 8, 64
    refused(lib.tccl_hold(C.byref(h), None), "pitch of 64 elements for 128 columns")
    h.ld, h.dtype = 128, _lib.F32
    refused(lib.tccl_hold(C.byref(h), None), "16-bit types", _lib.ERR_UNSUPPORTED)
    h.dtype, h.values = _lib.F16, 0x2008
    refused(lib.tccl_restore(C.byref(h), None), "on 16 bytes", _lib.ERR_UNSUPPORTED)
    h.values, h.x = 0x2000, 0x1001
    refused(lib.tccl_restore(C.byref(h), None), "not aligned to its type")

    n = _lib.NormDesc(x=0x1000, out=0x2000, mean=0x3000, rstd=0x4000, ld_x=64, ld_out=64, rows=4, cols=64, dtype=_lib.BF16, affine_dtype=_lib.BF16)
    n.cols = _lib.NORM_MAX_COLS + 1
    refused(lib.tccl_layer_norm(C.byref(n), None), "at most 32768", _lib.ERR_UNSUPPORTED)
    n.cols, n.dtype = 64, _lib.F8E4M3
    refused(lib.tccl_layer_norm(C.byref(n), None), "is not F16, BF16 or F32", _lib.ERR_UNSUPPORTED)
    n.dtype, n.residual = _lib.BF16, 0x5000
    refused(lib.tccl_layer_norm(C.byref(n), None), "residual and summed go together")
    n.residual, n.affine_dtype = None, _lib.F16
    refused(lib.tccl_layer_norm(C.byref(n), None), "x's type or F32", _lib.ERR_UNSUPPORTED)
    n.affine_dtype, n.values = _lib.F32, 0x6000
    refused(lib.tccl_layer_norm(C.byref(n), None), "values and scales go together")
    n.values, n.mean = None, None
    refused(lib.tccl_layer_norm(C.byref(n), None), "mean and rstd are NULL")
    n.rows = 0  # nothing to do, nothing to point at
    assert lib.tccl_layer_norm(C.byref(n), None) == 0

    g = _lib.NormGradDesc(grad=0x1000, dx=0x2000, mean=0x3000, rstd=0x4000, ld_grad=64, ld_dx=64, rows=4, cols=64, dtype=_lib.F16, affine_dtype=_lib.F16)
    refused(lib.tccl_layer_norm_grad(C.byref(g), None), "given as x or as values")
    g.x = g.values = 0x5000
    refused(lib.tccl_layer_norm_grad(C.byref(g), None), "given as x or as values")
    g.values, g.ld_x = None, 8
    refused(lib.tccl_layer_norm_grad(C.byref(g), None), "x has a pitch of 8")

    w = _lib.WeightGradientDesc(values=0x1000, scales=0x2000, grad=0x3000, out=0x4000, ld_grad=64, ld_out=64, rows=8, cols=128, outputs=0, dtype=_lib.BF16, out_dtype=_lib.F32)
    refused(lib.tccl_weight_gradient(C.byref(w), None), "must be positive")
    w.outputs, w.dtype = 64, _lib.F32
    refused(lib.tccl_weight_gradient(C.byref(w), None), "grad is F16 or BF16", _lib.ERR_UNSUPPORTED)
    w.dtype, w.out_dtype = _lib.BF16, _lib.F16
    refused(lib.tccl_weight_gradient(C.byref(w), None), "grad's type or F32", _lib.ERR_UNSUPPORTED)
    w.out_dtype, w.ld_grad = _lib.F32, 68
    refused(lib.tccl_weight_gradient(C.byref(w), None), "whole 16-byte vectors", _lib.ERR_UNSUPPORTED)
    w.ld_grad, w.ld_out = 64, 63
    refused(lib.tccl_weight_gradient(C.byref(w), None), "pitch below its 64 columns")
    w.ld_out, w.grad = 64, 0x3008
    refused(lib.tccl_weight_gradient(C.byref(w), None), "on 16 bytes", _lib.ERR_UNSUPPORTED)
    assert lib.tccl_weight_gradient_workspace(8, 0, 8) < 0 and lib.tccl_layer_norm_grad_workspace(8, 0, _lib.F16, 0) < 0


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_descriptors_as_gcc_sees_them(tmp_path):
    structs = {"tccl_held_desc": _lib.HeldDesc, "tccl_norm_desc": _lib.NormDesc, "tccl_norm_grad_desc": _lib.NormGradDesc, "tccl_weight_gradient_desc": _lib.WeightGradientDesc}
    body = ""
    for cname, py in structs.items():
        body += f'  printf("{cname} %zu\\n", sizeof({cname}));\n'
        for field, _ in py._fields_:
            body += f'  printf("{cname}.{field} %zu\\n", offsetof({cname}, {field}));\n'
    body += '  printf("rows %d\\ncols %d\\nmost %d\\n", TCCL_HELD_ROWS, TCCL_HELD_COLS, TCCL_NORM_MAX_COLS);\n'
    got = dict(line.split() for line in build_and_run(tmp_path, body).splitlines())
    for cname, py in structs.items():
        assert int(got[cname]) == C.sizeof(py)
        for field, _ in py._fields_:
            assert int(got[f"{cname}.{field}"]) == getattr(py, field).offset
    assert (int(got["rows"]), int(got["cols"]), int(got["most"])) == (_lib.HELD_ROWS, _lib.HELD_COLS, _lib.NORM_MAX_COLS)
