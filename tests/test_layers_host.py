"""The gated layer, weight gradients from an input in full and AdamW without a GPU: what they refuse, the descriptors as a C compiler lays
them out, and the oracle's own parts."""

import ctypes as C
import math
import shutil

import pytest
import torch

from oracle import layers as ref
from tests import test_gpu_gated
from tests.test_cabi_from_c import build_and_run
from tileccl_amd import _lib, ops, ops_adamw, ops_gated


def test_entry_points_are_public():
    for name in ("gated_linear", "gated_linear_backward", "GatedLinearResult", "GatedLinearGradients", "adamw_step", "adamw_moments", "AdamWState"):
        assert name in ops.__all__ and hasattr(ops, name)


def test_operands_must_be_on_the_gpu():
    x, w = torch.zeros(4, 8).half(), torch.zeros(8, 16).half()
    with pytest.raises(ValueError, match="weight must reside on the GPU"):
        ops.gated_linear(x, w)
    with pytest.raises(ValueError, match="weight must be a 2-D tensor, got 1"):
        ops.gated_linear(x, w[0])
    with pytest.raises(ValueError, match="activation must be one of 'silu', 'gelu', 'gelu_tanh', 'relu', got 'swish'"):
        ops.gated_linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="weight must reside on the GPU"):
        ops.gated_linear_backward(x, None, x, w)
    with pytest.raises(ValueError, match="activation must be"):
        ops.gated_linear_backward(x, None, x, w, activation="tanh")
    with pytest.raises(ValueError, match="grad must reside on the GPU"):
        ops.weight_gradient(x, x)
    p = [torch.zeros(4)]
    state = ops.AdamWState(torch.zeros(128), torch.zeros(128), None, None, None, (4,))
    with pytest.raises(ValueError, match=r"params\[0\] must reside on cuda:0"):
        ops.adamw_step(p, p, state, step=1)
    with pytest.raises(ValueError, match="1 params, 0 grads, a state of 1"):
        ops.adamw_step(p, [], state, step=1)
    with pytest.raises(ValueError, match="expected an AdamWState, got tuple"):
        ops.adamw_step(p, p, tuple(state), step=1)
    with pytest.raises(ValueError, match="expected an AdamWState"):
        ops.adamw_moments(p)
    assert ops.adamw_moments(state)[0] is state.first
    with pytest.raises(ValueError, match="8 or 32 bits, got 16"):
        ops.AdamWState.zeros(p, bits=16)
    with pytest.raises(ValueError, match="for params in 16 bits"):
        ops.AdamWState.zeros(p, master=True)


def test_state_layout():
    assert ops.AdamWState.offsets([]) == [0] and ops.AdamWState.offsets([1, 128, 0, 129]) == [0, 128, 256, 256, 512]
    params = [torch.arange(5.0).half(), torch.ones(3, 50).half()]
    state = ops.AdamWState.zeros(params, bits=8, master=True)
    assert state.first.shape == state.second.shape == (384,) and state.first.dtype == torch.uint8 and state.first_scales.shape == (3,)
    assert torch.equal(state.master[:5], torch.arange(5.0)) and bool((state.master[128:278] == 1).all()) and not bool(state.master[5:128].any())
    assert state.nbytes == 2 * 384 + 2 * 3 + 4 * 384


def refused(rc, text, code=None):
    assert rc == (_lib.ERR_INVALID if code is None else code)
    assert text in _lib.last_error()


def test_bad_gated_descriptors(lib):
    for entry in (lib.tccl_gated, lib.tccl_gated_grad, lib.tccl_gated_input_grad, lib.tccl_weight_gradient_full, lib.tccl_adamw, lib.tccl_adamw_moments):
        refused(entry(None, None), "the descriptor is NULL")

    def forward(**kw):
        d = _lib.GatedDesc(x=0x1000, weight=0x2000, out=0x3000, ld_x=64, ld_weight=256, up=128, ld_out=128, rows=4, inputs=64, outputs=128, dtype=_lib.BF16)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.tccl_gated(C.byref(d), None)

    def backward(**kw):
        d = _lib.GatedGradDesc(grad=0x1000, kept=0x5000, inner=0x3000, ld_grad=128, ld_kept=256, ld_inner=256, rows=4, inputs=64, outputs=128, dtype=_lib.F16)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.tccl_gated_grad(C.byref(d), None)

    un = _lib.ERR_UNSUPPORTED
    for call in (forward, backward):
        refused(call(rows=-1), "rows must not be negative")
        refused(call(inputs=0), "must be positive")
        refused(call(rows=_lib.TRAINING_MAX_ROWS + 1), "at most", un)
        refused(call(outputs=_lib.GATED_MAX_COLS + 1), f"at most {_lib.GATED_MAX_COLS}", un)
        refused(call(dtype=_lib.F32), "F16 or BF16", un)
        refused(call(activation=4), "activation=4")
        refused(call(activation=-1), "activation=-1")
        assert call(rows=0) == 0
    refused(forward(x=None), "x is NULL")
    refused(forward(out=None), "out is NULL")
    refused(forward(out=0x3001), "not aligned to its type")
    refused(forward(ld_out=100), "out has a pitch of 100 elements for 128 columns")
    refused(forward(kept=0x9000, ld_kept=255), "kept has a pitch of 255 elements for 256 columns")
    refused(forward(x=0x1001), "x is not aligned to its type")
    refused(forward(ld_x=8), "x has a pitch of 8")
    refused(forward(up=64), "lies 64 elements behind")
    refused(forward(up=136), "lies 136 elements behind")  # past the row's pitch
    refused(forward(kmajor=1, ld_weight=64, up=127 * 64), "lies 8128 elements behind")
    refused(forward(kmajor=1, ld_weight=56, up=128 * 64), "pitch of 56")
    for entry, desc in ((lib.tccl_gated_workspace, _lib.GatedDesc), (lib.tccl_gated_grad_workspace, _lib.GatedGradDesc),
                        (lib.tccl_weight_gradient_full_workspace, _lib.WeightGradientFullDesc)):
        assert entry(None) == -1 and "the descriptor is NULL" in _lib.last_error()
        assert entry(C.byref(desc(rows=4, outputs=8))) == -1 and "must be positive" in _lib.last_error()
    assert lib.tccl_gated_workspace(C.byref(_lib.GatedDesc(inputs=8, outputs=8, dtype=_lib.F16))) == 0  # no rows
    assert lib.tccl_gated_grad_workspace(C.byref(_lib.GatedGradDesc(kept=0x1000, rows=8, inputs=8, outputs=8, dtype=_lib.F16))) == 0
    def input_grad(**kw):
        d = _lib.GatedInputGradDesc(inner=0x1000, weight=0x2000, dx=0x3000, ld_inner=256, ld_weight=256, ld_dx=64, rows=4, inputs=64, outputs=128, dtype=_lib.F16)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.tccl_gated_input_grad(C.byref(d), None)

    assert input_grad(rows=0) == 0 and lib.tccl_gated_input_grad_workspace(None) == -1
    refused(input_grad(rows=-1), "rows must not be negative")
    refused(input_grad(dtype=_lib.F32), "F16 or BF16", un)
    refused(input_grad(inner=None), "inner is NULL")
    refused(input_grad(ld_inner=255), "inner has a pitch of 255 elements for 256 columns")
    refused(input_grad(ld_weight=200), "weight has a pitch of 200 elements for 256 columns")
    refused(input_grad(kmajor=1, ld_weight=60), "weight has a pitch of 60 elements for 64 columns")
    refused(input_grad(dx=0x3001), "dx is not aligned to its type")
    refused(input_grad(ld_dx=63), "dx has a pitch of 63 elements for 64 columns")
    refused(backward(grad=None), "grad is NULL")
    refused(backward(inner=None), "inner is NULL")
    refused(backward(ld_kept=128), "kept has a pitch of 128")
    refused(backward(kept=None), "x is NULL")


def test_bad_weight_gradient_descriptors(lib):
    def call(**kw):
        d = _lib.WeightGradientFullDesc(x=0x1000, grad=0x3000, out=0x4000, ld_x=128, ld_grad=64, ld_out=64, rows=8, cols=128, outputs=64, dtype=_lib.BF16, out_dtype=_lib.F32)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.tccl_weight_gradient_full(C.byref(d), None)

    un = _lib.ERR_UNSUPPORTED
    refused(call(outputs=0), "must be positive")
    refused(call(dtype=_lib.F32), "F16 or BF16", un)
    refused(call(out_dtype=_lib.F16), "grad's type or F32", un)
    refused(call(out=None), "out is NULL")
    refused(call(x=None), "x is NULL")
    refused(call(ld_x=(1 << 24) + 8), f"at most {1 << 24}", un)
    refused(call(ld_grad=56), "grad has a pitch of 56")
    refused(call(grad=0x3001), "grad is not aligned to its type")
    refused(call(ld_out=63), "pitch below its 64 columns")
    refused(call(transposed=1), "pitch below its 128 columns")
    refused(call(out=0x4002), "not aligned to its type")


def test_bad_adamw_descriptors(lib):
    def call(sizes=(64,), params=(0x1000,), grads=(0x2000,), **kw):
        n = len(sizes)
        d = _lib.AdamwDesc(params=C.cast((C.c_void_p * n)(*params), C.c_void_p), grads=C.cast((C.c_void_p * n)(*grads), C.c_void_p),
                           sizes=C.cast((C.c_int64 * n)(*sizes), C.c_void_p), first=0x10000, second=0x20000, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0,
                           tensors=n, dtype=_lib.F32, grad_dtype=_lib.F32, bits=32, step=1)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.tccl_adamw(C.byref(d), None)

    un = _lib.ERR_UNSUPPORTED
    refused(call(tensors=-1), "-1 tensors")
    refused(call(params=(None,)), "tensor 0 or its gradient is NULL")
    refused(call(sizes=(-1,)), "tensor 0 has -1 elements")
    refused(call(sizes=((1 << 38) + 1,)), "more than 2^38 elements", un)
    refused(call(params=(0x1002,)), "not aligned to its type")
    refused(call(dtype=_lib.F8E4M3), "F32, F16 or BF16", un)
    refused(call(grad_dtype=_lib.BF16), "of that type or F32", un)
    refused(call(master=0x30000), "master copy of F32")
    refused(call(bits=16), "must be 8 or 32")
    refused(call(bits=8), "scales of those in 8 bits")
    refused(call(first=None), "must be non-NULL")
    refused(call(second=0x20008), "on 16 bytes", un)
    refused(call(beta1=1.0), "betas must lie in [0, 1)")
    refused(call(beta2=math.nan), "betas must lie in [0, 1)")
    refused(call(eps=-1.0), "eps must not be negative")
    refused(call(step=0), "counted from 1")
    refused(call(step_at=0x1001), "not aligned")
    assert call(sizes=(0,), params=(None,), grads=(None,)) == 0  # nothing to do

    def moments(**kw):
        d = _lib.AdamwMomentsDesc(first=0x1000, second=0x2000, first_scales=0x3000, second_scales=0x4000, to_first=0x5000, to_second=0x6000, blocks=1)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.tccl_adamw_moments(C.byref(d), None)

    refused(moments(blocks=-1), "-1 blocks")
    refused(moments(first_scales=None), "must be non-NULL")
    refused(moments(to_second=0x6004), "on 16 bytes", un)
    assert moments(blocks=0) == 0


def gated_cut(lib, rows, inputs, outputs, kmajor=0, cus=256):
    got = [C.c_int32() for _ in range(4)]
    assert lib.tccl_gated_cut(rows, inputs, outputs, kmajor, cus, *map(C.byref, got)) == 0
    return tuple(g.value for g in got)


def test_how_calls_are_cut(lib):
    """What the GPU tests' shapes are for, on 256 compute units: (tile, rows, outputs of a part, splits)."""
    assert gated_cut(lib, 1, 4096, 8192, 1) == (0, 16, 32, 1) and gated_cut(lib, 13, 4096, 4096) == (0, 16, 64, 4)
    assert gated_cut(lib, 20, 4096, 4096) == (0, 32, 64, 4) and gated_cut(lib, 40, 4096, 1024) == (0, 64, 32, 8)
    assert gated_cut(lib, 40, 512, 512) == (0, 64, 16, 1) and gated_cut(lib, 64, 584, 8192, 1) == (0, 64, 32, 1)
    assert gated_cut(lib, 8192, 4096, 8192, 1) == (256, 256, 128, 1) and gated_cut(lib, 1003, 1001, 1035)[0] == 128
    assert gated_cut(lib, 112, 7168, 104, 1) == (0, 64, 16, 8) and gated_cut(lib, 1000, 4096, 512)[::3] == (128, 4)
    for rows, inputs, outputs, _, layout, _ in test_gpu_gated.LARGE:
        assert gated_cut(lib, rows, inputs, outputs, layout == "nk") == (256, 256, 128, 1)
    kinds = {(layout, *gated_cut(lib, rows, inputs, outputs, layout == "nk")[:3]) for rows, inputs, outputs, _, layout, _ in test_gpu_gated.SPLIT}
    assert all(("kn", *k) in kinds for k in ((0, 16, 64), (0, 32, 64), (0, 64, 16), (0, 64, 32), (128, 128, 64)))
    assert all(("nk", *k) in kinds for k in ((0, 16, 16), (0, 16, 32), (0, 32, 16), (0, 32, 32), (0, 64, 16), (0, 64, 32), (128, 128, 64)))
    splits = C.c_int32()
    for rows, inputs, outputs, _, _ in test_gpu_gated.LONG:
        assert lib.tccl_gated_input_grad_cut(rows, inputs, outputs, 256, C.byref(splits)) == 0 and splits.value >= 2
    for shape in ((64, 128, 2048), (2048, 2048, 4096), (300, 256, 600), (1, 4096, 4096)):
        assert lib.tccl_gated_input_grad_cut(*shape, 256, C.byref(splits)) == 0 and splits.value == 0
    refused(lib.tccl_gated_input_grad_cut(8, 8, 8, 256, None), "NULL result")
    got = [C.c_int32() for _ in range(3)]
    for shape, want in (((128, 4200, 2056), 256), ((1000, 1000, 3088), 128)):
        assert lib.tccl_weight_gradient_full_cut(*shape, 256, *map(C.byref, got)) == 0 and got[0].value == want
    assert lib.tccl_weight_gradient_full_cut(16384, 1024, 512, 256, *map(C.byref, got)) == 0 and got[1].value == 8
    refused(lib.tccl_gated_cut(8, 8, 8, 0, 0, *[C.byref(C.c_int32()) for _ in range(4)]), "0 compute units")
    refused(lib.tccl_weight_gradient_full_cut(8, 8, 8, 256, None, None, None), "NULL result")


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_descriptors_as_gcc_sees_them(tmp_path):
    structs = {"tccl_weight_gradient_full_desc": _lib.WeightGradientFullDesc, "tccl_gated_desc": _lib.GatedDesc, "tccl_gated_grad_desc": _lib.GatedGradDesc,
               "tccl_gated_input_grad_desc": _lib.GatedInputGradDesc,
               "tccl_adamw_desc": _lib.AdamwDesc, "tccl_adamw_moments_desc": _lib.AdamwMomentsDesc}
    body = ""
    for cname, py in structs.items():
        body += f'  printf("{cname} %zu\\n", sizeof({cname}));\n'
        for field, _ in py._fields_:
            body += f'  printf("{cname}.{field} %zu\\n", offsetof({cname}, {field}));\n'
    body += '  printf("cols %d\\nblock %d\\nacts %d%d%d%d\\n", TCCL_GATED_MAX_COLS, TCCL_MOMENT_BLOCK, TCCL_SILU, TCCL_GELU, TCCL_GELU_TANH, TCCL_RELU);\n'
    got = dict(line.split() for line in build_and_run(tmp_path, body).splitlines())
    for cname, py in structs.items():
        assert int(got[cname]) == C.sizeof(py)
        for field, _ in py._fields_:
            assert int(got[f"{cname}.{field}"]) == getattr(py, field).offset
    assert int(got["cols"]) == _lib.GATED_MAX_COLS and int(got["block"]) == _lib.MOMENT_BLOCK == ref.BLOCK
    assert got["acts"] == "".join(str(c) for c in ops_gated.ACTIVATIONS.values()) == "0123"


def test_oracle_codes():
    """Every finite code is its own neighbour, what lies between two codes has these, and the tables are what the hardware's type says."""
    native = torch.arange(256, dtype=torch.int64).to(torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(native.nan_to_num(9e9), ref.FIRST.nan_to_num(9e9))
    for table in (ref.FIRST, ref.SECOND):
        grid = torch.unique(table[torch.isfinite(table)].abs())
        low, high = ref.neighbours(grid, table)
        assert torch.equal(low, grid) and torch.equal(high, grid)
        middle = (grid[1:] + grid[:-1]) / 2
        low, high = ref.neighbours(middle, table)
        assert torch.equal(low, grid[:-1]) and torch.equal(high, grid[1:])
    assert ref.SECOND[1] == 2.0**-30 and ref.SECOND[249] == 2.0 and math.isnan(ref.SECOND[255])


def test_random_numbers_are_even_and_apart():
    """Of 4096 places and two steps: means within 5 standard deviations, no correlation between the moments' numbers, neighbours or steps."""
    n = 4096
    a, b = ref.uniforms(n, 7), ref.uniforms(n, 8)
    series = [a[0], a[1], b[0], b[1], a[0].roll(1), a[1].roll(1), a[0].roll(128)]
    for s in series:
        assert abs(float(s.mean()) - 0.5) < 5 * math.sqrt(1 / 12 / n)
    for i, s in enumerate(series):
        for t in series[i + 1:]:
            assert abs(float(((s - 0.5) * (t - 0.5)).mean()) * 12) < 5 / math.sqrt(n)


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_oracle_derivatives(name):
    g = torch.linspace(-8, 8, 401, dtype=torch.float64)
    step = 1e-6
    slope = (ref.activation(g + step, name)[0] - ref.activation(g - step, name)[0]) / (2 * step)
    assert float((slope - ref.activation(g, name)[1]).abs().max()) < 1e-8


def test_weights_that_are_no_layout():
    assert ops_gated._by_rows(torch.empty(4, 8)) and not ops_gated._by_rows(torch.empty(8, 4).t())
    assert ops_gated._by_rows(torch.empty(1, 8)) and ops_gated._by_rows(torch.empty(4, 20)[:, :8])
    lo, hi = ops_gated._weight_span(torch.empty(8, 6).t())
    assert hi - lo == 48 * 4


def test_adamw_explains_shared_memory(monkeypatch):
    """Two tensors of one place, a gradient inside a moment: found by the words, whatever the device."""
    monkeypatch.setattr(ops_adamw, "_tensor", lambda *a: None)
    p = torch.zeros(64)
    state = ops.AdamWState(torch.zeros(256), torch.zeros(256), None, None, None, (64, 64))
    with pytest.raises(ValueError, match=r"params\[0\] and params\[1\] share memory"):
        ops_adamw._refuse_adamw_step((p, p), (torch.ones(64), torch.ones(64)), state, 1, 1.0, 1.0)
    with pytest.raises(ValueError, match=r"first and grads\[0\] share memory"):
        ops_adamw._refuse_adamw_step((p, torch.zeros(64)), (state.first[:64], torch.ones(64)), state, 1, 1.0, 1.0)
