"""The gated linear layer and its gradients on the GPU against their definitions in 64 bits (bounds: layer_bounds.py)."""

import ctypes

import pytest
import torch

from oracle import layers as ref
from tests.layer_bounds import BF16, F16, F32, SUM, gated_bounds, half, inner_bounds, placed, rand, rounded, within
from tileccl_amd import _lib, ops

pytestmark = pytest.mark.gpu

ACTS = ("silu", "gelu", "gelu_tanh", "relu")


def weight_of(inputs, outputs, dtype, layout, seed, pad=0, offset=0):
    w = rand((inputs, 2 * outputs), seed, dtype, 1.2 * inputs**-0.5)
    if layout == "kn":
        return w, placed(w, 2 * outputs + pad, offset)
    return w, placed(w.t().contiguous(), inputs + pad, offset).t()


def check_forward(r, x, w, act, keep):
    k, dtype = x.shape[1], x.dtype
    g, u, s = ref.projections(x, w)
    want, bound = gated_bounds(g, u, s, k, dtype, act)
    within(r.out, want, bound, "out")
    if keep:
        z = torch.cat([g, u], dim=1)
        within(r.kept, z, rounded(z, k * SUM * s, dtype), "kept")
    else:
        assert r.kept is None


FORWARD = [
    # rows, inputs, outputs, type, layout, activation: one of everything, around vectors, tiles and K steps
    (1, 8, 8, BF16, "kn", "silu"), (1, 8, 1, F16, "nk", "silu"), (1, 1, 1, BF16, "kn", "relu"), (2, 64, 64, F16, "nk", "gelu"),
    (3, 72, 8, BF16, "nk", "gelu_tanh"), (13, 512, 96, F16, "kn", "gelu_tanh"), (16, 136, 32, BF16, "kn", "silu"), (17, 128, 40, BF16, "nk", "relu"),
    (33, 200, 64, F16, "kn", "gelu"), (64, 64, 136, BF16, "nk", "silu"), (65, 1000, 64, BF16, "kn", "silu"), (127, 256, 200, F16, "nk", "gelu_tanh"),
    (129, 72, 72, BF16, "kn", "gelu"), (128, 192, 128, F16, "nk", "silu"), (256, 640, 136, BF16, "nk", "silu"), (300, 328, 264, BF16, "kn", "relu"),
    (511, 64, 520, F16, "kn", "silu"), (520, 520, 392, BF16, "nk", "gelu"), (1024, 128, 1024, F16, "nk", "silu"), (1100, 200, 1288, BF16, "kn", "silu"),
    # few rows of many outputs
    (3, 72, 8232, BF16, "kn", "silu"), (16, 1000, 8200, BF16, "nk", "gelu"), (20, 136, 8192, F16, "nk", "silu"), (31, 520, 8200, F16, "kn", "relu"),
    (40, 64, 8200, BF16, "kn", "gelu_tanh"), (64, 584, 8192, BF16, "nk", "silu"),
    # nothing divides: copies
    (5, 7, 3, BF16, "kn", "silu"), (70, 65, 129, F16, "nk", "gelu"), (257, 1001, 67, BF16, "kn", "gelu_tanh"), (100, 96, 101, F16, "kn", "silu"),
]


@pytest.mark.parametrize("rows, inputs, outputs, dtype, layout, act", FORWARD)
@pytest.mark.parametrize("keep", [False, True])
def test_forward(rows, inputs, outputs, dtype, layout, act, keep):
    x = rand((rows, inputs), 1, dtype)
    w, wd = weight_of(inputs, outputs, dtype, layout, 2)
    check_forward(ops.gated_linear(x.cuda(), wd, activation=act, keep=keep), x, w, act, keep)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("rows", [1, 30, 200])
def test_pitches_and_places(rows, layout):
    """Rows apart from each other, results anywhere: whole vectors, then none; NaN around every operand, which has no part."""
    inputs, outputs = 136, 72
    x = rand((rows, inputs), 3, BF16)
    for pad, offset in ((8, 8), (0, 1), (3, 5), (1, 0)):
        w, wd = weight_of(inputs, outputs, BF16, layout, 4, pad, offset)
        memory = torch.full((rows * (outputs + 5) + 3,), 7.0, dtype=BF16, device="cuda")
        out = memory[3:].as_strided((rows, outputs), (outputs + 5, 1))
        r = ops.gated_linear(placed(x, inputs + pad, offset), wd, out=out)
        assert r.out is out
        check_forward(r, x, w, "silu", False)
        left = torch.ones_like(memory, dtype=torch.bool)
        left[3:].as_strided((rows, outputs), (outputs + 5, 1)).fill_(False)
        assert bool((memory[left] == 7.0).all()), "bytes around the result were written"


@pytest.mark.parametrize("rows, inputs, outputs, dtype, layout, act", [c for c in FORWARD if c[0] not in (2, 64, 511)])
@pytest.mark.parametrize("keep", [True, False])
def test_backward(rows, inputs, outputs, dtype, layout, act, keep):
    if act == "relu" and not keep:
        act = "silu"  # its derivative jumps: a projection near 0 that is computed again may be on the other side
    x, dh = rand((rows, inputs), 5, dtype), rand((rows, outputs), 6, dtype, 0.1)
    w, wd = weight_of(inputs, outputs, dtype, layout, 7)
    g, u, s = ref.projections(x, w)
    kept, eg, eu = None, inputs * SUM * s[:, :outputs], inputs * SUM * s[:, outputs:]
    if keep:
        kept = torch.cat([g, u], dim=1).to(dtype)
        g, u, eg, eu = kept[:, :outputs], kept[:, outputs:], torch.zeros_like(eg), torch.zeros_like(eu)
    d = ops.gated_linear_backward(dh.cuda(), None if kept is None else kept.cuda(), x.cuda(), wd, activation=act)
    want, bound = inner_bounds(dh, g, u, eg, eu, dtype, act)
    within(d.inner, want, bound, "inner")
    inner = d.inner.cpu().double()
    dx = inner @ w.double().t()
    within(d.x, dx, rounded(dx, 2 * outputs * SUM * (inner.abs() @ w.double().abs().t()), dtype), "dx")
    dw = x.double().t() @ inner
    assert d.weight.dtype == F32 and d.weight.stride() == ((2 * outputs, 1) if layout == "kn" else (1, inputs))
    within(d.weight, dw, (rows + 1) * SUM * (x.double().abs().t() @ inner.abs()), "dweight")


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("rows, inputs, outputs", [(1, 24, 8), (30, 136, 72), (200, 65, 36), (530, 264, 201)])
def test_backward_pitches_and_places(rows, inputs, outputs, layout):
    """Every operand and inner in rows apart from each other, anywhere, NaN around them: whole vectors, then none."""
    x, dh = rand((rows, inputs), 44, BF16), rand((rows, outputs), 45, BF16, 0.1)
    for pad, offset in ((8, 8), (0, 1), (5, 3)):
        w, wd = weight_of(inputs, outputs, BF16, layout, 46, pad, offset)
        g, u, s = ref.projections(x, w)
        kept = torch.cat([g, u], dim=1).to(BF16)
        for z in (None, placed(kept, 2 * outputs + pad, offset)):
            memory = torch.full((rows * (2 * outputs + pad) + offset + 9,), 7.0, dtype=BF16, device="cuda")
            out = memory[offset:].as_strided((rows, 2 * outputs), (2 * outputs + pad, 1))
            d = ops.gated_linear_backward(placed(dh, outputs + pad, offset), z, placed(x, inputs + pad, offset), wd, out=out)
            assert d.inner is out
            e = inputs * SUM * s if z is None else torch.zeros_like(s)
            a, b = (g, u) if z is None else (kept[:, :outputs], kept[:, outputs:])
            want, bound = inner_bounds(dh, a, b, e[:, :outputs], e[:, outputs:], BF16, "silu")
            within(out, want, bound, "inner")
            inner = out.cpu().double()
            dx = inner @ w.double().t()
            within(d.x, dx, rounded(dx, 2 * outputs * SUM * (inner.abs() @ w.double().abs().t()), BF16), "dx")
            within(d.weight, x.double().t() @ inner, (rows + 16) * SUM * (x.double().abs().t() @ inner.abs()), "dweight")
            out.fill_(7.0)
            assert bool((memory == 7.0).all()), "bytes around inner were written"


# Sums over the projections that are split over workgroups.
LONG = [(300, 264, 16384 // 2, BF16, "kn"), (1030, 232, 8200, F16, "nk"), (200, 1001, 8195, BF16, "kn"), (700, 703, 4100, F16, "nk"), (1003, 1000, 2100, BF16, "kn")]


@pytest.mark.parametrize("rows, inputs, outputs, dtype, layout", LONG)
def test_input_gradient_from_many_outputs(rows, inputs, outputs, dtype, layout):
    dh, kept = rand((rows, outputs), 61, dtype, 0.1), rand((rows, 2 * outputs), 62, dtype)
    w, wd = weight_of(inputs, outputs, dtype, layout, 63, pad=3 * (inputs % 8 > 0), offset=inputs % 8)
    for pad in (0, 5):
        d = ops.gated_linear_backward(dh.cuda(), placed(kept, 2 * outputs + pad, pad), None, wd, weights=False,
                                      out=torch.empty(rows, 2 * outputs + pad, dtype=dtype, device="cuda")[:, : 2 * outputs])
        inner = d.inner.cpu().double()
        want = inner @ w.double().t()
        within(d.x, want, rounded(want, 2 * outputs * SUM * (inner.abs() @ w.double().abs().t()), dtype), "dx")
        assert d.x.is_contiguous() and torch.equal(d.x, ops.gated_linear_backward(dh.cuda(), kept.cuda(), None, wd, weights=False).x)


def test_backward_against_differences():
    """The gradients are those of sum(dh * gated(x, w)): against differences of the 64-bit definition."""
    rows, inputs, outputs = 3, 16, 8
    for act in ("silu", "gelu", "gelu_tanh"):
        x, dh = rand((rows, inputs), 8, F16), rand((rows, outputs), 9, F16)
        w, wd = weight_of(inputs, outputs, F16, "kn", 10)

        def loss(x, w):
            g, u, _ = ref.projections(x, w)
            return float((dh.double() * ref.activation(g, act)[0] * u).sum())

        d = ops.gated_linear_backward(dh.cuda(), None, x.cuda(), wd, activation=act)
        step = 2.0**-16
        for grad, which in ((d.x.cpu().double(), 0), (d.weight.cpu().double(), 1)):
            for i, j in ((0, 0), (2, 7), (1, 15)):
                ends = []
                for sign in (1, -1):
                    args = [x.double().clone(), w.double().clone()]
                    args[which][i, j] += sign * step
                    ends.append(loss(*args))
                slope = (ends[0] - ends[1]) / (2 * step)
                # 16-bit roundings of inner (2^-11 of 16 or 3 terms) and of dx; differences are good to 2^-30 here.
                assert abs(float(grad[i, j]) - slope) <= 2.0**-10 * 16, (act, which, i, j)


def test_gradients_go_where_they_are_wanted():
    rows, inputs, outputs = 40, 64, 24
    x, dh = rand((rows, inputs), 11, BF16), rand((rows, outputs), 12, BF16)
    for layout in ("kn", "nk"):
        w, wd = weight_of(inputs, outputs, BF16, layout, 13)
        kept = ops.gated_linear(x.cuda(), wd, keep=True).kept
        plain = ops.gated_linear_backward(dh.cuda(), kept, x.cuda(), wd)
        more = rand((inputs, 2 * outputs), 14)
        md = more.cuda() if layout == "kn" else more.t().contiguous().cuda().t()
        summed = ops.gated_linear_backward(dh.cuda(), kept, x.cuda(), wd, add=md)
        want = plain.weight.cpu().double() + more.double()
        within(summed.weight, want, half(want.abs(), F32) * 4 + 2.0**-22, "dweight on top of another")
        assert summed.weight.stride() == plain.weight.stride()
        short = ops.gated_linear_backward(dh.cuda(), kept, x.cuda(), wd, out_dtype=BF16)
        assert short.weight.dtype == BF16
        within(short.weight, plain.weight.cpu(), half(plain.weight.cpu().abs(), BF16), "dweight in 16 bits")
        only = ops.gated_linear_backward(dh.cuda(), kept, x.cuda(), wd, inputs=False, weights=False)
        assert only.x is None and only.weight is None and torch.equal(only.inner, plain.inner)
        held = ops.checkpoint_activation(x.cuda())
        from_held = ops.gated_linear_backward(dh.cuda(), kept, held, wd, inputs=False)
        assert torch.equal(from_held.inner, plain.inner)
        xr = ops.restore_activation(held).cpu().double()
        inner = plain.inner.cpu().double()
        within(from_held.weight, xr.t() @ inner, (rows + 1) * SUM * (xr.abs().t() @ inner.abs()), "dweight from 8 bits")
        again = kept.clone()
        same = ops.gated_linear_backward(dh.cuda(), again, x.cuda(), wd, out=again)
        assert same.inner is again and torch.equal(again, plain.inner), "inner in the place of kept"


def test_no_rows():
    w, wd = weight_of(64, 24, BF16, "kn", 15)
    r = ops.gated_linear(torch.empty(0, 64, dtype=BF16, device="cuda"), wd, keep=True)
    assert r.out.shape == (0, 24) and r.kept.shape == (0, 48)
    for kept in (r.kept, None):
        d = ops.gated_linear_backward(torch.empty(0, 24, dtype=BF16, device="cuda"), kept, torch.empty(0, 64, dtype=BF16, device="cuda"), wd)
        assert d.inner.shape == (0, 48) and d.x.shape == (0, 64) and d.weight.shape == (64, 48) and not bool(d.weight.any())


@pytest.mark.parametrize("act", ACTS)
def test_values_at_the_ends(act):
    """Large and small projections, zeros, NaN and infinity in one input: what the definition makes of them, and nobody else's."""
    inputs, outputs = 8, 16
    x = torch.zeros(12, inputs, dtype=F32)
    x[:, 0] = torch.tensor([0.0, -0.0, 1e-3, 20.0, -20.0, 90.0, -90.0, 1e4, -1e4, float("nan"), float("inf"), 3.0])
    x[:, 1] = 1.0
    w = torch.zeros(inputs, 2 * outputs)
    w[0, :outputs], w[1, outputs:] = 1.0, 2.0
    x, w = x.to(BF16), w.to(BF16)
    r = ops.gated_linear(x.cuda(), w.cuda(), activation=act)
    g = x.double() @ w.double()[:, :outputs]
    g[10] = float("inf")  # inf * 1 + zeros; the other half has inf * 0
    want, _ = ref.activation(g, act)
    want = want * 2.0
    want[9], want[10] = float("nan"), float("nan")
    within(r.out, want, rounded(want, 2.0**-19 * (g.abs() + 1), BF16), "out")


@pytest.mark.parametrize("rows", [2, 200])
@pytest.mark.parametrize("up", [8, (1 << 22) + 8, 1 << 23])
def test_halves_far_from_each_other(lib, rows, up):
    """One row of a weight by rows, whose second half lies further on than a pitch may be: a copy, the C entry asks for room for it."""
    outputs = 8
    x, memory = rand((rows, 1), 51, BF16), torch.full((up + outputs,), float("nan"), dtype=BF16, device="cuda")
    w = rand((1, 2 * outputs), 52, BF16)
    memory[:outputs], memory[up:] = w[0, :outputs].cuda(), w[0, outputs:].cuda()
    xd, out = x.cuda(), torch.empty(rows, outputs, dtype=BF16, device="cuda")
    d = _lib.GatedDesc(x=xd.data_ptr(), weight=memory.data_ptr(), out=out.data_ptr(), ld_x=1, ld_weight=2 * outputs, up=up, ld_out=outputs, rows=rows, inputs=1,
                       outputs=outputs, dtype=_lib.BF16)
    d.workspace_bytes = lib.tccl_gated_workspace(ctypes.byref(d))
    assert d.workspace_bytes >= 256 * (1 + (up > 1 << 22))  # of x, and of the weight
    workspace = torch.empty(d.workspace_bytes, dtype=torch.uint8, device="cuda")
    d.workspace = workspace.data_ptr()
    assert lib.tccl_gated(ctypes.byref(d), torch.cuda.current_stream().cuda_stream) == 0
    g, u, s = ref.projections(x, w)
    want, bound = gated_bounds(g, u, s, 1, BF16, "silu")
    within(out, want, bound, "out")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows", [8, 300])
def test_gradients_at_the_ends(act, rows):
    """Projections as they were kept and computed again: large ones, zeros and NaN, whose gradients are NaN (relu's of the gate: 0)."""
    inputs, outputs = 8, 16
    ends = torch.tensor([0.0, 1e-3, 20.0, -20.0, 1e4, -1e4, 3e8, float("nan")])
    x = torch.zeros(rows, inputs)
    x[:8, 0], x[:, 1] = ends, 1.0
    w = torch.zeros(inputs, 2 * outputs)
    w[0, :outputs], w[1, outputs:] = 1.0, 2.0
    x, w, dh = x.to(BF16), w.to(BF16), torch.ones(rows, outputs, dtype=BF16)
    g, u = x.double() @ w.double()[:, :outputs], torch.full((rows, outputs), 2.0, dtype=torch.float64)
    g[7] = float("nan")
    kept = torch.cat([g, u], dim=1).to(BF16)
    exact, error = ref.gated_gradient(dh, g, u, act), 2.0**-18 * (g.nan_to_num(0.0).abs() + 1)
    bound = rounded(exact, torch.cat([error, error], dim=1), BF16)
    for z in (kept, None):
        inner = ops.gated_linear_backward(dh.cuda(), None if z is None else z.cuda(), x.cuda(), w.cuda(), activation=act, inputs=False, weights=False).inner.cpu()
        within(inner[:7], exact[:7], bound[:7], "inner")
        assert bool(torch.isnan(inner[7, outputs:]).all()), "du = dh act(NaN)"
        # (computed again, u of that row is 0 * NaN + 2, too: relu's dg is NaN * 0)
        assert bool(torch.isnan(inner[7, :outputs]).all()) or (act == "relu" and z is not None), "dg = dh u act'(NaN)"


@pytest.mark.parametrize("rows, layout", [(3, "nk"), (200, "kn"), (600, "nk")])
def test_graph_and_stream(rows, layout):
    """Recorded calls give the eager result at every replay, beside eager calls of their own; so does another stream."""
    inputs, outputs = 264, 136
    x, dh = rand((rows, inputs), 16, F16).cuda(), rand((rows, outputs), 17, F16).cuda()
    _, w = weight_of(inputs, outputs, F16, layout, 18)

    def both():
        r = ops.gated_linear(x, w, keep=True)
        return (*r, *ops.gated_linear_backward(dh, r.kept, x, w), *ops.gated_linear_backward(dh, None, x, w, inputs=False, weights=False)[:1])

    eager = [t.clone() for t in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, there))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = both()
    for replay in range(3):
        x.copy_(rand((rows, inputs), 19 + replay, F16))
        for t in recorded:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        now = both()
        assert all(torch.equal(a, b) for a, b in zip(recorded, now)), replay


# Inputs that are split over workgroups, in every kind of tile; 4104 and 2120 leave the last split a part of its blocks, 7175 no whole vector.
SPLIT = [
    (3, 4104, 40, BF16, "kn", "silu"), (1, 4104, 2056, F16, "kn", "gelu"), (20, 4104, 1032, BF16, "kn", "gelu_tanh"), (40, 4104, 1032, F16, "kn", "silu"),
    (61, 2120, 136, BF16, "kn", "relu"), (112, 7175, 104, BF16, "kn", "gelu"), (260, 4104, 264, BF16, "kn", "silu"), (130, 4104, 2056, F16, "kn", "silu"),
    (2, 4104, 8, F16, "nk", "silu"), (16, 4104, 1032, BF16, "nk", "gelu_tanh"), (25, 2120, 72, BF16, "nk", "silu"), (30, 4104, 1032, F16, "nk", "gelu"),
    (50, 2120, 101, BF16, "nk", "silu"), (64, 4104, 1032, BF16, "nk", "silu"), (260, 4104, 264, F16, "nk", "gelu"), (500, 4104, 1040, BF16, "nk", "silu"),
    (500, 4104, 516, F16, "nk", "gelu_tanh"), (500, 4104, 516, BF16, "kn", "silu"),
]


@pytest.mark.parametrize("rows, inputs, outputs, dtype, layout, act", SPLIT)
def test_inputs_split_over_workgroups(rows, inputs, outputs, dtype, layout, act):
    x, dh = rand((rows, inputs), 41, dtype), rand((rows, outputs), 42, dtype, 0.1)
    w, wd = weight_of(inputs, outputs, dtype, layout, 43)
    memory = torch.full((rows + 2, 2 * outputs + 3), 7.0, dtype=dtype, device="cuda")
    r = ops.gated_linear(x.cuda(), wd, activation=act, keep=True)
    check_forward(r, x, w, act, True)
    r = ops.gated_linear(x.cuda(), wd, activation=act, out=memory[1:-1, 1 : outputs + 1])
    check_forward(r, x, w, act, False)
    act = "silu" if act == "relu" else act
    g, u, s = ref.projections(x, w)
    want, bound = inner_bounds(dh, g, u, inputs * SUM * s[:, :outputs], inputs * SUM * s[:, outputs:], dtype, act)
    d = ops.gated_linear_backward(placed(dh, outputs + 5, 1), None, x.cuda(), wd, activation=act, inputs=False, weights=False, out=memory[1:-1, 1:-2])
    within(d.inner, want, bound, "inner")
    memory[1:-1, 1:-2].fill_(7.0)
    assert bool((memory == 7.0).all()), "bytes around a result were written"


# Beyond what small tiles take in one round of the device: 256 x 128 tiles, with parts of one at every edge.
LARGE = [(2100, 72, 2056, BF16, "kn", "silu"), (2056, 200, 2100, BF16, "nk", "gelu"), (4096, 64, 1024, F16, "kn", "gelu_tanh"), (2049, 328, 2048, F16, "nk", "silu")]


@pytest.mark.parametrize("rows, inputs, outputs, dtype, layout, act", LARGE)
def test_large_tiles(rows, inputs, outputs, dtype, layout, act):
    x, dh = rand((rows, inputs), 31, dtype), rand((rows, outputs), 32, dtype, 0.1)
    w, wd = weight_of(inputs, outputs, dtype, layout, 33)
    r = ops.gated_linear(x.cuda(), wd, activation=act, keep=True)
    check_forward(r, x, w, act, True)
    assert torch.equal(ops.gated_linear(x.cuda(), wd, activation=act).out, r.out)
    g, u, s = ref.projections(x, w)
    d = ops.gated_linear_backward(dh.cuda(), None, x.cuda(), wd, activation=act, inputs=False, weights=False)
    want, bound = inner_bounds(dh, g, u, inputs * SUM * s[:, :outputs], inputs * SUM * s[:, outputs:], dtype, act)
    within(d.inner, want, bound, "inner")
