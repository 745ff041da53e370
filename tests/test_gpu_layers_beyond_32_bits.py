"""The gated layer, weight gradients from an input in full and AdamW where offsets pass 32 bits: operands of more than 4 GiB, places in flat memory
beyond 2^32, the longest inputs and outputs.  What lies at both ends of an operand is held to 64 bits."""

import pytest
import torch

from oracle import layers as ref
from tests.layer_bounds import BF16, F16, F32, SUM, gated_bounds, inner_bounds, rand, rounded, within
from tests.test_gpu_adamw import HOW, check_held
from tests.test_gpu_gated import weight_of
from tileccl_amd import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory_goes_back():
    yield
    torch.cuda.empty_cache()


def tall(rows, cols, seed, dtype, ends):
    """A matrix of zeros but for 300 rows at either end, and these on the host."""
    t = torch.zeros(rows, cols, dtype=dtype, device="cuda")
    some = rand((600, cols), seed, dtype)
    t[ends] = some.cuda()
    return t, some


ROWS = 620_003


@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_many_rows(layout):
    """x of 5 GiB, 2^31 + 392 million elements of it, through tiles, and the weight gradient's sum over them."""
    inputs, outputs = 4096, 40
    ends = torch.cat([torch.arange(300), torch.arange(ROWS - 300, ROWS)])
    x, xs = tall(ROWS, inputs, 1, BF16, ends)
    dh, dhs = tall(ROWS, outputs, 2, BF16, ends)
    w, wd = weight_of(inputs, outputs, BF16, layout, 3)
    g, u, s = ref.projections(xs, w)
    out = ops.gated_linear(x, wd).out
    want, bound = gated_bounds(g, u, s, inputs, BF16, "silu")
    within(out[ends.cuda()], want, bound, "out")
    assert not bool(out[300:-300].any())
    d = ops.gated_linear_backward(dh, None, x, wd)
    want, bound = inner_bounds(dhs, g, u, inputs * SUM * s[:, :outputs], inputs * SUM * s[:, outputs:], BF16, "silu")
    inner = d.inner[ends.cuda()].cpu()
    within(inner, want, bound, "inner")
    dx = inner.double() @ w.double().t()
    within(d.x[ends.cuda()], dx, rounded(dx, 2 * outputs * SUM * (inner.double().abs() @ w.double().abs().t()), BF16), "dx")
    assert not bool(d.x[300:-300].any())
    dw = xs.double().t() @ inner.double()
    within(d.weight, dw, (600 + 16) * SUM * (xs.double().abs().t() @ inner.double().abs()), "dweight")  # (zeros add nothing; splits: 16)


def test_results_with_a_large_pitch():
    """Pitches of 2^21 + 8 elements put the last rows beyond 4 GiB of the first."""
    rows, inputs, outputs, pitch = 1100, 64, 48, (1 << 21) + 8
    memory = torch.full((rows * pitch,), 7.0, dtype=F16, device="cuda")
    x, out = memory.as_strided((rows, inputs), (pitch, 1)), memory.as_strided((rows, outputs), (pitch, 1), 1 << 20)
    xs = rand((rows, inputs), 4, F16)
    x.copy_(xs)
    w, wd = weight_of(inputs, outputs, F16, "kn", 5)
    with pytest.raises(ValueError, match="out overlaps x"):  # rows between rows count as the matrix's
        ops.gated_linear(x, wd, out=out)
    r = ops.gated_linear(x, wd, keep=True)
    g, u, s = ref.projections(xs, w)
    want, bound = gated_bounds(g, u, s, inputs, F16, "silu")
    within(r.out, want, bound, "out")
    other = torch.zeros(rows * pitch, dtype=F16, device="cuda")
    apart = other.as_strided((rows, outputs), (pitch, 1), 3)
    ops.gated_linear(xs.cuda(), wd, out=apart)
    within(apart, want, bound, "out with a pitch")
    apart.zero_()
    assert not bool(other.any())


@pytest.mark.parametrize("rows, inputs, outputs, layout", [(2, _lib.GATED_MAX_COLS, 3, "kn"), (3, _lib.GATED_MAX_COLS, 8, "nk"), (2, 8, _lib.GATED_MAX_COLS, "kn"),
                                                            (2, 8, _lib.GATED_MAX_COLS - 5, "nk"), (66, 8, 262139, "nk")])
def test_longest_inputs_and_outputs(rows, inputs, outputs, layout):
    """Operands of -1, 0 and 1, whose sums are exact."""
    draw = torch.Generator().manual_seed(6)
    x, w = ((torch.randint(-1, 2, shape, generator=draw)).to(BF16) for shape in ((rows, inputs), (inputs, 2 * outputs)))
    dh = rand((rows, outputs), 7, BF16)
    wd = w.cuda() if layout == "kn" else w.t().contiguous().cuda().t()
    g, u, s = ref.projections(x, w)
    r = ops.gated_linear(x.cuda(), wd)
    want, bound = gated_bounds(g, u, s, 0, BF16, "silu")
    within(r.out, want, bound, "out")
    none = torch.zeros_like(g)
    want, bound = inner_bounds(dh, g, u, none, none, BF16, "silu")
    d = ops.gated_linear_backward(dh.cuda(), None, x.cuda(), wd, inputs=False, out_dtype=BF16)
    within(d.inner, want, bound, "inner")
    inner = d.inner.cpu().double()
    dw = x.double().t() @ inner
    within(d.weight, dw, rounded(dw, (rows + 1) * SUM * (x.double().abs().t() @ inner.abs()), BF16), "dweight")


def test_adamw_places_beyond_32_bits():
    """2^32 + 5000 weights in 16 bits, moments in 8: the last ones and the first."""
    n, step = (1 << 32) + 5000, 12
    p, g = torch.zeros(n, dtype=BF16, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda")
    spans = [slice(0, 640), slice(n - 5128, n)]  # from whole blocks on
    held = [(rand((t.stop - t.start,), 9 + i, BF16), rand((t.stop - t.start,), 11 + i, BF16, 0.1)) for i, t in enumerate(spans)]
    for t, (ps, gs) in zip(spans, held):
        p[t], g[t] = ps.cuda(), gs.cuda()
    state = ops.AdamWState.zeros([p], bits=8)
    ops.adamw_step([p], [g], state, step=step, **HOW)
    for t, (ps, gs) in zip(spans, held):
        zero = torch.zeros(ps.numel(), dtype=torch.float64)
        want_p, want_m, want_v = ref.adamw(ps, gs, zero, zero, step=step, grad_scale=1.0, **HOW)
        within(p[t], want_p, rounded(want_p, 2.0**-21 * ps.double().abs() + 2.0**-19 * want_p.abs() + 2.0**-19 * 10 * HOW["lr"], BF16), "params")
        fill = -ps.numel() % ref.BLOCK
        h = [ref.noise(t.start + i, step) for i in range(ps.numel() + fill)]
        um, uv = (torch.tensor([x & 0xFFFF for x in h], dtype=torch.float64) / 65536, torch.tensor([x >> 16 for x in h], dtype=torch.float64) / 65536)
        mask = torch.arange(ps.numel() + fill) < ps.numel()
        blocks = slice(t.start // ref.BLOCK, (t.start + len(h)) // ref.BLOCK)
        bytes_ = slice(t.start, t.start + len(h))
        pad = lambda y: torch.cat([y, torch.zeros(fill, dtype=torch.float64)])  # noqa: E731
        check_held(state.first[bytes_].cpu(), state.first_scales[blocks].cpu(), pad(want_m), um, ref.FIRST, ref.first_exponent, 0.0, "first", mask)
        check_held(state.second[bytes_].cpu(), state.second_scales[blocks].cpu(), pad(want_v), uv, ref.SECOND, ref.second_exponent, 2.0**-30, "second", mask)
    assert not bool(p[640 : n - 5128].any()) and not bool(state.second[640 : n - 5128].any())


def test_largest_second_moments():
    """v in [2^127, 2^128), where the code above the last is no fp32: held as one of the codes around it that are."""
    n = 4096
    g = (2.0 ** torch.linspace(63.5, 63.999, n, dtype=torch.float64)).float()
    p = torch.zeros(n, device="cuda")
    state = ops.AdamWState.zeros([p], bits=8)
    ops.adamw_step([p], [g.cuda()], state, step=3, betas=(0.0, 0.0), lr=0.5, weight_decay=0.0)
    v = g.double() ** 2 / 2.0**127
    got = ops.adamw_moments(state)[1].cpu().double() / 2.0**127
    assert bool((state.second_scales == 254).all()) and bool(torch.isfinite(got).all())
    low, high = ref.neighbours(v, ref.SECOND)
    assert bool(((got == low) | (got == high.clamp(max=1.875)) | ((v - high).abs() < 1e-5) | ((v - low).abs() < 1e-5)).all())
    assert torch.allclose(p.cpu(), torch.full((n,), -0.5), rtol=2.0**-20)  # m / sqrt(v) = 1
