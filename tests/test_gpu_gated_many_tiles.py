"""The gated layer over more rows than a launch has workgroups for: what lies at both ends, zeros between."""

import pytest
import torch

from oracle import layers as ref
from tests.layer_bounds import BF16, SUM, gated_bounds, inner_bounds, rand, rounded, within
from tests.test_gpu_gated import weight_of
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory_goes_back():
    yield
    torch.cuda.empty_cache()


SOME = 300


def tall(rows, cols, seed):
    """A matrix of zeros but for some rows at either end, and these on the host."""
    t = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    some = rand((2 * SOME, cols), seed, BF16)
    t[:SOME], t[-SOME:] = some[:SOME].cuda(), some[SOME:].cuda()
    return t, some


def ends(t):
    return torch.cat([t[:SOME], t[-SOME:]])


def nothing_between(t):
    return not any(bool(part.any()) for part in t[SOME:-SOME].split(1 << 28))


def test_projections():
    rows, inputs, outputs = (1 << 30) + 300, 8, 8
    x, xs = tall(rows, inputs, 1)
    w, wd = weight_of(inputs, outputs, BF16, "nk", 2)
    g, u, s = ref.projections(xs, w)
    out = ops.gated_linear(x, wd).out
    want, bound = gated_bounds(g, u, s, inputs, BF16, "silu")
    within(ends(out), want, bound, "out")
    assert nothing_between(out)
    dh, dhs = tall(rows, outputs, 3)
    inner = ops.gated_linear_backward(dh, None, x, wd, inputs=False, weights=False).inner
    want, bound = inner_bounds(dhs, g, u, inputs * SUM * s[:, :outputs], inputs * SUM * s[:, outputs:], BF16, "silu")
    within(ends(inner), want, bound, "inner")
    assert nothing_between(inner)


@pytest.mark.parametrize("rows, inputs", [((1 << 30) + 300, 8), ((1 << 29) + 300, 13)])
def test_input_gradient(rows, inputs):
    outputs = 8
    _, wd = weight_of(inputs, outputs, BF16, "kn", 4)
    dh, _ = tall(rows, outputs, 5)
    kept, _ = tall(rows, 2 * outputs, 6)
    d = ops.gated_linear_backward(dh, kept, None, wd, out=kept, weights=False)
    inner = ends(d.inner).cpu().double()
    want = inner @ wd.cpu().double().t()
    within(ends(d.x), want, rounded(want, 2 * outputs * SUM * (inner.abs() @ wd.cpu().double().abs().t()), BF16), "dx")
    assert nothing_between(d.x)
