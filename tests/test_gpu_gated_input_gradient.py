"""``dx`` of the gated layer: where the GEMM does not reach over an operand, 4 GiB from a tile's base on, and in rows next to each other whichever kernel
makes it."""

import pytest
import torch

from tests.layer_bounds import BF16, F16, SUM, rand, rounded, within
from tests.test_gpu_gated import weight_of
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory_goes_back():
    yield
    torch.cuda.empty_cache()


def check(d, w, dtype):
    """``d.x`` against ``d.inner`` times the transpose of ``w`` (inputs, 2 * outputs), on the host."""
    inner, w = d.inner.cpu().double(), w.double()
    want = inner @ w.t()
    within(d.x, want, rounded(want, w.shape[1] * SUM * (inner.abs() @ w.abs().t()), dtype), "dx")


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("inputs, outputs", [(16384, 65536), (16379, 65541)])
def test_weight_of_more_than_4_gib(rows, inputs, outputs):
    """2 * outputs rows of inputs, as a linear layer holds them: zeros but for the first and the last ones."""
    some = 150
    ends = torch.cat([torch.arange(some), torch.arange(2 * outputs - some, 2 * outputs)])
    ws = rand((2 * some, inputs), 1, BF16, 0.05)
    held = torch.zeros(2 * outputs, inputs, dtype=BF16, device="cuda")
    held[ends.cuda()] = ws.cuda()
    dh, kept = rand((rows, outputs), 2, BF16).cuda(), rand((rows, 2 * outputs), 3, BF16).cuda()
    d = ops.gated_linear_backward(dh, kept, None, held.t(), weights=False)
    part = d.inner[:, ends.cuda()].cpu().double()
    want = part @ ws.double()
    within(d.x, want, rounded(want, 2 * some * SUM * (part.abs() @ ws.double().abs()), BF16), "dx")  # (zeros add nothing)


@pytest.mark.parametrize("rows", [4, 130])
def test_rows_of_a_weight_far_apart(rows):
    """By rows, 2^24 elements from each other."""
    inputs, outputs, pitch = 24, 40, 1 << 24
    w = rand((inputs, 2 * outputs), 4, F16)
    wd = torch.full((inputs * pitch,), float("nan"), dtype=F16, device="cuda").as_strided((inputs, 2 * outputs), (pitch, 1))
    wd.copy_(w)
    x, dh = rand((rows, inputs), 5, F16).cuda(), rand((rows, outputs), 6, F16).cuda()
    check(ops.gated_linear_backward(dh, None, x, wd), w, F16)


@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_rows_of_inner_far_apart(layout):
    rows, inputs, outputs, pitch = 5, 24, 40, (1 << 23) + 65536
    w, wd = weight_of(inputs, outputs, F16, layout, 7)
    out = torch.full((rows * pitch,), float("nan"), dtype=F16, device="cuda").as_strided((rows, 2 * outputs), (pitch, 1))
    x, dh = rand((rows, inputs), 8, F16).cuda(), rand((rows, outputs), 9, F16).cuda()
    d = ops.gated_linear_backward(dh, None, x, wd, out=out)
    assert d.inner is out
    check(d, w, F16)


@pytest.mark.parametrize("rows, inputs, outputs, layout", [(0, 13, 8, "kn"), (1, 13, 8, "nk"), (70, 65, 36, "kn"), (530, 263, 201, "nk"), (300, 264, 72, "kn"), (1500, 1001, 24, "nk"),
                                                            (4, 1001, 4100, "kn"), (60, 333, 2000, "nk"), (3000, 2049, 300, "kn")])
def test_rows_next_to_each_other(rows, inputs, outputs, layout):
    w, wd = weight_of(inputs, outputs, BF16, layout, 10)
    x, dh = rand((rows, inputs), 11, BF16).cuda(), rand((rows, outputs), 12, BF16).cuda()
    d = ops.gated_linear_backward(dh, None, x, wd, weights=False)
    assert d.x.shape == (rows, inputs) and d.x.is_contiguous()
    check(d, w, BF16)
