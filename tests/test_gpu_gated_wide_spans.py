"""The kernels for few rows, of the gated layer and of the GEMM that makes its input's gradient, where an operand reaches further than 32 bits from a
tile's first row: what lies past the summed index reads as zero there, too.  NaN between the rows, which has no part, and sums that end within a step of
64."""

import pytest
import torch

from tests.layer_bounds import F16, rand
from tests.test_gpu_gated import weight_of
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory_goes_back():
    yield
    torch.cuda.empty_cache()


def apart(t, pitch):
    """``t`` on the GPU, its rows ``pitch`` elements from each other, NaN between them."""
    rows, cols = t.shape
    view = torch.full((rows * pitch,), float("nan"), dtype=t.dtype, device="cuda").as_strided((rows, cols), (pitch, 1))
    view.copy_(t)
    return view


@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_rows_of_x_far_apart(layout):
    rows, inputs, outputs = 1100, 72, 48
    xs, dh = rand((rows, inputs), 1, F16), rand((rows, outputs), 2, F16, 0.1).cuda()
    x, packed = apart(xs, (1 << 21) + 8), xs.cuda()
    _, w = weight_of(inputs, outputs, F16, layout, 3)
    want = ops.gated_linear(packed, w, keep=True)
    assert bool(torch.isfinite(want.out).all())
    got = ops.gated_linear(x, w, keep=True)
    assert torch.equal(got.out, want.out) and torch.equal(got.kept, want.kept)
    inner = [ops.gated_linear_backward(dh, None, t, w, inputs=False, weights=False).inner for t in (x, packed)]
    assert torch.equal(*inner)


@pytest.mark.parametrize("rows", [5, 20, 40])
def test_rows_of_a_weight_far_apart(rows):
    inputs, outputs = 72, 600
    x = rand((rows, inputs), 4, F16).cuda()
    ws = rand((2 * outputs, inputs), 5, F16, inputs**-0.5)
    want = ops.gated_linear(x, ws.cuda().t(), keep=True)
    assert bool(torch.isfinite(want.out).all())
    got = ops.gated_linear(x, apart(ws, 1 << 22).t(), keep=True)
    assert torch.equal(got.out, want.out) and torch.equal(got.kept, want.kept)


def test_input_gradient_of_rows_far_apart():
    rows, inputs, outputs = 1100, 16, 36
    dh, kept = rand((rows, outputs), 6, F16, 0.1).cuda(), rand((rows, 2 * outputs), 7, F16).cuda()
    _, w = weight_of(inputs, outputs, F16, "kn", 8)
    out = apart(torch.zeros(rows, 2 * outputs, dtype=F16), (1 << 21) + 8)
    want = ops.gated_linear_backward(dh, kept, None, w, weights=False)
    assert bool(torch.isfinite(want.x).all())
    got = ops.gated_linear_backward(dh, kept, None, w, weights=False, out=out)
    assert torch.equal(got.inner, want.inner) and torch.equal(got.x, want.x)


def test_input_gradient_of_a_weight_far_apart():
    rows, inputs, outputs = 5, 600, 36
    dh, kept = rand((rows, outputs), 9, F16, 0.1).cuda(), rand((rows, 2 * outputs), 10, F16).cuda()
    ws = rand((inputs, 2 * outputs), 11, F16, 0.1)
    want = ops.gated_linear_backward(dh, kept, None, ws.cuda(), weights=False)
    assert bool(torch.isfinite(want.x).all())
    assert torch.equal(ops.gated_linear_backward(dh, kept, None, apart(ws, 1 << 22), weights=False).x, want.x)


def test_input_gradient_of_many_rows_far_apart():
    """The GEMM in 128 tiles."""
    rows, inputs, outputs = 5000, 512, 36
    dh, kept = rand((rows, outputs), 12, F16, 0.1).cuda(), rand((rows, 2 * outputs), 13, F16).cuda()
    _, w = weight_of(inputs, outputs, F16, "kn", 14)
    want = ops.gated_linear_backward(dh, kept, None, w, weights=False)
    assert bool(torch.isfinite(want.x).all())
    got = ops.gated_linear_backward(dh, kept, None, w, weights=False, out=apart(torch.zeros(rows, 2 * outputs, dtype=F16), (1 << 20) + 8))
    assert torch.equal(got.inner, want.inner) and torch.equal(got.x, want.x)


def test_input_gradient_of_many_rows_of_a_weight_far_apart():
    rows, inputs, outputs = 1100, 2000, 36
    dh, kept = rand((rows, outputs), 15, F16, 0.1).cuda(), rand((rows, 2 * outputs), 16, F16).cuda()
    ws = rand((inputs, 2 * outputs), 17, F16, 0.1)
    want = ops.gated_linear_backward(dh, kept, None, ws.cuda(), weights=False)
    assert bool(torch.isfinite(want.x).all())
    assert torch.equal(ops.gated_linear_backward(dh, kept, None, apart(ws, 1 << 21), weights=False).x, want.x)
