"""Weight gradients from an input in full against their definition in 64 bits (bounds: layer_bounds.py)."""

import pytest
import torch

from tests.layer_bounds import BF16, F16, F32, SUM, half, placed, rand, rounded, within
from tileccl_amd import ops

pytestmark = pytest.mark.gpu

SHAPES = [
    # tokens, inputs, outputs: one of each, around steps of 64, vectors and tiles; long sums of few outputs
    (1, 8, 8), (1, 1, 1), (2, 16, 64), (63, 64, 72), (64, 128, 128), (65, 136, 120), (200, 256, 64), (129, 264, 520), (700, 512, 256), (1000, 384, 640),
    (4100, 64, 48), (5000, 256, 264), (257, 1288, 520),
    (7, 5, 3), (100, 67, 33), (300, 129, 1001), (1003, 250, 70),
]


@pytest.mark.parametrize("tokens, inputs, outputs", SHAPES)
@pytest.mark.parametrize("dtype, out_dtype, layout, add", [(BF16, F32, "kn", False), (F16, F32, "nk", True), (BF16, BF16, "nk", False), (F16, F16, "kn", True)])
def test_weight_gradient(tokens, inputs, outputs, dtype, out_dtype, layout, add):
    x, dy = rand((tokens, inputs), 1, dtype), rand((tokens, outputs), 2, dtype, 0.1)
    shape = (inputs, outputs) if layout == "kn" else (outputs, inputs)
    more = rand(shape, 3, out_dtype) if add else None
    got = ops.weight_gradient(x.cuda(), dy.cuda(), layout=layout, out_dtype=out_dtype, add=None if more is None else more.cuda())
    want, top = x.double().t() @ dy.double(), x.double().abs().t() @ dy.double().abs()
    if layout == "nk":
        want, top = want.t(), top.t()
    if add:
        want, top = want + more.double(), top + more.double().abs()
    assert got.dtype == out_dtype and got.is_contiguous()
    within(got, want, rounded(want, (tokens + 8) * SUM * top, out_dtype), "dweight")


@pytest.mark.parametrize("tokens", [1, 64, 70, 128, 200, 449])
@pytest.mark.parametrize("inputs, outputs, layout", [(4200, 2056, "kn"), (2056, 4200, "nk"), (4096, 2304, "nk")])
def test_large_tiles(tokens, inputs, outputs, layout):
    x, dy = rand((tokens, inputs), 21, BF16), rand((tokens, outputs), 22, BF16)
    got = ops.weight_gradient(x.cuda(), dy.cuda(), layout=layout)
    want, top = x.double().t() @ dy.double(), x.double().abs().t() @ dy.double().abs()
    if layout == "nk":
        want, top = want.t(), top.t()
    within(got, want, rounded(want, tokens * SUM * top, F32), "dweight")
    # on top of another, into it, and with rows that are no vectors
    shape = tuple(got.shape)
    for pitch, offset in ((shape[1], 0), (shape[1] + 4, 4), (shape[1] + 1, 1)):
        memory = torch.zeros(shape[0] * pitch + offset, device="cuda")
        more = memory[offset:].as_strided(shape, (pitch, 1))
        more.copy_(rand(shape, 23))
        first = more.cpu().double()
        assert ops.weight_gradient(x.cuda(), dy.cuda(), layout=layout, add=more, out=more) is more
        within(more, want + first, rounded(want + first, (tokens + 1) * SUM * (top + first.abs()), F32), "dweight on top of another")


def test_pitches_and_places():
    tokens, inputs, outputs = 150, 72, 200
    x, dy = rand((tokens, inputs), 4, BF16), rand((tokens, outputs), 5, BF16)
    want, top = x.double().t() @ dy.double(), x.double().abs().t() @ dy.double().abs()
    for pad, offset in ((8, 16), (3, 0), (0, 1)):
        memory = torch.full((inputs * (outputs + 3) + 1,), 7.0, device="cuda")
        out = memory[1:].as_strided((inputs, outputs), (outputs + 3, 1))
        got = ops.weight_gradient(placed(x, inputs + pad, offset), placed(dy, outputs + pad, offset), out=out)
        assert got is out
        within(got, want, rounded(want, tokens * SUM * top, F32), "dweight")
        left = torch.ones_like(memory, dtype=torch.bool)
        left[1:].as_strided((inputs, outputs), (outputs + 3, 1)).fill_(False)
        assert bool((memory[left] == 7.0).all())
        total = out.clone()
        ops.weight_gradient(placed(x, inputs + pad, offset), placed(dy, outputs + pad, offset), add=out, out=out)
        within(out, 2 * total.cpu().double(), 4 * half(2 * total.cpu().abs(), F32) + tokens * SUM * top, "dweight onto itself")


def test_no_tokens_and_the_same_bits():
    x, dy = torch.empty(0, 40, dtype=F16, device="cuda"), torch.empty(0, 24, dtype=F16, device="cuda")
    assert not bool(ops.weight_gradient(x, dy).any())
    more = rand((40, 24), 6).cuda()
    assert torch.equal(ops.weight_gradient(x, dy, add=more), more)
    x, dy = rand((3000, 128), 7, BF16).cuda(), rand((3000, 64), 8, BF16).cuda()
    once = ops.weight_gradient(x, dy)
    for _ in range(3):
        assert torch.equal(ops.weight_gradient(x, dy), once)


def test_what_is_not_finite_stays_in_its_row_and_column():
    x, dy = rand((90, 64), 9, F16), rand((90, 136), 10, F16)
    x[5, 3], dy[70, 130] = float("nan"), float("inf")
    got = ops.weight_gradient(x.cuda(), dy.cuda()).cpu()
    fine = torch.isfinite(got)
    assert not fine[3].any() and not fine[:, 130].any()
    fine[3], fine[:, 130] = True, True
    assert fine.all()


def test_graph():
    x, dy = rand((2500, 136), 11, BF16).cuda(), rand((2500, 72), 12, BF16).cuda()
    ops.weight_gradient(x, dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.weight_gradient(x, dy)
    for replay in range(3):
        x.copy_(rand((2500, 136), 13 + replay, BF16))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.weight_gradient(x, dy))
