"""The norm in the place of its input, with the 8-bit checkpoint of that input: one launch and two, rows on and off 16 bytes.

The checkpoint is compared bit for bit with that of the input as it was before the call; the bounds of the norm are those of
``test_gpu_training.py``."""

import pytest
import torch

from oracle import training as ref
from tests.test_gpu_training import BF16, F16, F32, check_forward, placed, rand
from tileccl_amd import ops

pytestmark = pytest.mark.gpu

# columns, pitch, first element: whole vectors; ends inside a vector; off 16 bytes; more columns than one launch holds, of either kind
ROWS = [(256, 256, 0), (300, 300, 0), (1003, 1003, 0), (256, 259, 1), (256, 264, 3), (5, 5, 0), (8192, 8192, 0), (8200, 8200, 0), (16390, 16390, 0)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("place", ["x", "x with a residual", "residual"])
@pytest.mark.parametrize("cols, pitch, offset", ROWS)
def test_checkpoint_of_an_input_that_is_overwritten(lib, cols, pitch, offset, place, dtype):
    x, w, b = rand((21, cols), 1, dtype, 2.0, 0.5), rand((cols,), 3, dtype, 0.2, 1.0), rand((cols,), 4, dtype, 0.3)
    more = None if place == "x" else rand((21, cols), 2, dtype)
    s = x if more is None else (x.float() + more.float()).to(dtype)
    a, m = placed(x, pitch, offset), None if more is None else placed(more, pitch, offset)
    r = ops.layer_norm(a, w.cuda(), b.cuda(), residual=m, checkpoint=True, out=m if place == "residual" else a)
    assert torch.equal(ops.restore_activation(r.checkpoint).cpu().double(), ref.held(s)), "not the checkpoint of the norm's input"
    assert more is None or torch.equal(r.summed.cpu(), s)
    check_forward(r, s, w, b)


@pytest.mark.parametrize("rows", [64, 61])
def test_weight_gradient_in_the_gradients_place_is_refused(lib, rows):
    """As many inputs as tokens: the result has the gradient's shape, and other tiles still read what one has written."""
    grad = rand((rows, 72), 1, BF16).cuda()
    held = ops.checkpoint_activation(rand((rows, rows), 2, BF16).cuda())
    with pytest.raises(ValueError, match="out overlaps grad"):
        ops.weight_gradient(held, grad, out=grad)


def test_results_across_other_operands(lib):
    """Every operand has a place in one allocation.  Results that begin in it, end in it or have one row there are refused before
    anything is written; right in front of it, right behind it and with rows on either side they are what they are elsewhere."""
    rows, cols = 24, 64
    g, a = rand((rows, cols), 1, BF16).cuda(), rand((rows, cols), 2, BF16).cuda()
    memory, places = torch.zeros(2 << 20, dtype=torch.uint8, device="cuda"), iter(range(1 << 20, 2 << 20, 1 << 14))

    def put(t):
        place = memory[next(places):][: t.numel() * t.element_size()]
        place.copy_(t.contiguous().view(-1).view(torch.uint8))
        return place.view(t.dtype).view(t.shape)

    w, mean, rstd = put(rand((cols,), 3, F32, 0.2, 1.0).cuda()), put(rand((rows,), 4).cuda()), put(rand((rows,), 5, F32, 0.1, 1.0).cuda())
    h = ops.checkpoint_activation(a)
    held = ops.ActivationCheckpoint(put(h.values), put(h.scales), rows, cols, BF16)
    before = memory.clone()
    eight_bits = {"the checkpoint's values": held.values, "the checkpoint's scales": held.scales}
    statistics = {"mean": mean, "rstd": rstd, "weight": w}
    calls = [
        (rows, {"weight": w}, lambda out: ops.layer_norm(a, w, out=out).out),
        (rows, {"bias": w}, lambda out: ops.layer_norm(a, bias=w, out=out).out),
        (rows, statistics, lambda out: ops.layer_norm_backward(g, a, mean, rstd, w, out=out).x),
        (rows, statistics | eight_bits, lambda out: ops.layer_norm_backward(g, held, mean, rstd, w, out=out).x),
        (rows, eight_bits, lambda out: ops.restore_activation(held, out=out)),
        (cols, eight_bits, lambda out: ops.weight_gradient(held, g, out_dtype=BF16, out=out)),
    ]
    for out_rows, operands, call in calls:
        def at(first, pitch=cols):
            return memory[first:first // 2 * 2 + 2 * ((out_rows - 1) * pitch + cols)].view(BF16).as_strided((out_rows, cols), (pitch, 1))

        want = call(None)
        for name, t in operands.items():
            first, behind, size = t.data_ptr() - memory.data_ptr(), t.data_ptr() - memory.data_ptr() + t.numel() * t.element_size(), out_rows * cols * 2
            for out in (at(first), at(behind - 16), at(first + 16 - size), at(first - 3 * 8192, 4096)):
                with pytest.raises(ValueError, match=f"out overlaps ({'|'.join(operands)})"):
                    call(out)
            assert torch.equal(memory, before), "a refused call has written"
            for out in (at(first - size), at(behind), at(first + 4096 - 3 * 8192, 4096)):
                assert torch.equal(call(out), want), name
                memory.copy_(before)
