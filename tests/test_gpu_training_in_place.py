"""The norm in the place of its input, with the 8-bit checkpoint of that input: one launch and two, rows on and off 16 bytes.

The checkpoint is compared bit for bit with that of the input as it was before the call; the bounds of the norm are those of
``test_gpu_training.py``."""

import pytest
import torch

from oracle import training as ref
from tests.test_gpu_training import BF16, F16, check_forward, placed, rand
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
