"""Layer norm of rows whose mean is far larger than their spread, of rows with a step between wavefronts and of constant rows,
by bounds that are linear in the mean (``norm_bounds.py``); one wavefront to sixteen, one row at a time to eight."""

import pytest
import torch

from oracle import training as ref
from tests import norm_bounds
from tests.test_gpu_training import BF16, F16, F32, rand
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, cols", [(10, 300), (10, 512), (15, 1003), (20, 4096), (2100, 520), (10, 8190), (10, 12000), (10, 20000), (5, 32768)])
def test_means_beside_the_spread(lib, rows, cols, dtype):
    s = norm_bounds.rows_with_means(rows, cols, dtype, 1)
    w, b, dy = rand((cols,), 2, F32, 0.2, 1.0), rand((cols,), 3, F32, 0.3), rand((rows, cols), 4, dtype)
    r = ops.layer_norm(s.cuda(), w.cuda(), b.cuda())
    norm_bounds.forward(r.out, r.mean, r.rstd, s, w, b)
    d = ops.layer_norm_backward(dy.cuda(), s.cuda(), r.mean, r.rstd, w.cuda())
    norm_bounds.backward(d.x, d.weight, d.bias, dy, s, r.mean, r.rstd, w, dtype)
    if dtype == F32:
        return
    r = ops.layer_norm(s.cuda(), w.cuda(), b.cuda(), checkpoint=True)
    norm_bounds.forward(r.out, r.mean, r.rstd, s, w, b)
    d = ops.layer_norm_backward(dy.cuda(), r.checkpoint, r.mean, r.rstd, w.cuda())
    norm_bounds.backward(d.x, d.weight, d.bias, dy, ref.held(s), r.mean, r.rstd, w, dtype)
