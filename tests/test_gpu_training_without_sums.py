"""The norm's backward pass without the gradients of weight and bias: the same dx, and nothing stored for sums that nobody reads."""

import ctypes as C

import pytest
import torch

from oracle import training as ref
from tests.test_gpu_training import BF16, E, F16, F32, rand
from tileccl_amd import _lib, ops

pytestmark = pytest.mark.gpu

CODES = {F16: _lib.F16, BF16: _lib.BF16, F32: _lib.F32}


# few rows and many, from 8 bits and in full, several groups in a workgroup, ends inside a vector, under eight columns
@pytest.mark.parametrize("rows, cols, dtype, held", [(40, 300, BF16, False), (1000, 512, F16, True), (1000, 5, BF16, False), (1500, 264, BF16, True), (3000, 1003, F32, False),
                                                     (1100, 8200, F16, False), (1030, 16400, F32, False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_the_workspace_stays_as_it_is(lib, rows, cols, dtype, held, in_place):
    s, dy, w = rand((rows, cols), 1, dtype, 2.0, 0.5).cuda(), rand((rows, cols), 2, dtype, 0.1).cuda(), rand((cols,), 3, dtype, 0.2, 1.0).cuda()
    _, mean, rstd = ref.layer_norm(s.cpu())
    mean, rstd = mean.float().cuda(), rstd.float().cuda()
    x = ops.checkpoint_activation(s) if held else s
    want = ops.layer_norm_backward(dy.clone(), x, mean, rstd, w, affine=True)
    assert torch.equal(ops.layer_norm_backward(dy.clone(), x, mean, rstd, w, affine=False).x, want.x)
    size = lib.tccl_layer_norm_grad_workspace(rows, cols, CODES[dtype], int(held))
    workspace = torch.full((size // 4,), 7.0, device="cuda")
    g = dy.clone()
    dx = g if in_place else torch.empty_like(g)
    sums = torch.empty(2, cols, device="cuda")
    p = torch.Tensor.data_ptr
    d = _lib.NormGradDesc(grad=p(g), dx=p(dx), mean=p(mean), rstd=p(rstd), weight=p(w), workspace=p(workspace), workspace_bytes=size, ld_grad=cols, ld_x=cols, ld_dx=cols,
                          rows=rows, cols=cols, dtype=CODES[dtype], affine_dtype=CODES[dtype], **({"values": p(x.values), "scales": p(x.scales)} if held else {"x": p(x)}))
    assert lib.tccl_layer_norm_grad(C.byref(d), None) == 0
    torch.cuda.synchronize()
    assert torch.equal(dx, want.x) and bool((workspace == 7.0).all()), "partial sums were stored"
    g.copy_(dy)
    d.dbias = p(sums[1])  # one of the two
    assert lib.tccl_layer_norm_grad(C.byref(d), None) == 0
    torch.cuda.synchronize()
    # In another order where dx takes grad's place: either sum is off by E of the sum of magnitudes at most.
    assert torch.equal(dx, want.x) and bool(((sums[1] - want.bias).abs() <= 2 * E * dy.float().abs().sum(0)).all())
