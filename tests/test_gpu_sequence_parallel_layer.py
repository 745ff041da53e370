"""The example's layer against autograd in 64 bits: two and three ranks, two micro-batches, sizes that no tile divides."""

import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import training as ref

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parent.parent / "examples" / "sequence_parallel_layer.py"


def example():
    spec = importlib.util.spec_from_file_location("sequence_parallel_layer", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


@pytest.mark.parametrize("world, tokens, hidden, outputs", [(2, 256, 256, 256), (2, 768, 264, 272), (3, 1536, 512, 384)])
def test_layer_forward_and_backward(lib, world, tokens, hidden, outputs):
    """Against exact gradients.  Rounded to bf16 (each value off by 2^-9 of itself): x's sum, the norm, Z; dZ's product before and after
    its sum, dx.  Held in 8 bits (2^-4): what the gradients of W and gamma multiply, and the projection in dx; errors of neighbours
    are independent, so that they cannot take a sum's norm further off than each value is.  beta's gradient has bf16's only."""
    module = example()
    bf = torch.bfloat16
    g = torch.Generator().manual_seed(1)
    rand = lambda *shape: torch.randn(*shape, generator=g).to(bf)  # noqa: E731
    rows = tokens // world
    weight, gamma, beta = (rand(hidden, outputs).float() * hidden**-0.5).to(bf), 1 + 0.25 * rand(hidden), 0.25 * rand(hidden)
    batches = [[rand(tokens, n) for n in (hidden, hidden, outputs, hidden)] for _ in range(2)]
    cut = lambda t: [part.contiguous().cuda() for part in t.split(rows)]  # noqa: E731
    ctxs = module.tileccl.init_local(world_size=world, heap_size=64 << 20)
    try:
        layer = module.SequenceParallelLayer(ctxs, tokens, weight.cuda(), gamma.cuda(), beta.cuda())
        w = weight.double().requires_grad_()
        for x, residual, dz, ds in batches:
            zs, summed, kept = layer.forward(cut(x), cut(residual))
            dxs, dgamma, dbeta = layer.backward([dz.cuda()] * world, cut(ds), kept)
            s = (x.float() + residual.float()).to(bf)
            assert torch.equal(torch.cat(summed).cpu(), s)
            leaf, a, b = (t.double().requires_grad_() for t in (s, gamma, beta))
            z = torch.nn.functional.layer_norm(leaf, (hidden,), a, b) @ w
            z.backward(dz.double())
            for r in range(world):
                assert off(zs[r], z.detach()) < 3 * 2.0**-9
            assert off(torch.cat(dxs), leaf.grad + ds.double()) < 2.0**-4 + 4 * 2.0**-9
            assert off(dgamma, a.grad) < 2.0**-4 + 3 * 2.0**-9
            assert off(dbeta, b.grad) < 3 * 2.0**-9
        assert off(torch.cat(layer.weight_grad, 1), w.grad) < 2.0**-4 + 3 * 2.0**-9
        held = kept[0][3]
        y = layer.gathered[0].cpu()
        assert torch.equal(module.ops.restore_activation(held).cpu().double(), ref.held(y)), "what is kept of Y is not Y in 8 bits"
        layer.close()
    finally:
        for c in ctxs:
            c.heap.cleanup()


def test_refuses_what_does_not_divide():
    with pytest.raises(ValueError, match="over 2 ranks"):
        example().SequenceParallelLayer([None, None], 192, torch.zeros(8, 16), None, None)
