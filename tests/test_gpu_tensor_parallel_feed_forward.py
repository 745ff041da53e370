"""The example's feed-forward layer against autograd and AdamW in 64 bits: gated projections, weight gradients from inputs in full and the
update, run together over two and three ranks, with sizes that no tile divides."""

import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import layers as ref
from tests.layer_bounds import BF16, F32

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parent.parent / "examples" / "tensor_parallel_feed_forward.py"
HOW = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def example():
    spec = importlib.util.spec_from_file_location("tensor_parallel_feed_forward", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


ROUNDING = 2.0**-8  # of a value in bf16, at most


@pytest.mark.parametrize("world, tokens, hidden, outputs, recompute, bits",
                         [(2, 256, 256, 256, False, 8), (2, 768, 264, 272, True, 32), (3, 1536, 512, 408, False, 32), (2, 512, 1096, 1040, True, 8)])
def test_layer_learns_as_the_formulas_do(lib, world, tokens, hidden, outputs, recompute, bits):
    """Roundings on the way, each at most 2^-8 of its value, and an error of g or u reaches h and inner at most 1.2 times as large; those of
    neighbours are independent, so a product's norm is off by no more than its operands are.
    Result: the norm (with g and u, 2.4), h, partial sums, their sum: at most 6.  D's gradient: h's 4.  inner: dh, the norm in u and slope
    (2.4), z as kept in both (2.4), its own: 7; W's gradient: the norm's, too, 8.  dx: inner's, the partial sums, their sum, its own: 10, as
    the norm's own gradients without the last.  A second batch follows an update: the weights that it starts from are the layer's own.
    Update: p is good to 4 roundings of 2^-24 of it, and a step, at most 10 lr where b1 is 0.9 and b2 0.99, to 30 of its own."""
    module = example()
    g = torch.Generator().manual_seed(1)
    rand = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    rows, part = tokens // world, outputs // world
    gate, up = ((rand(hidden, outputs) * hidden**-0.5).to(BF16) for _ in range(2))
    down, gamma, beta = (rand(outputs, hidden) * outputs**-0.5).to(BF16), (1 + 0.25 * rand(hidden)).to(BF16), (0.25 * rand(hidden)).to(BF16)
    cut = lambda t: [p.contiguous().cuda() for p in t.split(rows)]  # noqa: E731
    ctxs = module.tileccl.init_local(world_size=world, heap_size=64 << 20)
    try:
        layer = module.FeedForward(ctxs, tokens, *(t.cuda() for t in (gate, up, down, gamma, beta)), recompute=recompute, bits=bits)
        for step in (1, 2):
            held = [[w.cpu() for w in ws] for ws in layer.weights]
            leaves = [torch.cat([ws[0][:, :part] for ws in held], 1), torch.cat([ws[0][:, part:] for ws in held], 1), torch.cat([ws[1] for ws in held]), held[0][2], held[0][3]]
            assert step > 1 or all(torch.equal(a, b) for a, b in zip(leaves, (gate, up, down, gamma, beta)))
            x, dy = rand(tokens, hidden).to(BF16), rand(tokens, hidden).to(BF16)
            results, kept = layer.forward(cut(x))
            inner_sums = torch.cat([op.out for op in layer.scatter]).cpu()
            dxs, grads = layer.backward(cut(dy), kept)
            leaf, wg, wu, d, a, b = (t.double().requires_grad_() for t in (x, *leaves))
            y = torch.nn.functional.layer_norm(leaf, (hidden,), a, b)
            out = (ref.activation(y @ wg, "silu")[0] * (y @ wu)) @ d
            (leaf + out).backward(dy.double())
            assert off(inner_sums, out.detach()) < 6 * ROUNDING
            assert torch.equal(torch.cat(results).cpu(), (x.float() + inner_sums.float()).to(BF16))
            assert off(torch.cat(dxs), leaf.grad) < 10 * ROUNDING
            for r, (dw, dd, dgamma, dbeta) in enumerate(grads):
                cols = slice(r * part, (r + 1) * part)
                assert dw.dtype == dd.dtype == F32
                assert off(dw, torch.cat([wg.grad[:, cols], wu.grad[:, cols]], 1)) < 8 * ROUNDING
                assert off(dd, d.grad[cols]) < 4 * ROUNDING
                assert off(dgamma, a.grad) < 9 * ROUNDING and off(dbeta, b.grad) < 9 * ROUNDING
            before = [(s.master.cpu().double(), *(m.cpu().double() for m in module.ops.adamw_moments(s))) for s in layer.states]
            layer.update(grads, step, **HOW)
            for ws, gs, state, (p, m, v) in zip(layer.weights, grads, layer.states, before):
                at = module.ops.AdamWState.offsets(state.sizes)
                for w, g_, start, n in zip(ws, gs, at, state.sizes):
                    want, _, _ = ref.adamw(p[start : start + n], g_.cpu().reshape(-1), m[start : start + n], v[start : start + n], step=step, grad_scale=1.0, **HOW)
                    got = state.master[start : start + n].cpu()
                    assert float((got - want).abs().max()) <= 2.0**-22 * float(p[start : start + n].abs().max()) + 2.0**-19 * 10 * HOW["lr"]
                    assert torch.equal(w.reshape(-1).cpu(), got.to(BF16)), "weights are the master copy's rounded values"
            assert all(torch.equal(a, b) for ws in layer.weights[1:] for a, b in zip(ws[2:], layer.weights[0][2:])), "every rank has the same norm"
        layer.close()
    finally:
        for c in ctxs:
            c.heap.cleanup()


def test_refuses_what_does_not_divide():
    with pytest.raises(ValueError, match="over 2 ranks"):
        example().FeedForward([None, None], 256, torch.zeros(8, 24), None, None, None, None)
