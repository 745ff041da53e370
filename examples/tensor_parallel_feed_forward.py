"""A gated feed-forward layer that learns, its columns and rows over the ranks: norm, gated projections, product back, update.

Between the calls every rank has its own tokens.  Forward: the norm of the rank's rows, gathered; ``h = act(Y Wg) * (Y Wu)`` with the rank's
columns of both projections; ``h @ D`` with its rows of ``D``, summed over the ranks and scattered by rows, on top of ``x``.  Backward, from
the gradient of that: ``D``'s, through ``h`` to the projections (kept from the forward pass, or computed again), the weights',
``inner @ W.t()`` summed and scattered, and the norm's.  Then one AdamW call updates all weights of the rank, with moments in 8 or 32 bits.

    python examples/tensor_parallel_feed_forward.py [--tokens 8192] [--hidden 4096] [--outputs 8192] [--world 2] [--bits 8] [--recompute]

Ranks are slices of one GPU's memory and call one after the other.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import tileccl_amd as tileccl  # noqa: E402
from tileccl_amd import ops  # noqa: E402
from tileccl_amd.primitives import allgather_staged, allreduce_staged  # noqa: E402
from tileccl_amd.v2 import FusedGemmReduceScatter, SymmetricHeap  # noqa: E402

DTYPE = torch.bfloat16


class FeedForward:
    """``ctxs``: one context per rank; ``gate``, ``up``: hidden x outputs; ``down``: outputs x hidden; ``gamma``, ``beta``: the norm's.  Every
    rank has a multiple of 128 tokens (the reduce-scatter's shards) and of 8 outputs; hidden is a multiple of 8."""

    def __init__(self, ctxs, tokens: int, gate, up, down, gamma, beta, *, activation: str = "silu", recompute: bool = False, bits: int = 8) -> None:
        hidden, outputs = gate.shape
        world = len(ctxs)
        if tokens % (128 * world) or outputs % (8 * world) or hidden % 8:
            raise ValueError(f"{tokens} tokens, {hidden} x {outputs} weights over {world} ranks")
        self.ctxs, self.activation, self.recompute = ctxs, activation, recompute
        self.heaps = [c.heap for c in ctxs]
        parts = [slice(r * outputs // world, (r + 1) * outputs // world) for r in range(world)]
        self.weights = [[torch.cat([gate[:, p], up[:, p]], 1).contiguous(), down[p].contiguous(), gamma.clone(), beta.clone()] for p in parts]
        self.states = [ops.AdamWState.zeros(w, bits=bits, master=True) for w in self.weights]
        zeros = lambda *shape, dtype=DTYPE: [c.zeros(*shape, dtype=dtype) for c in ctxs]  # noqa: E731
        self.rows, self.gathered = zeros(tokens // world, hidden), zeros(tokens, hidden)
        self.grad_rows, self.grad_gathered = zeros(tokens // world, hidden), zeros(tokens, hidden)
        # The last rank to call finds every rank's product there and makes all ranks' sums.
        self.scatter_heaps = SymmetricHeap.create_all(4 * tokens * hidden + (16 << 20), world)
        self.scatter = [FusedGemmReduceScatter(h, tokens, hidden, partial_dtype=DTYPE, out_dtype=DTYPE, emulate_peer=h.rank == world - 1)
                        for h in self.scatter_heaps]
        self.sums = zeros(2, hidden, dtype=torch.float32)

    def forward(self, xs):
        """Every rank's rows of the result, and what ``backward`` wants."""
        normed = [ops.layer_norm(x, gamma, beta, out=out) for x, (_, _, gamma, beta), out in zip(xs, self.weights, self.rows)]
        allgather_staged(self.rows, self.gathered, self.heaps)
        hs = [ops.gated_linear(y, w, activation=self.activation, keep=not self.recompute) for y, (w, *_) in zip(self.gathered, self.weights)]
        for op, h, (_, down, *_) in zip(self.scatter, hs, self.weights):
            op(h.out, down, "s0")
        return [x + op.out for x, op in zip(xs, self.scatter)], [(x, n.mean, n.rstd, *h) for x, n, h in zip(xs, normed, hs)]

    def backward(self, grads, kept):
        """The gradient of every rank's ``x``, and of its weights, from those of the results."""
        for g, rows in zip(grads, self.grad_rows):
            rows.copy_(g)
        allgather_staged(self.grad_rows, self.grad_gathered, self.heaps)
        inner, weight_grads = [], []
        for dy, y, (_, _, _, h, z), (w, down, *_) in zip(self.grad_gathered, self.gathered, kept, self.weights):
            d = ops.gated_linear_backward(dy @ down.t(), z, y, w, activation=self.activation, inputs=False, out=z)
            inner.append(d.inner)
            weight_grads.append([d.weight, ops.weight_gradient(h, dy)])
        for op, d, (w, *_) in zip(self.scatter, inner, self.weights):
            op(d, w.t(), "s0")
        back = [ops.layer_norm_backward(op.out, x, mean, rstd, gamma, grad_summed=g)
                for op, (x, mean, rstd, _, _), (_, _, gamma, _), g in zip(self.scatter, kept, self.weights, grads)]
        for sums, b in zip(self.sums, back):
            sums[0].copy_(b.weight)
            sums[1].copy_(b.bias)
        allreduce_staged(self.sums, self.heaps)
        return [b.x for b in back], [[*g, s[0], s[1]] for g, s in zip(weight_grads, self.sums)]

    def update(self, weight_grads, step: int, **how) -> None:
        for weights, grads, state in zip(self.weights, weight_grads, self.states):
            ops.adamw_step(weights, grads, state, step=step, **how)

    def close(self) -> None:
        for h in self.scatter_heaps:
            h.cleanup()


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--tokens", type=int, default=8192)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--outputs", type=int, default=8192)
    p.add_argument("--world", type=int, default=2)
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--bits", type=int, default=8, choices=(8, 32))
    p.add_argument("--recompute", action="store_true", help="compute the projections again in the backward pass instead of keeping them")
    a = p.parse_args()
    ctxs = tileccl.init_local(world_size=a.world, heap_size=2 * a.tokens * a.hidden * 4 + (64 << 20))
    rand = lambda *shape: torch.randn(*shape, device="cuda").to(DTYPE)  # noqa: E731
    layer = FeedForward(ctxs, a.tokens, rand(a.hidden, a.outputs) * a.hidden**-0.5, rand(a.hidden, a.outputs) * a.hidden**-0.5,
                        rand(a.outputs, a.hidden) * a.outputs**-0.5, 1 + 0.1 * rand(a.hidden), 0.1 * rand(a.hidden), recompute=a.recompute, bits=a.bits)
    rows = a.tokens // a.world
    xs, grads = [rand(rows, a.hidden) for _ in ctxs], [rand(rows, a.hidden) for _ in ctxs]
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for step in range(a.steps + 3):
        if step == 3:
            start.record()
        _, kept = layer.forward(xs)
        _, weight_grads = layer.backward(grads, kept)
        layer.update(weight_grads, step + 1, lr=1e-4, weight_decay=0.1)
    end.record()
    torch.cuda.synchronize()
    print(f"{a.world} ranks in turn, {a.tokens} x {a.hidden} x {a.outputs}: {start.elapsed_time(end) / max(a.steps, 1):.3f} ms a step, "
          f"optimizer state {sum(s.nbytes for s in layer.states) / 2**20:.0f} MiB")
    layer.close()
    for c in ctxs:
        c.heap.cleanup()


if __name__ == "__main__":
    main()
