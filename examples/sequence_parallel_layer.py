"""A sequence-parallel layer, forward and backward: layer norm, all-gather, column-parallel linear layer, reduce-scatter.

Between the calls every rank has its own tokens.  Forward: ``s = x + residual`` and its norm on the rank's rows, the norms
gathered, ``Z = Y @ W`` with each rank's columns of ``W``.  Backward, from the gradient of ``Z``: the gradient of the rank's
weight columns, ``dY = dZ @ W.t()`` summed over the ranks and scattered by rows, the norm's gradients on the rank's rows, and
the sums for its weight and bias over all ranks.  What is kept in between is in 8 bits: ``s`` on its rank, ``Y`` on every rank.

    python examples/sequence_parallel_layer.py [--tokens 8192] [--hidden 4096] [--outputs 4096] [--world 2] [--steps 20]

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


class SequenceParallelLayer:
    """``ctxs``: one context per rank; ``weight``: hidden x outputs; ``gamma``, ``beta``: the norm's.  Every rank has a multiple
    of 128 tokens (the reduce-scatter's shards) and of 8 columns."""

    def __init__(self, ctxs, tokens: int, weight: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor) -> None:
        hidden, outputs = weight.shape
        world = len(ctxs)
        if tokens % (128 * world) or outputs % (8 * world):
            raise ValueError(f"{tokens} tokens and {outputs} outputs over {world} ranks")
        self.ctxs, self.gamma, self.beta = ctxs, gamma, beta
        self.heaps = [c.heap for c in ctxs]
        self.columns = [slice(r * outputs // world, (r + 1) * outputs // world) for r in range(world)]
        zeros = lambda *shape, dtype=DTYPE: [c.zeros(*shape, dtype=dtype) for c in ctxs]  # noqa: E731
        self.weight = zeros(hidden, outputs // world)
        for w, cols in zip(self.weight, self.columns):
            w.copy_(weight[:, cols])
        self.norms, self.gathered, self.z = zeros(tokens // world, hidden), zeros(tokens, hidden), zeros(tokens, outputs)
        # The last rank to call finds every rank's product there and makes all ranks' sums.
        self.scatter_heaps = SymmetricHeap.create_all(4 * tokens * hidden + (16 << 20), world)
        self.scatter = [FusedGemmReduceScatter(h, tokens, hidden, partial_dtype=DTYPE, out_dtype=DTYPE, emulate_peer=h.rank == world - 1)
                        for h in self.scatter_heaps]
        self.sums = zeros(2, hidden, dtype=torch.float32)
        self.weight_grad = [torch.zeros(hidden, outputs // world, device=w.device) for w in self.weight]  # summed over the steps

    def forward(self, xs, residuals):
        """Z on every rank, the summed inputs, and what ``backward`` wants."""
        normed = [ops.layer_norm(x, self.gamma, self.beta, residual=r, checkpoint=True, out=out)
                  for x, r, out in zip(xs, residuals, self.norms)]
        allgather_staged(self.norms, self.gathered, self.heaps)
        held = [ops.checkpoint_activation(y) for y in self.gathered]
        for ctx, y, w, z in zip(self.ctxs, self.gathered, self.weight, self.z):
            ops.gemm_allgather(y, w, z, ctx=ctx, variant="s0")
        return self.z, [n.summed for n in normed], [(n.checkpoint, n.mean, n.rstd, y) for n, y in zip(normed, held)]

    def backward(self, grad_z, grad_summed, kept):
        """The gradient of every rank's ``x`` (and residual), and of gamma and beta; the weight's is added to ``weight_grad``."""
        mine = [g[:, cols] for g, cols in zip(grad_z, self.columns)]
        for op, g, w in zip(self.scatter, mine, self.weight):
            op(g, w.t(), "s0")
        for g, (_, _, _, y), into in zip(mine, kept, self.weight_grad):
            ops.weight_gradient(y, g, add=into, out=into)
        grads = [ops.layer_norm_backward(op.out, s, mean, rstd, self.gamma, grad_summed=g)
                 for op, (s, mean, rstd, _), g in zip(self.scatter, kept, grad_summed)]
        for sums, g in zip(self.sums, grads):
            sums[0].copy_(g.weight)
            sums[1].copy_(g.bias)
        allreduce_staged(self.sums, self.heaps)
        return [g.x for g in grads], self.sums[0][0], self.sums[0][1]

    def close(self) -> None:
        for h in self.scatter_heaps:
            h.cleanup()


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--tokens", type=int, default=8192)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--outputs", type=int, default=4096)
    p.add_argument("--world", type=int, default=2)
    p.add_argument("--steps", type=int, default=20)
    a = p.parse_args()
    heap = 2 * (2 * a.tokens * a.hidden + a.tokens * a.outputs + a.hidden * a.outputs) + (64 << 20)
    ctxs = tileccl.init_local(world_size=a.world, heap_size=heap)
    rand = lambda *shape: torch.randn(*shape, device="cuda").to(DTYPE)  # noqa: E731
    rows = a.tokens // a.world
    layer = SequenceParallelLayer(ctxs, a.tokens, rand(a.hidden, a.outputs) * a.hidden**-0.5, 1 + 0.1 * rand(a.hidden), 0.1 * rand(a.hidden))
    xs, residuals = [rand(rows, a.hidden) for _ in ctxs], [rand(rows, a.hidden) for _ in ctxs]
    grad_z, grad_s = [rand(a.tokens, a.outputs) for _ in ctxs], [rand(rows, a.hidden) for _ in ctxs]
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for step in range(a.steps + 3):
        if step == 3:
            start.record()
        _, _, kept = layer.forward(xs, residuals)
        layer.backward(grad_z, grad_s, kept)
    end.record()
    torch.cuda.synchronize()
    held = sum(c.values.nbytes + c.scales.nbytes for k in kept for c in (k[0], k[3]))
    print(f"{a.world} ranks in turn, {a.tokens} x {a.hidden} x {a.outputs}: {start.elapsed_time(end) / max(a.steps, 1):.3f} ms a step, "
          f"{held / 2**20:.0f} MiB kept for the backward pass ({2 * a.hidden * (a.tokens + a.world * a.tokens) / 2**20:.0f} MiB in 16 bits)")
    layer.close()
    for c in ctxs:
        c.heap.cleanup()


if __name__ == "__main__":
    main()
