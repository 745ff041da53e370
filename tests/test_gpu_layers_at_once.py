"""Calls of the gated layer, weight gradients and AdamW on two streams at once, and recorded into graphs that share their memory: workspaces (copies of
operands, sums of splits) are a call's own."""

import pytest
import torch

from tests.layer_bounds import BF16, rand
from tests.test_gpu_gated import weight_of
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


class Layer:
    """One layer's operands, in rows that need copies, with inputs and tokens that are split over workgroups."""

    def __init__(self, seed, layout):
        self.x, self.dh = rand((2500, 1003), seed, BF16).cuda(), rand((2500, 72), seed + 1, BF16).cuda()
        _, self.w = weight_of(1003, 72, BF16, layout, seed + 2)
        self.few, self.few_dh = rand((5, 4104), seed + 3, BF16).cuda(), rand((5, 1032), seed + 4, BF16).cuda()
        _, self.wide = weight_of(4104, 1032, BF16, layout, seed + 5)

    def pass_(self):
        d = ops.gated_linear_backward(self.dh, None, self.x, self.w)
        f = ops.gated_linear(self.few, self.wide, keep=True)
        e = ops.gated_linear_backward(self.few_dh, None, self.few, self.wide, weights=False)
        p, g = (t if t.stride(1) == 1 else t.t() for t in (self.w, d.weight))
        p = p.clone()
        state = ops.AdamWState.zeros([p], bits=8)
        ops.adamw_step([p], [g], state, step=7)
        return [*d, *f, *e[:2], p, *state[:4], *ops.adamw_moments(state)]


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams():
    layers = [Layer(10, "kn"), Layer(30, "nk")]
    want = [[t.clone() for t in layer.pass_()] for layer in layers]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        for s, layer in zip(streams, layers):
            with torch.cuda.stream(s):
                got.append(layer.pass_())
    torch.cuda.synchronize()
    assert all(same(g, want[i % 2]) for i, g in enumerate(got))


def test_graphs_of_one_pool():
    """Recorded one behind the other into one pool, replayed in turn, with eager calls in between."""
    layers = [Layer(50, "nk"), Layer(70, "kn")]
    for layer in layers:
        layer.pass_()
    graphs, kept = [], []
    pool = torch.cuda.graph_pool_handle()
    for layer in layers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            kept.append(layer.pass_())
        graphs.append(graph)
    for replay in range(3):
        for layer, graph, out in zip(layers, graphs, kept):
            layer.x.copy_(rand(tuple(layer.x.shape), 90 + replay, BF16))
            layer.few.copy_(rand(tuple(layer.few.shape), 95 + replay, BF16))
            graph.replay()
            torch.cuda.synchronize()
            assert same(out, layer.pass_()), replay
