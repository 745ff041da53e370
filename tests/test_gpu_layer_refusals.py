"""What the gated layer, weight gradients from an input in full and AdamW refuse of tensors on the GPU, before anything is launched."""

import pytest
import torch

from tests.layer_bounds import BF16, F16, F32
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


def zeros(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def test_gated_linear():
    x, w = zeros(4, 16), zeros(16, 16)
    refusals = [
        (dict(x=zeros(4, 8)), "x has 8 columns, weight 16 rows"),
        (dict(x=zeros(4, 16, dtype=F16)), "x must"),
        (dict(x=x.cpu()), "x must"),
        (dict(x=zeros(16, 4).t()), "x"),
        (dict(x=zeros(1, 16).expand(4, 16)), "x"),
        (dict(x=zeros(16)), "x must be a 2-D tensor"),
        (dict(weight=zeros(16, 15)), r"weight must be \(inputs, 2 \* outputs\)"),
        (dict(weight=zeros(16, 16, dtype=F32)), "float16 or bfloat16"),
        (dict(weight=zeros(16, 32)[:, ::2]), "contiguous rows"),
        (dict(weight=zeros(16, 1).expand(16, 16)), "contiguous rows"),
        (dict(out=zeros(4, 16)), "out must have shape"),
        (dict(out=zeros(4, 8, dtype=F16)), "out must"),
        (dict(out=x[:, :8]), "out overlaps x"),
        (dict(out=w[:4, :8]), "out overlaps weight"),
    ]
    for change, text in refusals:
        with pytest.raises(ValueError, match="gated_linear: .*" + text):
            args = dict(x=x, weight=w) | change
            ops.gated_linear(args.pop("x"), args.pop("weight"), **args)


def test_gated_linear_backward():
    grad, kept, x, w = zeros(4, 8), torch.ones(4, 16, dtype=BF16, device="cuda"), zeros(4, 16), zeros(16, 16)
    held = ops.checkpoint_activation(x)
    refusals = [
        (dict(grad=zeros(4, 16)), "grad has 16 columns, weight is for 8 outputs"),
        (dict(grad=zeros(4, 8, dtype=F16)), "grad must"),
        (dict(kept=zeros(4, 8)), "kept must have shape"),
        (dict(kept=zeros(3, 16)), "kept must have shape"),
        (dict(x=zeros(4, 24)), "x has 24 columns, weight 16 rows"),
        (dict(x=zeros(5, 16)), "x has 5 rows, grad 4"),
        (dict(x=ops.checkpoint_activation(zeros(4, 24))), "x has 24 columns, weight 16 rows"),
        (dict(x=None), "wants x"),
        (dict(kept=None, x=held), "not from a checkpoint"),
        (dict(kept=None, x=zeros(4, 24), weights=False), "x must have shape"),
        (dict(add=zeros(16, 8, dtype=F32)), "add must have shape"),
        (dict(out=grad), "out must have shape"),
        (dict(out=torch.empty(64, dtype=BF16, device="cuda")[:64].view(4, 16)[:, ::2]), "out"),
        (dict(kept=None, out=x), "out overlaps x"),
        (dict(out=w[:4]), "out overlaps weight"),
    ]
    for change, text in refusals:
        with pytest.raises(ValueError, match="gated_linear_backward: .*" + text):
            args = dict(grad=grad, kept=kept, x=x, weight=w) | change
            ops.gated_linear_backward(args.pop("grad"), args.pop("kept"), args.pop("x"), args.pop("weight"), **args)
    with pytest.raises(ValueError, match="x has 24 columns"):
        ops.gated_linear_backward(grad, kept, zeros(4, 24), w, out=kept)
    assert bool((kept == 1).all()), "kept was written by a refused call"
    memory = zeros(40)
    with pytest.raises(ValueError, match="out"):  # beside kept by a few elements
        ops.gated_linear_backward(zeros(2, 8), memory[:32].view(2, 16), None, w, out=memory[4:36].view(2, 16), weights=False, inputs=False)


def test_weight_gradient():
    x, grad = zeros(6, 16), zeros(6, 8)
    refusals = [
        (dict(grad=zeros(5, 8)), "rows"),
        (dict(grad=zeros(6, 8, dtype=F16)), "grad"),
        (dict(x=x.cpu()), "x"),
        (dict(x=zeros(16, 6).t()), "x"),
        (dict(out_dtype=F16), "float32 or torch.bfloat16"),
        (dict(out=zeros(8, 16, dtype=F32)), "out must have shape"),
        (dict(add=zeros(8, 16, dtype=F32)), "add must have shape"),
        (dict(layout="nk", add=zeros(16, 8, dtype=F32)), "add must have shape"),
        (dict(layout="mn"), "layout must be"),
    ]
    for change, text in refusals:
        args = dict(x=x, grad=grad) | change
        with pytest.raises(ValueError, match="weight_gradient: .*" + text):
            ops.weight_gradient(args.pop("x"), args.pop("grad"), **args)
    memory = zeros(8, 16)
    for args in ((memory[:, :8], zeros(8, 8)), (zeros(8, 8), memory[:, 8:])):
        with pytest.raises(ValueError, match="out overlaps (x|grad)"):
            ops.weight_gradient(*args, out=memory.view(-1)[:64].view(8, 8))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(bits):
    p, g = [zeros(130), zeros(4, 8)], [zeros(130), zeros(4, 8)]
    state = ops.AdamWState.zeros(p, bits=bits, master=True)
    word = zeros(1, dtype=torch.int32)
    refusals = [
        (dict(grads=[g[0], zeros(8, 4)]), r"grads\[1\] must have shape"),
        (dict(grads=[g[0], g[1].float()]), "grads must all be"),
        (dict(grads=[t.half() for t in g]), "grads must all be"),
        (dict(params=[p[0], zeros(8, 4).t()]), r"params\[1\] must be contiguous"),
        (dict(params=[p[0], p[1].float()], grads=[g[0], g[1]]), "params must share"),
        (dict(params=[zeros(131), p[1]], grads=[zeros(131), g[1]]), "the state is for 130 elements"),
        (dict(params=[t.cpu() for t in p]), "must reside on cuda:0"),
        (dict(params=[p[0][:32], p[0][16:48]], grads=[g[0][:32], g[0][:32]], state=ops.AdamWState.zeros([p[0][:32]] * 2, bits=bits)), "share memory"),
        (dict(params=[p[0], p[0]], grads=[g[0], g[0]], state=ops.AdamWState.zeros([p[0]] * 2, bits=bits)), "share memory"),
        (dict(grads=[p[0], g[1]]), "share memory"),
        (dict(state=state._replace(first=state.first[:128])), "first must be"),
        (dict(state=state._replace(second=state.first)), "share memory"),
        (dict(state=state._replace(master=state.master.half())), "master must be"),
        (dict(step=0), "counted from 1"),
        (dict(step=2**31), "counted from 1"),
        (dict(step=2**70), "adamw_step"),
        (dict(step="one"), "adamw_step"),
        (dict(step=word.long()), "step must be"),
        (dict(step=zeros(2, dtype=torch.int32)), "step must be"),
        (dict(lr=word), "lr must be"),
        (dict(lr=state.master[3]), "lr shares memory"),
        (dict(grad_scale=state.master[131:132]), "grad_scale shares memory"),
        (dict(step=state.master[5:6].view(torch.int32)), "step shares memory"),
        (dict(betas=(0.9,)), "betas are two numbers"),
        (dict(betas=(0.9, "b")), "adamw_step"),
        (dict(betas=(0.9, 1.0)), "betas must lie"),
        (dict(eps=-1.0), "eps must not"),
    ]
    if bits == 8:
        refusals.append((dict(state=state._replace(second_scales=None)), "second_scales"))
        refusals.append((dict(state=state._replace(first_scales=state.first_scales[:1])), "first_scales must be"))
        with pytest.raises(ValueError, match="whole blocks"):
            ops.adamw_moments(state._replace(first=state.first[:-16]))
    for change, text in refusals:
        with pytest.raises(ValueError, match=text):
            args = dict(params=p, grads=g, state=state, step=1) | change
            ops.adamw_step(args.pop("params"), args.pop("grads"), args.pop("state"), **args)
    assert not any(bool(t.any()) for t in (*p, state.first, state.second, state.master))
    assert all(t._version == 0 for t in p)
