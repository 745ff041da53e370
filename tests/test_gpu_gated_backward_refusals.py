"""What ``gated_linear_backward`` refuses of a call that wants the weight's gradient: ahead of the first launch, which may write ``inner`` where the
kept projections are."""

import pytest
import torch

from tests.layer_bounds import BF16, F16, F32
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


def zeros(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def held_from(dtype):
    return ops.checkpoint_activation(zeros(4, 16, dtype=dtype))


def off_vectors():
    """A checkpoint whose values do not start on 16 bytes."""
    held = held_from(BF16)
    memory = torch.zeros(held.values.numel() + 8, dtype=torch.uint8, device="cuda")
    return held._replace(values=memory[8:].view(held.values.shape))


REFUSED = {
    "type of the result": (lambda: dict(out_dtype=F16), "float32 or torch.bfloat16"),
    "type of what is added": (lambda: dict(add=zeros(16, 16, dtype=F16)), "float32 or torch.bfloat16"),
    "layout of what is added": (lambda: dict(add=zeros(16, 16, dtype=F32).t()), "add must"),
    "rows of what is added": (lambda: dict(add=zeros(1, 16, dtype=F32).expand(16, 16)), "add"),
    "place of what is added": (lambda: dict(add=torch.zeros(16, 16)), "add must reside"),
    "what is added is no tensor": (lambda: dict(add=[0.0]), "add must be a 2-D tensor"),
    "type of x": (lambda: dict(x=zeros(4, 16, dtype=F16)), "x must have dtype"),
    "rows of x": (lambda: dict(x=zeros(16, 4).t()), "x must have contiguous rows"),
    "place of x": (lambda: dict(x=torch.zeros(4, 16, dtype=BF16)), "x must reside"),
    "pitch of x": (lambda: dict(x=torch.empty(3 * ((1 << 24) + 8) + 16, dtype=BF16, device="cuda").as_strided((4, 16), ((1 << 24) + 8, 1))), "x has 16 columns .*at most"),
    "type that x was held from": (lambda: dict(x=held_from(F16)), "the checkpoint is of torch.float16"),
    "values of x off 16 bytes": (lambda: dict(x=off_vectors()), "16 bytes"),
}


@pytest.mark.parametrize("which", REFUSED)
def test_kept_outlives_a_refused_call(which):
    make, text = REFUSED[which]
    grad, kept, w = zeros(4, 8), torch.ones(4, 16, dtype=BF16, device="cuda"), zeros(16, 16)
    args = dict(x=zeros(4, 16)) | make()
    with pytest.raises(ValueError, match="gated_linear_backward: .*" + text):
        ops.gated_linear_backward(grad, kept, args.pop("x"), w, out=kept, **args)
    assert bool((kept == 1).all()), "kept was written by a refused call"


def test_what_is_added_lies_as_the_weight():
    grad, kept, x, w = zeros(4, 8), torch.ones(4, 16, dtype=BF16, device="cuda"), zeros(4, 16), zeros(16, 16).t()
    add = zeros(16, 16, dtype=F32)
    add[0, 1] = 1.0
    with pytest.raises(ValueError, match="gated_linear_backward: .*add must"):
        ops.gated_linear_backward(grad, kept, x, w, out=kept, add=add)
    assert bool((kept == 1).all())
    assert torch.equal(ops.gated_linear_backward(grad, kept, x, w, out=kept, add=add.t()).weight, add.t())


def test_a_pitch_that_the_weight_gradient_does_not_take():
    rows, pitch = 4, (1 << 24) + 8
    kept = torch.zeros(3 * pitch + 16, dtype=BF16, device="cuda").as_strided((rows, 16), (pitch, 1))
    kept.fill_(1.0)
    for x in (zeros(rows, 16), held_from(BF16)):
        with pytest.raises(ValueError, match="out has a pitch"):
            ops.gated_linear_backward(zeros(rows, 8), kept, x, zeros(16, 16), out=kept)
    assert bool((kept == 1).all())
    ops.gated_linear_backward(zeros(rows, 8), kept, None, zeros(16, 16), out=kept, inputs=False, weights=False)
    assert not bool(kept.any())


def across_x():
    x = torch.ones(4, 16, dtype=BF16, device="cuda")
    return dict(x=x, out=x), x


def across_values():
    held = held_from(BF16)
    return dict(x=held, out=held.values.view(-1)[64:192].view(BF16).view(4, 16)), held.values


def across_scales():
    memory = torch.full((256,), 127, dtype=torch.uint8, device="cuda")
    return dict(x=held_from(BF16)._replace(scales=memory[96:112].view(1, 16)), out=memory[:128].view(BF16).view(4, 16)), memory


def across_add():
    add = torch.ones(16, 16, device="cuda")
    return dict(x=zeros(4, 16), add=add, out=add.view(-1)[64:96].view(BF16).view(4, 16)), add


@pytest.mark.parametrize("make, name", [(across_x, "x"), (across_values, "the checkpoint's values"), (across_scales, "the checkpoint's scales"), (across_add, "add")])
def test_inner_across_what_the_weight_gradient_reads(make, name):
    args, memory = make()
    before = memory.clone()
    with pytest.raises(ValueError, match="gated_linear_backward: out overlaps " + name):
        ops.gated_linear_backward(zeros(4, 8), zeros(4, 16), args.pop("x"), zeros(16, 16), **args)
    assert torch.equal(memory, before)


@pytest.mark.parametrize("rows", [1, 4])
def test_inner_beside_what_the_weight_gradient_reads(rows):
    """Rows of one buffer: x, then kept, in whose place inner goes; and x's place where x has no part."""
    memory = torch.randn(rows, 32, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    x, kept, grad = memory[:, :16], memory[:, 16:], torch.randn(rows, 8, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    w = torch.randn(16, 16, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    want = ops.gated_linear_backward(grad, kept.clone(), x.clone(), w)
    before = memory.clone()
    got = ops.gated_linear_backward(grad, kept, x, w, out=kept)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(x, before[:, :16])
    elsewhere = ops.gated_linear_backward(grad, before[:, 16:].clone(), x, w, out=x, weights=False)
    assert torch.equal(elsewhere.inner, want.inner) and torch.equal(elsewhere.x, want.x)
