"""Views that stand for their memory's values negated (``torch.is_neg``), as a conjugate's imaginary part is one: refused, since the kernels read the memory."""

import pytest
import torch

from tests.layer_bounds import BF16, F32
from tileccl_amd import ops

pytestmark = pytest.mark.gpu


def negated(*shape, dtype=BF16):
    t = torch._neg_view(torch.ones(*shape, dtype=dtype, device="cuda"))
    assert t.is_neg()
    return t


def ones(*shape, dtype=BF16):
    return torch.ones(*shape, dtype=dtype, device="cuda")


CALLS = {
    "gated_linear x": lambda: ops.gated_linear(negated(4, 16), ones(16, 16)),
    "gated_linear weight": lambda: ops.gated_linear(ones(4, 16), negated(16, 16)),
    "gated_linear out": lambda: ops.gated_linear(ones(4, 16), ones(16, 16), out=negated(4, 8)),
    "gated_linear_backward grad": lambda: ops.gated_linear_backward(negated(4, 8), None, ones(4, 16), ones(16, 16)),
    "gated_linear_backward kept": lambda: ops.gated_linear_backward(ones(4, 8), negated(4, 16), ones(4, 16), ones(16, 16)),
    "gated_linear_backward add": lambda: ops.gated_linear_backward(ones(4, 8), None, ones(4, 16), ones(16, 16), add=negated(16, 16, dtype=F32)),
    "weight_gradient x": lambda: ops.weight_gradient(negated(4, 16), ones(4, 8)),
    "weight_gradient grad": lambda: ops.weight_gradient(ops.checkpoint_activation(ones(4, 16)), negated(4, 8)),
    "layer_norm x": lambda: ops.layer_norm(negated(4, 16)),
    "layer_norm weight": lambda: ops.layer_norm(ones(4, 16), negated(16)),
    "checkpoint_activation x": lambda: ops.checkpoint_activation(negated(4, 16)),
}


@pytest.mark.parametrize("which", CALLS)
def test_operators(which):
    op, name = which.split()
    with pytest.raises(ValueError, match=f"{op}: {name} .*negated"):
        CALLS[which]()


@pytest.mark.parametrize("field", ["first", "second", "master"])
def test_adamw_state(field):
    p = [ones(130)]
    state = ops.AdamWState.zeros(p, master=True)
    bad = state._replace(**{field: torch._neg_view(getattr(state, field))})
    with pytest.raises(ValueError, match=f"adamw_step: the state's {field} .*negated"):
        ops.adamw_step(p, [ones(130)], bad, step=1)


@pytest.mark.parametrize("word, dtype", [("step", torch.int32), ("lr", F32), ("grad_scale", F32)])
def test_adamw_words(word, dtype):
    p = [ones(130)]
    state = ops.AdamWState.zeros(p)
    with pytest.raises(ValueError, match=f"adamw_step: {word} .*negated"):
        ops.adamw_step(p, [ones(130)], state, **({"step": 1} | {word: negated(1, dtype=dtype)}))
    for args in ((negated(130), ones(130)), (ones(130), negated(130))):
        with pytest.raises(ValueError, match="adamw_step: (params|grads).*negated"):
            ops.adamw_step([args[0]], [args[1]], state, step=1)
