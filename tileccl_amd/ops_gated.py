"""The gated linear layer of a feed-forward block, and its gradients.

The reference ends at the GEMM and the collective (``/root/reference/tileccl/ops.py``) and has no counterpart of these.  With a
rank's columns of both projections the layer is column-parallel: its input is what an all-gather has left, the gradient of
its input is a partial sum that a GEMM + reduce-scatter (``tileccl_amd.v2.FusedGemmReduceScatter``) makes of
``gated_linear_backward(..., inputs=False).inner`` and the weight's transpose.

* ``gated_linear``: ``act(x @ W[:, :F]) * (x @ W[:, F:])`` for a weight ``W`` of 2 F columns; both projections are never in memory
  unless they are kept for the backward pass.
* ``gated_linear_backward``: the gradients of the two projections (from the kept ones, or from ones that are computed again), of the
  input and of the weight.

Tensors may lie on a symmetric heap or elsewhere on device 0; launches go to torch's current stream.  Nothing is recorded for autograd,
as in ``ops_training``.
"""

from __future__ import annotations

from typing import Any, NamedTuple, NoReturn

import torch

from tileccl_amd import _lib, ops_training
from tileccl_amd.ops_training import ActivationCheckpoint, _apart, _bytes_of, _clear, _held, _matrix, _not_negated, _span, _unexplained, weight_gradient

__all__ = ["GatedLinearResult", "GatedLinearGradients", "gated_linear", "gated_linear_backward"]

ACTIVATIONS = {"silu": _lib.SILU, "gelu": _lib.GELU, "gelu_tanh": _lib.GELU_TANH, "relu": _lib.RELU}
_TYPES = (torch.float16, torch.bfloat16)
_MOST_PITCH = 1 << 24  # of what weight gradients read


class GatedLinearResult(NamedTuple):
    out: torch.Tensor
    kept: torch.Tensor | None


class GatedLinearGradients(NamedTuple):
    inner: torch.Tensor
    x: torch.Tensor | None
    weight: torch.Tensor | None


def _activation(name: str, op: str) -> int:
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"{op}: activation must be one of {', '.join(map(repr, ACTIVATIONS))}, got {name!r}")
    return code


def _device0(t: torch.Tensor, name: str, op: str) -> None:
    if t.device.index != 0:
        raise ValueError(f"{op}: {name} must reside on cuda:0, where the ranks live, got {t.device}")


def _weight(w: Any, op: str) -> None:
    if not isinstance(w, torch.Tensor) or w.ndim != 2:
        raise ValueError(f"{op}: weight must be a 2-D tensor, got {getattr(w, 'ndim', type(w).__name__)}")
    if not w.is_cuda:
        raise ValueError(f"{op}: weight must reside on the GPU, got {w.device}")
    _device0(w, "weight", op)
    _not_negated(w, "weight", op)
    inputs, columns = w.shape
    if columns % 2 or not columns or not inputs:
        raise ValueError(f"{op}: weight must be (inputs, 2 * outputs), got {tuple(w.shape)}")
    if max(inputs, columns // 2) > _lib.GATED_MAX_COLS:
        raise ValueError(f"{op}: weight of {tuple(w.shape)}, at most {_lib.GATED_MAX_COLS} inputs and outputs")
    if w.dtype not in _TYPES:
        raise ValueError(f"{op}: weight must be float16 or bfloat16, got {w.dtype}")
    by_rows = w.stride(1) == 1 and (inputs == 1 or w.stride(0) >= columns)
    if not by_rows and not ((inputs == 1 or w.stride(0) == 1) and w.stride(1) >= inputs):
        raise ValueError(f"{op}: weight must have contiguous rows, or be the .t() view of a tensor that has, got strides {tuple(w.stride())}")


def _by_rows(w: torch.Tensor) -> bool:
    return w.stride(1) == 1 and (w.shape[0] == 1 or w.stride(0) >= w.shape[1])


def _weight_span(w: torch.Tensor) -> tuple[int, int]:
    return _span(w if _by_rows(w) else w.t())


def _elsewhere(out: torch.Tensor, op: str, **others: "tuple[int, int]") -> None:
    lo, hi = _span(out)
    for name, (a, b) in others.items():
        if a < hi and lo < b:
            raise ValueError(f"{op}: out overlaps {name}")


def _beside(a: torch.Tensor, b: torch.Tensor) -> bool:
    """No byte of either matrix's rows lies in the other's; rows of one pitch may lie beside each other."""
    (lo, hi), (start, end) = _span(a), _span(b)
    if end <= lo or hi <= start:
        return True
    step = a.stride(0) * a.element_size()
    if min(a.shape[0], b.shape[0]) < 2 or step != b.stride(0) * b.element_size():
        return False
    ahead = (start - lo) % step
    return ahead >= a.shape[1] * a.element_size() and ahead + b.shape[1] * b.element_size() <= step


def gated_linear(x: torch.Tensor, weight: torch.Tensor, *, activation: str = "silu", keep: bool = False, out: torch.Tensor | None = None) -> GatedLinearResult:
    """``act(x @ weight[:, :F]) * (x @ weight[:, F:])`` for ``x`` (rows, inputs) and ``weight`` (inputs, 2 * F), float16 or bfloat16.

    ``weight`` has contiguous rows, or is the ``.t()`` view of a (2 * F, inputs) tensor that has, as a linear layer holds it.
    ``activation``: ``"silu"``, ``"gelu"`` (by the normal distribution), ``"gelu_tanh"`` (its approximation) or ``"relu"``.
    ``keep``: also hand back ``x @ weight`` in ``x``'s type (rows, 2 * F), which ``gated_linear_backward`` takes.  Sums,
    activation and product are float32, rounded once.  ``out`` lies across no operand.

    Rows that are no whole 16-byte vectors (inputs, F or a pitch no multiple of 8) are copied first, the weight's among them: a program
    that calls with few rows holds its weight in rows that are.
    """
    code = _activation(activation, "gated_linear")
    native = ops_training._native or ops_training._bind()
    result = native.gated_linear(x, weight, code, keep, out)
    if result is None:
        _refuse_gated_linear(x, weight, out)
    return result


def _refuse_gated_linear(x, weight, out) -> NoReturn:
    op = "gated_linear"
    _weight(weight, op)
    _matrix(x, "x", op, dtype=weight.dtype)
    _device0(x, "x", op)
    if x.shape[1] != weight.shape[0]:
        raise ValueError(f"{op}: x has {x.shape[1]} columns, weight {weight.shape[0]} rows")
    if out is not None:
        _matrix(out, "out", op, shape=(x.shape[0], weight.shape[1] // 2), dtype=x.dtype)
        _device0(out, "out", op)
        _elsewhere(out, op, x=_span(x), weight=_weight_span(weight))
    _unexplained(op)


def gated_linear_backward(
    grad: torch.Tensor,
    kept: torch.Tensor | None,
    x: "torch.Tensor | ActivationCheckpoint",
    weight: torch.Tensor,
    *,
    activation: str = "silu",
    inputs: bool = True,
    weights: bool = True,
    out_dtype: torch.dtype = torch.float32,
    add: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> GatedLinearGradients:
    """Gradients of ``gated_linear`` from the gradient ``grad`` of its output.

    ``inner`` (rows, 2 * F): the gradient of ``x @ weight``, made of ``kept``, or, where that is None, of the product computed
    again, which is then not rounded on the way (``x`` must be the tensor itself); rounded once.  ``out`` is where it goes: ``kept``
    itself, which has no further use, or memory that lies across no operand (with ``weights`` ``x``, its checkpoint and ``add`` are some).
    ``x``: ``inner @ weight.t()``, contiguous, in ``grad``'s type; ``inputs=False``: not wanted, for instance because it is summed over ranks.
    ``weight``: ``x.t() @ inner`` in ``out_dtype`` (float32 or ``grad``'s type; ``add``'s where that is given), of ``weight``'s shape and
    layout, on top of ``add`` (of that layout, too): ``ops.weight_gradient``, from ``x`` in full or its 8-bit checkpoint.
    ``weights=False``: not wanted.
    """
    op = "gated_linear_backward"
    code = _activation(activation, op)
    native = ops_training._native or ops_training._bind()
    # What the weight's gradient would refuse is refused here, ahead of a result that may lie in kept's place.
    inner = native.gated_gradient(grad, kept, x, weight, code, out, weights, out_dtype, add)
    if inner is None:
        _refuse_backward(grad, kept, x, weight, out, weights, out_dtype, add)
    dx = dw = None
    if weights:
        by_rows = _by_rows(weight)
        dw = weight_gradient(x, inner, layout="kn" if by_rows else "nk", out_dtype=out_dtype, add=add if add is None or by_rows else add.t())
        dw = dw if by_rows else dw.t()
    if inputs:
        dx = native.input_gradient(inner, weight)
        if dx is None:
            _unexplained(op)
    return GatedLinearGradients(inner, dx, dw)


def _refuse_shapes(grad, x, weight, add, op) -> None:
    if isinstance(x, ActivationCheckpoint):
        rows, columns = x.rows, x.columns
    elif isinstance(x, torch.Tensor) and x.ndim == 2:
        rows, columns = x.shape
    else:
        raise ValueError(f"{op}: the weight's gradient wants x, a 2-D tensor or its checkpoint, got {type(x).__name__}")
    if add is not None and (not isinstance(add, torch.Tensor) or add.ndim != 2):
        raise ValueError(f"{op}: add must be a 2-D tensor, got {getattr(add, 'ndim', type(add).__name__)}")
    if isinstance(weight, torch.Tensor) and isinstance(grad, torch.Tensor) and weight.ndim == grad.ndim == 2:  # (else refused with their names)
        if columns != weight.shape[0]:
            raise ValueError(f"{op}: x has {columns} columns, weight {weight.shape[0]} rows")
        if rows != grad.shape[0]:
            raise ValueError(f"{op}: x has {rows} rows, grad {grad.shape[0]}")
        if add is not None and add.shape != weight.shape:
            raise ValueError(f"{op}: add must have shape {tuple(weight.shape)}, got {tuple(add.shape)}")


def _refuse_weight_gradient(grad, x, weight, out, out_dtype, add, op) -> None:
    """What ``weight_gradient`` would refuse."""
    if isinstance(x, ActivationCheckpoint):
        _held(x, op, grad.device)
        if x.dtype != grad.dtype:
            raise ValueError(f"{op}: the checkpoint is of {x.dtype}, grad is {grad.dtype}")
        if x.values.data_ptr() % 16:
            raise ValueError(f"{op}: the checkpoint's values must lie on 16 bytes")
    else:
        pitch = _matrix(x, "x", op, dtype=grad.dtype)
        _device0(x, "x", op)
        if pitch > _MOST_PITCH:
            raise ValueError(f"{op}: x has {x.shape[1]} columns (pitch {pitch}), at most {_MOST_PITCH}")
    if out is not None and out.shape[0] > 1 and out.stride(0) > _MOST_PITCH:
        raise ValueError(f"{op}: out has a pitch of {out.stride(0)} elements, at most {_MOST_PITCH} where the weight's gradient is made of it")
    if out is not None:
        if isinstance(x, ActivationCheckpoint):
            _clear(out, op, **_bytes_of(x))
        for t, name in ((x, "x"), (add if add is None or _by_rows(weight) else add.t(), "add")):
            if isinstance(t, torch.Tensor) and not _beside(out, t):
                raise ValueError(f"{op}: out overlaps {name}")
    if add is None:
        if out_dtype not in (torch.float32, grad.dtype):
            raise ValueError(f"{op}: the weight's gradient must be float32 or {grad.dtype}, got {out_dtype}")
        return
    if add.dtype not in (torch.float32, grad.dtype):
        raise ValueError(f"{op}: add must be float32 or {grad.dtype}, got {add.dtype}")
    lies = add if _by_rows(weight) else add.t()
    if lies.shape[1] > 1 and lies.stride(1) != 1:
        raise ValueError(f"{op}: add must have contiguous rows where weight has, columns where weight has these, got strides {tuple(add.stride())}")
    _matrix(lies, "add", op)
    _device0(add, "add", op)


def _refuse_backward(grad, kept, x, weight, out, weights, out_dtype, add) -> NoReturn:
    op = "gated_linear_backward"
    if weights:
        _refuse_shapes(grad, x, weight, add, op)
    _weight(weight, op)
    outputs = weight.shape[1] // 2
    _matrix(grad, "grad", op, dtype=weight.dtype)
    _device0(grad, "grad", op)
    rows = grad.shape[0]
    if grad.shape[1] != outputs:
        raise ValueError(f"{op}: grad has {grad.shape[1]} columns, weight is for {outputs} outputs")
    if kept is not None:
        _matrix(kept, "kept", op, shape=(rows, 2 * outputs), dtype=weight.dtype)
        _device0(kept, "kept", op)
    elif isinstance(x, ActivationCheckpoint):
        raise ValueError(f"{op}: without kept the projections are computed from x itself, not from a checkpoint of it")
    else:
        _matrix(x, "x", op, shape=(rows, weight.shape[0]), dtype=weight.dtype)
        _device0(x, "x", op)
    if out is not None:
        _matrix(out, "out", op, shape=(rows, 2 * outputs), dtype=weight.dtype)
        _device0(out, "out", op)
        _elsewhere(out, op, grad=_span(grad), weight=_weight_span(weight), **({"x": _span(x)} if kept is None else {}))
        _apart(out, "out", op, kept)
    if weights:
        _refuse_weight_gradient(grad, x, weight, out, out_dtype, add, op)
    _unexplained(op)
