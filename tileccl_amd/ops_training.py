"""What a training step has between its GEMMs and collectives: layer norm, activations in 8 bits, weight gradients.

The reference ends at the GEMM and the collective (``/root/reference/tileccl/ops.py``) and has no counterpart of these.
They work on each rank's own rows: the norm in front of a column-parallel layer's all-gather or behind a row-parallel
layer's reduce-scatter, the two activations that a step keeps for its backward pass (the norm's input, the linear layer's
input) in half their size, and what the backward pass makes of them:

* ``layer_norm`` / ``layer_norm_backward``: ``y = (s - mean) * rstd * weight + bias`` over the columns of each row, ``s = x``
  or ``x + residual``; the gradients of ``s``, ``weight`` and ``bias``.
* ``checkpoint_activation`` / ``restore_activation``: a 16-bit tensor to e4m3 with one power-of-two scale per block of 8
  rows x 128 columns, and back.
* ``weight_gradient``: ``x.t() @ grad`` of a linear layer whose input is held in 8 bits, or is there in full.

Tensors may lie on a symmetric heap or elsewhere on the device; launches go to torch's current stream.  Nothing is recorded for
autograd: results are detached from inputs that require gradients, and a program calls the backward operators itself (in the
``backward`` of an ``autograd.Function`` of its own, say).
"""

from __future__ import annotations

import ctypes as C
from typing import Any, NamedTuple, NoReturn

import torch

from tileccl_amd import _launch, _lib

__all__ = [
    "ActivationCheckpoint",
    "LayerNormResult",
    "LayerNormGradients",
    "layer_norm",
    "layer_norm_backward",
    "checkpoint_activation",
    "restore_activation",
    "weight_gradient",
]

_HELD_TYPES = (torch.float16, torch.bfloat16)
_TYPES = (torch.float16, torch.bfloat16, torch.float32)


class ActivationCheckpoint(NamedTuple):
    """A ``rows x columns`` tensor of ``dtype`` in 8 bits.

    ``values``: uint8 ``[ceil(rows / 8), 128 * ceil(columns / 128), 8]``, the e4m3 codes by row block, column, row in the
    block (zeros beyond the tensor); ``scales``: uint8 ``[ceil(columns / 128), ceil(rows / 8) rounded up to 16]``, the
    exponents of the blocks' scales plus 127.
    """

    values: torch.Tensor
    scales: torch.Tensor
    rows: int
    columns: int
    dtype: torch.dtype

    @staticmethod
    def shapes(rows: int, columns: int) -> tuple[tuple[int, int, int], tuple[int, int]]:
        """Shapes of ``values`` and ``scales``."""
        row_blocks, column_blocks = -(-rows // _lib.HELD_ROWS), -(-columns // _lib.HELD_COLS)
        return (row_blocks, column_blocks * _lib.HELD_COLS, _lib.HELD_ROWS), (column_blocks, -(-row_blocks // 16) * 16)

    @staticmethod
    def empty(rows: int, columns: int, dtype: torch.dtype, device: Any) -> "ActivationCheckpoint":
        """Memory for a tensor of this shape, its contents undefined."""
        values, scales = ActivationCheckpoint.shapes(rows, columns)
        return ActivationCheckpoint(torch.empty(values, dtype=torch.uint8, device=device), torch.empty(scales, dtype=torch.uint8, device=device),
                                    rows, columns, dtype)

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.scales.numel()


class LayerNormResult(NamedTuple):
    out: torch.Tensor
    mean: torch.Tensor
    rstd: torch.Tensor
    summed: torch.Tensor | None
    checkpoint: ActivationCheckpoint | None


class LayerNormGradients(NamedTuple):
    x: torch.Tensor
    weight: torch.Tensor | None
    bias: torch.Tensor | None


_native = None  # the operators of the extension module, once they have been used


def _bind() -> Any:
    """The host side of the operators (``csrc/tccl_host_ops.cpp``): checks, outputs, workspace, launch."""
    global _native
    if _native is None:
        host, lib = _lib.host(), _lib.load()
        entries = (lib.tccl_layer_norm, lib.tccl_layer_norm_grad, lib.tccl_layer_norm_grad_workspace, lib.tccl_hold, lib.tccl_restore,
                   lib.tccl_weight_gradient, lib.tccl_weight_gradient_workspace)
        host.bind_operators(_launch._raw_stream or (lambda _device: _launch.stream_ptr()), _lib.check,
                            (LayerNormResult, LayerNormGradients, ActivationCheckpoint), _TYPES,
                            tuple(C.cast(e, C.c_void_p).value for e in entries))
        from tileccl_amd.ops_gated import GatedLinearResult

        entries = (lib.tccl_weight_gradient_full, lib.tccl_weight_gradient_full_workspace, lib.tccl_gated, lib.tccl_gated_grad, lib.tccl_adamw,
                   lib.tccl_adamw_moments, lib.tccl_gated_workspace, lib.tccl_gated_grad_workspace, lib.tccl_gemm,
                   lib.tccl_pack_matrices, lib.tccl_gated_input_grad_workspace, lib.tccl_gated_input_grad_cut, lib.tccl_gated_input_grad)
        host.bind_layers(GatedLinearResult, tuple(C.cast(e, C.c_void_p).value for e in entries))
        _native = host
    return _native


# Each operator is one call of the extension module, which answers None to arguments that it does not take.  The functions
# from here on say what is wrong with them.


def _unexplained(op: str) -> NoReturn:
    raise RuntimeError(f"{op}: arguments were refused for no reason that is known here")


def _not_negated(t: torch.Tensor, name: str, op: str) -> None:
    if t.is_neg():
        raise ValueError(f"{op}: {name} is a view of negated values, call resolve_neg() on it")


def _matrix(t: Any, name: str, op: str, *, like: torch.Tensor | None = None, shape: tuple[int, int] | None = None, dtype=None) -> int:
    """Checks a 2-D device tensor with contiguous rows; its row pitch."""
    if not isinstance(t, torch.Tensor) or t.ndim != 2:
        raise ValueError(f"{op}: {name} must be a 2-D tensor, got {getattr(t, 'ndim', type(t).__name__)}")
    if not t.is_cuda:
        raise ValueError(f"{op}: {name} must reside on the GPU, got {t.device}")
    _not_negated(t, name, op)
    if like is not None:
        shape, dtype = tuple(like.shape), like.dtype
        if t.device != like.device:
            raise ValueError(f"{op}: {name} must reside on {like.device}, got {t.device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{op}: {name} must have shape {shape}, got {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{op}: {name} must have dtype {dtype}, got {t.dtype}")
    rows, cols = t.shape
    if cols == 0:
        raise ValueError(f"{op}: {name} has no columns")
    if rows > _lib.TRAINING_MAX_ROWS:
        raise ValueError(f"{op}: {name} has {rows} rows, at most {_lib.TRAINING_MAX_ROWS}")
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{op}: {name} must have contiguous rows (stride(1) == 1), got strides {tuple(t.stride())}")
    pitch = t.stride(0) if rows > 1 else cols
    if pitch < cols:
        raise ValueError(f"{op}: {name}'s rows overlap (strides {tuple(t.stride())})")
    return pitch


def _vector(t: Any, name: str, op: str, n: int, device: torch.device, types: tuple) -> None:
    if not isinstance(t, torch.Tensor) or t.shape != (n,) or t.device != device or t.dtype not in types or not t.is_contiguous():
        got = f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{op}: {name} must be a contiguous vector of {n} elements of {' or '.join(map(str, types))} on {device}, got {got}")
    _not_negated(t, name, op)


def _held(c: Any, op: str, device: torch.device | None = None) -> None:
    if not isinstance(c, ActivationCheckpoint):
        raise ValueError(f"{op}: expected an ActivationCheckpoint, got {type(c).__name__}")
    if c.dtype not in _HELD_TYPES:
        raise ValueError(f"{op}: a checkpoint holds float16 or bfloat16, not {c.dtype}")
    if not (0 <= c.rows <= _lib.TRAINING_MAX_ROWS and c.columns >= 1):
        raise ValueError(f"{op}: a checkpoint of {c.rows} x {c.columns}; rows are 0 to {_lib.TRAINING_MAX_ROWS}, columns 1 or more")
    values, scales = ActivationCheckpoint.shapes(c.rows, c.columns)
    for t, shape, name in ((c.values, values, "values"), (c.scales, scales, "scales")):
        if tuple(t.shape) != shape or t.dtype != torch.uint8 or not t.is_contiguous():
            raise ValueError(f"{op}: the checkpoint's {name} must be contiguous uint8 of shape {shape}, got {t.dtype} {tuple(t.shape)}")
        if not t.is_cuda or t.device != (device or c.values.device):
            raise ValueError(f"{op}: the checkpoint's {name} must reside on {device or 'the GPU'}, got {t.device}")


def _span(t: torch.Tensor) -> tuple[int, int]:
    rows, cols = t.shape
    start = t.data_ptr()
    return start, start + (((rows - 1) * t.stride(0) + cols) * t.element_size() if t.numel() else 0)


def _apart(out: torch.Tensor, name: str, op: str, *inputs: torch.Tensor | None) -> None:
    """An output may be an input itself, element by element, but not lie across one otherwise."""
    lo, hi = _span(out)
    for t in inputs:
        if t is None:
            continue
        a, b = _span(t)
        if a < hi and lo < b and not (a == lo and t.stride() == out.stride() and t.dtype == out.dtype):
            raise ValueError(f"{op}: {name} overlaps an input without being the same tensor")


def _bytes_of(c: ActivationCheckpoint) -> dict[str, torch.Tensor]:
    return {"the checkpoint's values": c.values, "the checkpoint's scales": c.scales}


def _clear(out: torch.Tensor, op: str, **inputs: torch.Tensor | None) -> None:
    """No row of ``out`` lies across a contiguous input that is not made of its rows."""
    lo, size = out.data_ptr(), out.element_size()
    width, step = out.shape[1] * size, (out.stride(0) if out.shape[0] > 1 else out.shape[1]) * size
    for name, t in inputs.items():
        if t is None or not t.numel() or not out.shape[0]:
            continue
        start = t.data_ptr() - lo
        row = 0 if start < width else (start - width) // step + 1  # the first one that ends behind the input's start
        if row < out.shape[0] and row * step < start + t.numel() * t.element_size():
            raise ValueError(f"{op}: out overlaps {name}")


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    eps: float = 1e-5,
    residual: torch.Tensor | None = None,
    checkpoint: bool = False,
    out: torch.Tensor | None = None,
) -> LayerNormResult:
    """Layer norm over the columns of every row of ``x`` (float16, bfloat16 or float32; up to 32768 columns).

    With ``residual`` the norm is that of ``x + residual``, rounded once to ``x``'s type and returned as ``summed``.
    ``weight`` and ``bias`` are of ``x``'s type or float32.  ``mean`` and ``rstd`` are float32; sums are float32.
    ``checkpoint``: also hold the norm's input in 8 bits, for ``layer_norm_backward``.  ``out`` (for instance on the
    symmetric heap) may be ``x`` or ``residual`` itself (the checkpoint is that of the norm's input as it was), and lies
    across no other operand.
    """
    result = (_native or _bind()).layer_norm(x, weight, bias, eps, residual, checkpoint, out)
    if result is None:
        _refuse_layer_norm(x, weight, bias, residual, checkpoint, out)
    return result


def _refuse_layer_norm(x, weight, bias, residual, checkpoint, out) -> NoReturn:
    op = "layer_norm"
    _matrix(x, "x", op)
    if x.dtype not in _TYPES:
        raise ValueError(f"{op}: x must be float16, bfloat16 or float32, got {x.dtype}")
    cols = x.shape[1]
    if cols > _lib.NORM_MAX_COLS:
        raise ValueError(f"{op}: {cols} columns, at most {_lib.NORM_MAX_COLS}")
    if checkpoint and x.dtype not in _HELD_TYPES:
        raise ValueError(f"{op}: a checkpoint holds float16 or bfloat16, not {x.dtype}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _vector(t, name, op, cols, x.device, (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{op}: weight and bias must share one dtype, got {weight.dtype} and {bias.dtype}")
    if residual is not None:
        _matrix(residual, "residual", op, like=x)
    if out is not None:
        _matrix(out, "out", op, like=x)
        _apart(out, "out", op, x, residual)
        _clear(out, op, weight=weight, bias=bias)
    _unexplained(op)


def layer_norm_backward(
    grad: torch.Tensor,
    x: "torch.Tensor | ActivationCheckpoint",
    mean: torch.Tensor,
    rstd: torch.Tensor,
    weight: torch.Tensor | None = None,
    *,
    grad_summed: torch.Tensor | None = None,
    affine: bool = True,
    out: torch.Tensor | None = None,
) -> LayerNormGradients:
    """Gradients of ``layer_norm`` for its input, weight and bias, from the gradient ``grad`` of its output.

    ``x``: the norm's input (``summed`` where there was a residual), or the checkpoint of it.  ``grad_summed``: the
    gradient that reaches the norm's input along the residual stream, added to the result.  The sums for weight and bias
    are float32, in a fixed order (the same call gives the same bits); ``affine=False``: nothing of them is stored or added up.  ``out`` may be ``grad`` or
    ``grad_summed`` itself, and lies across no other operand.
    """
    result = (_native or _bind()).layer_norm_backward(grad, x, mean, rstd, weight, grad_summed, affine, out)
    if result is None:
        _refuse_layer_norm_backward(grad, x, mean, rstd, weight, grad_summed, out)
    return result


def _refuse_layer_norm_backward(grad, x, mean, rstd, weight, grad_summed, out) -> NoReturn:
    op = "layer_norm_backward"
    _matrix(grad, "grad", op)
    if grad.dtype not in _TYPES:
        raise ValueError(f"{op}: grad must be float16, bfloat16 or float32, got {grad.dtype}")
    rows, cols = grad.shape
    if cols > _lib.NORM_MAX_COLS:
        raise ValueError(f"{op}: {cols} columns, at most {_lib.NORM_MAX_COLS}")
    full = isinstance(x, torch.Tensor)
    if full:
        _matrix(x, "x", op, like=grad)
    else:
        _held(x, op, grad.device)
        if (x.rows, x.columns) != (rows, cols) or x.dtype != grad.dtype:
            raise ValueError(f"{op}: the checkpoint is of {x.dtype} {(x.rows, x.columns)}, grad is {grad.dtype} {(rows, cols)}")
    _vector(mean, "mean", op, rows, grad.device, (torch.float32,))
    _vector(rstd, "rstd", op, rows, grad.device, (torch.float32,))
    if weight is not None:
        _vector(weight, "weight", op, cols, grad.device, (grad.dtype,) if grad.dtype == torch.float32 else (grad.dtype, torch.float32))
    if grad_summed is not None:
        _matrix(grad_summed, "grad_summed", op, like=grad)
    if out is not None:
        _matrix(out, "out", op, like=grad)
        _apart(out, "out", op, grad, grad_summed, x if full else None)
        _clear(out, op, mean=mean, rstd=rstd, weight=weight, **({} if full else _bytes_of(x)))
    _unexplained(op)


def checkpoint_activation(x: torch.Tensor) -> ActivationCheckpoint:
    """``x`` (float16 or bfloat16) in 8 bits.

    Each block of 8 rows x 128 columns has the smallest scale ``2**e``, ``e >= -117``, that its largest finite value
    fits under (``448 * 2**e``); values are rounded to the nearest e4m3, ties to even (to the one below it where that is more
    than ``x``'s type can hold); what is not finite is held as NaN.
    """
    result = (_native or _bind()).checkpoint_activation(x)
    if result is None:
        op = "checkpoint_activation"
        _matrix(x, "x", op)
        if x.dtype not in _HELD_TYPES:
            raise ValueError(f"{op}: x must be float16 or bfloat16, got {x.dtype}")
        _unexplained(op)
    return result


def restore_activation(held: ActivationCheckpoint, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that a checkpoint stands for, in the type of the tensor it was made of (exactly).  ``out`` lies
    across neither the values nor the scales."""
    result = (_native or _bind()).restore_activation(held, out)
    if result is None:
        op = "restore_activation"
        _held(held, op)
        if out is not None:
            _matrix(out, "out", op, shape=(held.rows, held.columns), dtype=held.dtype)
            if out.device != held.values.device:
                raise ValueError(f"{op}: out must reside on {held.values.device}, got {out.device}")
            _clear(out, op, **_bytes_of(held))
        _unexplained(op)
    return result


def weight_gradient(
    x: "ActivationCheckpoint | torch.Tensor",
    grad: torch.Tensor,
    *,
    layout: str = "kn",
    out_dtype: torch.dtype = torch.float32,
    add: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x.t() @ grad``: the gradient of a linear layer's weight from the layer's input ``x``, held in 8 bits or in full (float16 or
    bfloat16), and the gradient of its output, of the type of ``x``, or the one that it was held from.

    ``layout``: ``"kn"`` (inputs, outputs), as the GEMMs here take a row-major B; ``"nk"`` (outputs, inputs), as a linear
    layer holds it.  Sums are float32, rounded once to ``out_dtype`` (float32 or ``grad``'s type; that of ``out`` or
    ``add`` where one is given).  ``add``: what earlier micro-batches have summed, of the result's shape and type; ``out``
    may be ``add`` itself, and lies across no other operand.
    """
    if layout not in ("kn", "nk"):
        raise ValueError(f"weight_gradient: layout must be 'kn' or 'nk', got {layout!r}")
    if out is not None:
        out_dtype = out.dtype
    elif add is not None:
        out_dtype = add.dtype
    native = _native or _bind()
    if isinstance(x, torch.Tensor):
        result = native.weight_gradient_full(x, grad, layout == "nk", out_dtype, add, out)
        if result is None:
            _refuse_weight_gradient(x, grad, layout, out_dtype, add, out)
        return result
    result = native.weight_gradient(x, grad, None, layout == "nk", out_dtype, add, out)
    if result is not None:
        return result
    op = "weight_gradient"
    _matrix(grad, "grad", op)
    _held(x, op, grad.device)
    rows, outputs = grad.shape
    if grad.dtype != x.dtype or rows != x.rows:
        raise ValueError(f"{op}: the checkpoint is of {x.dtype} with {x.rows} rows, grad is {grad.dtype} with {rows}")
    if out_dtype not in (torch.float32, grad.dtype):
        raise ValueError(f"{op}: the result must be float32 or {grad.dtype}, got {out_dtype}")
    shape = (x.columns, outputs) if layout == "kn" else (outputs, x.columns)
    for t, name in ((add, "add"), (out, "out")):
        if t is not None:
            _matrix(t, name, op, shape=shape, dtype=out_dtype)
            if t.device != grad.device:
                raise ValueError(f"{op}: {name} must reside on {grad.device}, got {t.device}")
    if out is not None:
        _apart(out, "out", op, add)
        lo, hi = _span(out)
        if lo < _span(grad)[1] and _span(grad)[0] < hi:
            raise ValueError(f"{op}: out overlaps grad")
        _clear(out, op, **_bytes_of(x))
    width = -(-outputs // 8) * 8
    if rows and (width != outputs or grad.stride(0) % 8 or grad.data_ptr() % 16):
        # The kernel reads 16-byte vectors: a gradient without them is copied first, as the GEMMs' operands are.
        (packed,) = _launch._pack([(grad, rows, width, "weight_gradient")])
        result = _native.weight_gradient(x, packed, outputs, layout == "nk", out_dtype, add, out)
    if result is None:
        _unexplained(op)
    return result


def _refuse_weight_gradient(x, grad, layout, out_dtype, add, out) -> NoReturn:
    op = "weight_gradient"
    _matrix(grad, "grad", op)
    _matrix(x, "x", op)
    for t, name in ((x, "x"), (grad, "grad")):
        if t.dtype not in _HELD_TYPES:
            raise ValueError(f"{op}: {name} must be float16 or bfloat16, got {t.dtype}")
        if t.device.index != 0:
            raise ValueError(f"{op}: {name} must reside on cuda:0, where the ranks live, got {t.device}")
        if max(t.shape[1], t.stride(0)) > 1 << 24:
            raise ValueError(f"{op}: {name} has {t.shape[1]} columns (pitch {t.stride(0)}), at most {1 << 24}")
    rows, outputs = grad.shape
    if grad.dtype != x.dtype or rows != x.shape[0]:
        raise ValueError(f"{op}: x is {x.dtype} with {x.shape[0]} rows, grad is {grad.dtype} with {rows}")
    if out_dtype not in (torch.float32, grad.dtype):
        raise ValueError(f"{op}: the result must be float32 or {grad.dtype}, got {out_dtype}")
    inputs = x.shape[1]
    shape = (inputs, outputs) if layout == "kn" else (outputs, inputs)
    for t, name in ((add, "add"), (out, "out")):
        if t is not None:
            _matrix(t, name, op, shape=shape, dtype=out_dtype)
            if t.device != grad.device:
                raise ValueError(f"{op}: {name} must reside on {grad.device}, got {t.device}")
    if out is not None:
        _apart(out, "out", op, add)
        for t, name in ((grad, "grad"), (x, "x")):
            lo, hi = _span(out)
            if lo < _span(t)[1] and _span(t)[0] < hi:
                raise ValueError(f"{op}: out overlaps {name}")
    _unexplained(op)
