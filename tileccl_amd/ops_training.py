"""What a training step has between its GEMMs and collectives: layer norm, activations in 8 bits, weight gradients.

The reference ends at the GEMM and the collective (``/root/reference/tileccl/ops.py``) and has no counterpart of these.
They work on each rank's own rows: the norm in front of a column-parallel layer's all-gather or behind a row-parallel
layer's reduce-scatter, the two activations that a step keeps for its backward pass (the norm's input, the linear layer's
input) in half their size, and what the backward pass makes of them:

* ``layer_norm`` / ``layer_norm_backward``: ``y = (s - mean) * rstd * weight + bias`` over the columns of each row, ``s = x``
  or ``x + residual``; the gradients of ``s``, ``weight`` and ``bias``.
* ``checkpoint_activation`` / ``restore_activation``: a 16-bit tensor to e4m3 with one power-of-two scale per block of 8
  rows x 128 columns, and back.
* ``weight_gradient``: ``x.t() @ grad`` of a linear layer whose input is held in 8 bits.

Tensors may lie on a symmetric heap or elsewhere on the device; launches go to torch's current stream.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Any, NamedTuple

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


@dataclass(frozen=True, slots=True)
class ActivationCheckpoint:
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


def _matrix(t: Any, name: str, op: str, *, like: torch.Tensor | None = None, shape: tuple[int, int] | None = None, dtype=None) -> int:
    """Checks a 2-D device tensor with contiguous rows; its row pitch."""
    if not isinstance(t, torch.Tensor) or t.ndim != 2:
        raise ValueError(f"{op}: {name} must be a 2-D tensor, got {getattr(t, 'ndim', type(t).__name__)}")
    if not t.is_cuda:
        raise ValueError(f"{op}: {name} must reside on the GPU, got {t.device}")
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


def _held(c: Any, op: str, device: torch.device | None = None) -> None:
    if not isinstance(c, ActivationCheckpoint):
        raise ValueError(f"{op}: expected an ActivationCheckpoint, got {type(c).__name__}")
    if c.dtype not in _HELD_TYPES:
        raise ValueError(f"{op}: a checkpoint holds float16 or bfloat16, not {c.dtype}")
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
    symmetric heap) may be ``x`` or ``residual`` itself.
    """
    op = "layer_norm"
    ld_x = _matrix(x, "x", op)
    if x.dtype not in _TYPES:
        raise ValueError(f"{op}: x must be float16, bfloat16 or float32, got {x.dtype}")
    rows, cols = x.shape
    if checkpoint and x.dtype not in _HELD_TYPES:
        raise ValueError(f"{op}: a checkpoint holds float16 or bfloat16, not {x.dtype}")
    d = _lib.NormDesc()
    affine = None
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _vector(t, name, op, cols, x.device, (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32))
            if affine is not None and t.dtype != affine:
                raise ValueError(f"{op}: weight and bias must share one dtype, got {affine} and {t.dtype}")
            affine = t.dtype
    summed = None
    if residual is not None:
        d.ld_residual = _matrix(residual, "residual", op, like=x)
        summed = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
        d.residual, d.summed, d.ld_summed = residual.data_ptr(), summed.data_ptr(), cols
    if out is None:
        out = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
        d.ld_out = cols
    else:
        d.ld_out = _matrix(out, "out", op, like=x)
        _apart(out, "out", op, x, residual)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    held = None
    if checkpoint:
        held = ActivationCheckpoint.empty(rows, cols, x.dtype, x.device)
        d.values, d.scales = held.values.data_ptr(), held.scales.data_ptr()
    d.x, d.out, d.mean, d.rstd = x.data_ptr(), out.data_ptr(), mean.data_ptr(), rstd.data_ptr()
    d.weight, d.bias = _launch.ptr(weight), _launch.ptr(bias)
    d.ld_x, d.rows, d.cols, d.eps = ld_x, rows, cols, eps
    d.dtype = _launch.dtype_code(x.dtype)
    d.affine_dtype = d.dtype if affine is None else _launch.dtype_code(affine)
    rc = _lib.load().tccl_layer_norm(C.byref(d), _launch.stream_ptr())
    if rc:
        _lib.check(rc, "tccl_layer_norm")
    return LayerNormResult(out, mean, rstd, summed, held)


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
    are float32, in an order that depends on the sizes only; ``affine=False`` leaves them out.  ``out`` may be ``grad`` or
    ``grad_summed`` itself.
    """
    op = "layer_norm_backward"
    d = _lib.NormGradDesc()
    d.ld_grad = _matrix(grad, "grad", op)
    if grad.dtype not in _TYPES:
        raise ValueError(f"{op}: grad must be float16, bfloat16 or float32, got {grad.dtype}")
    rows, cols = grad.shape
    device = grad.device
    held = not isinstance(x, torch.Tensor)
    if held:
        _held(x, op, device)
        if (x.rows, x.columns) != (rows, cols) or x.dtype != grad.dtype:
            raise ValueError(f"{op}: the checkpoint is of {x.dtype} {(x.rows, x.columns)}, grad is {grad.dtype} {(rows, cols)}")
        d.values, d.scales = x.values.data_ptr(), x.scales.data_ptr()
    else:
        d.ld_x = _matrix(x, "x", op, like=grad)
        d.x = x.data_ptr()
    _vector(mean, "mean", op, rows, device, (torch.float32,))
    _vector(rstd, "rstd", op, rows, device, (torch.float32,))
    d.dtype = d.affine_dtype = _launch.dtype_code(grad.dtype)
    if weight is not None:
        _vector(weight, "weight", op, cols, device, (grad.dtype,) if grad.dtype == torch.float32 else (grad.dtype, torch.float32))
        d.weight, d.affine_dtype = weight.data_ptr(), _launch.dtype_code(weight.dtype)
    if grad_summed is not None:
        d.ld_grad_summed = _matrix(grad_summed, "grad_summed", op, like=grad)
        d.grad_summed = grad_summed.data_ptr()
    if out is None:
        out = torch.empty((rows, cols), dtype=grad.dtype, device=device)
        d.ld_dx = cols
    else:
        d.ld_dx = _matrix(out, "out", op, like=grad)
        _apart(out, "out", op, grad, grad_summed, None if held else x)
    sums = None
    if affine:
        sums = torch.empty((2, cols), dtype=torch.float32, device=device)
        d.dweight, d.dbias = sums.data_ptr(), sums.data_ptr() + 4 * cols
    lib = _lib.load()
    need = lib.tccl_layer_norm_grad_workspace(rows, cols, d.dtype, int(held))
    if need < 0:
        _lib.check(_lib.ERR_UNSUPPORTED, "tccl_layer_norm_grad")
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    d.grad, d.mean, d.rstd, d.dx = grad.data_ptr(), mean.data_ptr(), rstd.data_ptr(), out.data_ptr()
    d.workspace, d.workspace_bytes = workspace.data_ptr(), need
    d.rows, d.cols = rows, cols
    rc = lib.tccl_layer_norm_grad(C.byref(d), _launch.stream_ptr())
    if rc:
        _lib.check(rc, "tccl_layer_norm_grad")
    return LayerNormGradients(out, None if sums is None else sums[0], None if sums is None else sums[1])


def _held_desc(t: torch.Tensor, pitch: int, held: ActivationCheckpoint) -> _lib.HeldDesc:
    return _lib.HeldDesc(t.data_ptr(), held.values.data_ptr(), held.scales.data_ptr(), pitch, held.rows, held.columns, _launch.dtype_code(t.dtype))


def checkpoint_activation(x: torch.Tensor) -> ActivationCheckpoint:
    """``x`` (float16 or bfloat16) in 8 bits.

    Each block of 8 rows x 128 columns has the smallest scale ``2**e``, ``e >= -117``, that its largest finite value
    fits under (``448 * 2**e``); values are rounded to the nearest e4m3, ties to even (to the one below it where that is more
    than ``x``'s type can hold); what is not finite is held as NaN.
    """
    op = "checkpoint_activation"
    pitch = _matrix(x, "x", op)
    if x.dtype not in _HELD_TYPES:
        raise ValueError(f"{op}: x must be float16 or bfloat16, got {x.dtype}")
    held = ActivationCheckpoint.empty(int(x.shape[0]), int(x.shape[1]), x.dtype, x.device)
    rc = _lib.load().tccl_hold(C.byref(_held_desc(x, pitch, held)), _launch.stream_ptr())
    if rc:
        _lib.check(rc, "tccl_hold")
    return held


def restore_activation(held: ActivationCheckpoint, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that a checkpoint stands for, in the type of the tensor it was made of (exactly)."""
    op = "restore_activation"
    _held(held, op)
    if out is None:
        out = torch.empty((held.rows, held.columns), dtype=held.dtype, device=held.values.device)
        pitch = held.columns
    else:
        pitch = _matrix(out, "out", op, shape=(held.rows, held.columns), dtype=held.dtype)
        if out.device != held.values.device:
            raise ValueError(f"{op}: out must reside on {held.values.device}, got {out.device}")
    rc = _lib.load().tccl_restore(C.byref(_held_desc(out, pitch, held)), _launch.stream_ptr())
    if rc:
        _lib.check(rc, "tccl_restore")
    return out


def weight_gradient(
    x: ActivationCheckpoint,
    grad: torch.Tensor,
    *,
    layout: str = "kn",
    out_dtype: torch.dtype = torch.float32,
    add: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x.t() @ grad``: the gradient of a linear layer's weight from the layer's input ``x``, held in 8 bits, and the
    gradient of its output, of the type that ``x`` was held from.

    ``layout``: ``"kn"`` (inputs, outputs), as the GEMMs here take a row-major B; ``"nk"`` (outputs, inputs), as a linear
    layer holds it.  Sums are float32, rounded once to ``out_dtype`` (float32 or ``grad``'s type).  ``add``: what earlier
    micro-batches have summed, of the result's shape and type; ``out`` may be ``add`` itself.
    """
    op = "weight_gradient"
    if layout not in ("kn", "nk"):
        raise ValueError(f"{op}: layout must be 'kn' or 'nk', got {layout!r}")
    pitch = _matrix(grad, "grad", op)
    _held(x, op, grad.device)
    rows, outputs = grad.shape
    if grad.dtype != x.dtype or rows != x.rows:
        raise ValueError(f"{op}: the checkpoint is of {x.dtype} with {x.rows} rows, grad is {grad.dtype} with {rows}")
    if out is not None:
        out_dtype = out.dtype
    elif add is not None:
        out_dtype = add.dtype
    if out_dtype not in (torch.float32, grad.dtype):
        raise ValueError(f"{op}: the result must be float32 or {grad.dtype}, got {out_dtype}")
    shape = (x.columns, outputs) if layout == "kn" else (outputs, x.columns)
    d = _lib.WeightGradientDesc()
    if add is not None:
        d.ld_add = _matrix(add, "add", op, shape=shape, dtype=out_dtype)
        d.add = add.data_ptr()
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=grad.device)
        d.ld_out = shape[1]
    else:
        d.ld_out = _matrix(out, "out", op, shape=shape, dtype=out_dtype)
        if add is not None:
            _apart(out, "out", op, add)
    for t, name in ((add, "add"), (out, "out")):
        if t is not None and t.device != grad.device:
            raise ValueError(f"{op}: {name} must reside on {grad.device}, got {t.device}")
    if rows and (outputs % 8 or pitch % 8 or grad.data_ptr() % 16):
        # The kernel reads 16-byte vectors: a gradient without them is copied first, as the GEMMs' operands are.
        width = -(-outputs // 8) * 8
        (grad,) = _launch._pack([(grad, rows, width, "weight_gradient")])
        pitch = width
    lib = _lib.load()
    need = lib.tccl_weight_gradient_workspace(rows, x.columns, outputs)
    if need < 0:
        _lib.check(_lib.ERR_INVALID, "tccl_weight_gradient")
    workspace = torch.empty(need, dtype=torch.uint8, device=grad.device) if need else None
    d.values, d.scales, d.grad, d.out = x.values.data_ptr(), x.scales.data_ptr(), grad.data_ptr(), out.data_ptr()
    d.workspace, d.workspace_bytes = _launch.ptr(workspace), need
    d.ld_grad, d.rows, d.cols, d.outputs = pitch, rows, x.columns, outputs
    d.dtype, d.out_dtype, d.transposed = _launch.dtype_code(grad.dtype), _launch.dtype_code(out_dtype), int(layout == "nk")
    rc = lib.tccl_weight_gradient(C.byref(d), _launch.stream_ptr())
    if rc:
        _lib.check(rc, "tccl_weight_gradient")
    return out
