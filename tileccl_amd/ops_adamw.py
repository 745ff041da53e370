"""The update of a model's weights: AdamW over many tensors in one call, moments in 32 or 8 bits.

The reference ends at the GEMM and the collective (``/root/reference/tileccl/ops.py``) and has no counterpart.  A rank updates its own shards:
``ops.weight_gradient`` leaves their gradients in float32 beside weights in 16 bits, and that is what ``adamw_step`` takes, with a
copy of the weights in float32 (``master``) that collects updates smaller than the weights' own spacing.

Moments lie one tensor behind another in flat memory (``AdamWState``).  In 8 bits each block of 128 shares a power-of-two scale and values
are rounded at random, up or down, so that they are right on average: a second moment that moves by a thousandth of itself a step would
otherwise never leave its code.  The random numbers come from the step's number and the element's place: the same call
gives the same bits.  Tensors live on device 0; launches go to torch's current stream.
"""

from __future__ import annotations

from typing import Any, NamedTuple, NoReturn, Sequence

import torch

from tileccl_amd import _lib, ops_training
from tileccl_amd.ops_training import _not_negated, _unexplained

__all__ = ["AdamWState", "adamw_step", "adamw_moments"]

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class AdamWState(NamedTuple):
    """What ``adamw_step`` keeps of a list of tensors.

    ``first``, ``second``: flat moments, float32 or 8-bit codes (uint8); tensor ``i`` of ``sizes[i]`` elements starts at
    ``offsets(sizes)[i]``.  ``first_scales``, ``second_scales``: a byte for each 128 codes (None in 32 bits).  ``master``: the tensors in float32,
    laid out as the moments, or None.
    """

    first: torch.Tensor
    second: torch.Tensor
    first_scales: torch.Tensor | None
    second_scales: torch.Tensor | None
    master: torch.Tensor | None
    sizes: tuple[int, ...]

    @staticmethod
    def offsets(sizes: Sequence[int]) -> list[int]:
        """Where each tensor starts in flat memory, and, last, how much of that there is: multiples of 128."""
        at = [0]
        for n in sizes:
            at.append(at[-1] + -(-n // _lib.MOMENT_BLOCK) * _lib.MOMENT_BLOCK)
        return at

    @staticmethod
    def zeros(params: Sequence[torch.Tensor], *, bits: int = 32, master: bool = False) -> "AdamWState":
        """The state ahead of the first step: moments of zero and, with ``master``, the values of ``params`` in float32."""
        if bits not in (8, 32):
            raise ValueError(f"AdamWState: moments have 8 or 32 bits, got {bits}")
        params = list(params)
        device = params[0].device if params else "cuda"
        sizes = tuple(p.numel() for p in params)
        at = AdamWState.offsets(sizes)
        total = at[-1]
        copy = None
        if master:
            if any(p.dtype == torch.float32 for p in params):
                raise ValueError("AdamWState: a master copy is for params in 16 bits")
            copy = torch.zeros(total, dtype=torch.float32, device=device)
            for p, start, n in zip(params, at, sizes):
                copy[start : start + n].copy_(p.detach().reshape(-1))
        moments = [torch.zeros(total, dtype=torch.float32 if bits == 32 else torch.uint8, device=device) for _ in range(2)]
        scales = [torch.full((total // _lib.MOMENT_BLOCK,), 127, dtype=torch.uint8, device=device) for _ in range(2)] if bits == 8 else [None, None]
        return AdamWState(*moments, *scales, copy, sizes)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self[:5] if t is not None)


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    state: AdamWState,
    *,
    step: "int | torch.Tensor",
    lr: "float | torch.Tensor" = 1e-3,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    grad_scale: "float | torch.Tensor" = 1.0,
) -> None:
    """One AdamW step on every tensor of ``params``, in place, with the gradients ``grads``; ``state`` goes along.

    With ``g = grad * grad_scale``: ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g * g``,
    ``p = p (1 - lr weight_decay) - lr (m / (1 - b1**step)) / (sqrt(v / (1 - b2**step)) + eps)``, in float32, on the master copy where the
    state has one, of which ``params`` then are the rounded values.  The update takes m and v before they are held in 8 bits.

    ``params``: contiguous tensors of one type, float32, float16 or bfloat16; ``grads``: contiguous, of their shapes, all of that type or
    all float32.  Without a master copy 16-bit params are rounded to nearest: updates below half their spacing are lost.
    ``step`` counts from 1.  ``step``, ``lr`` and ``grad_scale`` may be tensors of one element on the device (int32, float32, float32),
    read when the launch runs: a step that is recorded into a graph then counts on as the program moves them (``step.add_(1)``).
    What is not finite is carried as the formulas carry it.  Nothing that is written may share memory with anything else.
    """
    native = ops_training._native or ops_training._bind()
    params, grads = tuple(params), tuple(grads)
    if not isinstance(betas, (tuple, list)) or len(betas) != 2:
        raise ValueError(f"adamw_step: betas are two numbers, got {betas!r}")
    b1, b2 = betas
    try:
        done = native.adamw_step(params, grads, tuple(state), step, lr, b1, b2, eps, weight_decay, grad_scale)
    except (TypeError, OverflowError) as e:
        raise ValueError(f"adamw_step: {e}") from e
    if done is None:
        _refuse_adamw_step(params, grads, state, step, lr, grad_scale)


def _tensor(t: Any, name: str, op: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{op}: {name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda or t.device.index != 0:
        raise ValueError(f"{op}: {name} must reside on cuda:0, got {t.device}")
    _not_negated(t, name, op)


def _flat(t: Any, name: str, op: str, dtype: torch.dtype, least: int, aligned: bool = True) -> None:
    _tensor(t, f"the state's {name}", op)
    if t.ndim != 1 or not t.is_contiguous() or t.dtype != dtype or t.numel() < least or (aligned and t.data_ptr() % 16):
        raise ValueError(f"{op}: the state's {name} must be {least} or more contiguous elements of {dtype}{' on 16 bytes' if aligned else ''}, "
                         f"got {t.dtype} {tuple(t.shape)}")


def _refuse_adamw_step(params, grads, state, step, lr, grad_scale) -> NoReturn:
    op = "adamw_step"
    if not isinstance(state, AdamWState):
        raise ValueError(f"{op}: expected an AdamWState, got {type(state).__name__}")
    if len(params) != len(grads) or len(params) != len(state.sizes):
        raise ValueError(f"{op}: {len(params)} params, {len(grads)} grads, a state of {len(state.sizes)}")
    for i, (p, g, n) in enumerate(zip(params, grads, state.sizes)):
        for t, name in ((p, f"params[{i}]"), (g, f"grads[{i}]")):
            _tensor(t, name, op)
            if not t.is_contiguous():
                raise ValueError(f"{op}: {name} must be contiguous, got strides {tuple(t.stride())}")
        if p.dtype not in _TYPES or p.dtype != params[0].dtype:
            raise ValueError(f"{op}: params must share float32, float16 or bfloat16, got {p.dtype} in params[{i}]")
        if g.dtype not in (p.dtype, torch.float32) or g.dtype != grads[0].dtype:
            raise ValueError(f"{op}: grads must all be of the params' type or all float32, got {g.dtype} in grads[{i}]")
        if p.shape != g.shape:
            raise ValueError(f"{op}: grads[{i}] must have shape {tuple(p.shape)}, got {tuple(g.shape)}")
        if p.numel() != n:
            raise ValueError(f"{op}: the state is for {n} elements in params[{i}], got {p.numel()}")
    total = AdamWState.offsets(state.sizes)[-1]
    eight = state.first_scales is not None
    moment = torch.uint8 if eight else torch.float32
    _flat(state.first, "first", op, moment, total)
    _flat(state.second, "second", op, moment, total)
    if eight or state.second_scales is not None:
        _flat(state.first_scales, "first_scales", op, torch.uint8, total // _lib.MOMENT_BLOCK, False)
        _flat(state.second_scales, "second_scales", op, torch.uint8, total // _lib.MOMENT_BLOCK, False)
    if state.master is not None:
        if params and params[0].dtype == torch.float32:
            raise ValueError(f"{op}: a master copy is for params in 16 bits")
        _flat(state.master, "master", op, torch.float32, total)
    for t, name, dtype in ((step, "step", torch.int32), (lr, "lr", torch.float32), (grad_scale, "grad_scale", torch.float32)):
        if isinstance(t, torch.Tensor):
            _tensor(t, name, op)
            if t.dtype != dtype or t.numel() != 1:
                raise ValueError(f"{op}: {name} must be a number or one element of {dtype}, got {t.dtype} {tuple(t.shape)}")
    if not isinstance(step, torch.Tensor) and not 1 <= step < 1 << 31:
        raise ValueError(f"{op}: steps are counted from 1, got {step}")
    written = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), name)
               for t, name in [(p, f"params[{i}]") for i, p in enumerate(params)] + list(zip(state[:5], state._fields)) if t is not None and t.numel()]
    read = [(g.data_ptr(), g.data_ptr() + g.numel() * g.element_size(), f"grads[{i}]") for i, g in enumerate(grads) if g.numel()]
    for i, (lo, hi, name) in enumerate(written):
        for a, b, other in written[i + 1 :] + read:
            if a < hi and lo < b:
                raise ValueError(f"{op}: {name} and {other} share memory")
        for t, word in ((step, "step"), (lr, "lr"), (grad_scale, "grad_scale")):
            if isinstance(t, torch.Tensor) and lo - 4 < t.data_ptr() < hi:
                raise ValueError(f"{op}: {word} shares memory with {name}")
    _unexplained(op)


def adamw_moments(state: AdamWState) -> tuple[torch.Tensor, torch.Tensor]:
    """(first, second) moments of a state, flat as they lie there: its own tensors in 32 bits; in 8 bits the values that the codes stand
    for, in bfloat16, which holds them exactly."""
    op = "adamw_moments"
    if not isinstance(state, AdamWState):
        raise ValueError(f"{op}: expected an AdamWState, got {type(state).__name__}")
    if state.first_scales is None:
        return state.first, state.second
    result = (ops_training._native or ops_training._bind()).adamw_moments(*state[:4])
    if result is None:
        _tensor(state.first, "first", op)
        n = state.first.numel()
        if n % _lib.MOMENT_BLOCK:
            raise ValueError(f"{op}: {n} moments are no whole blocks of {_lib.MOMENT_BLOCK}")
        _flat(state.first, "first", op, torch.uint8, n)
        _flat(state.second, "second", op, torch.uint8, n)
        for t, name in ((state.first_scales, "first_scales"), (state.second_scales, "second_scales")):
            _flat(t, name, op, torch.uint8, n // _lib.MOMENT_BLOCK, False)
        if state.second.numel() != n:
            raise ValueError(f"{op}: {n} first moments, {state.second.numel()} second ones")
        _unexplained(op)
    return result
