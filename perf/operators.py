"""The operators that a training step has between its GEMMs and collectives, as cases that can be timed.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges.  ``prepare(case, seed)`` makes what a
program holds before the call, ``run(state)`` is one pass: the operators of ``tileccl_amd.ops`` where ``own`` is true,
elementary torch operations in 32 bits where it is not.  ``work(case)`` is what one pass cannot do without, and
``exact(case, seed)`` the outputs by their definition in 64 bits.

The kinds of case (``kind``) and what each stands for:

==================  ====================================================================================
norm                ``ops.layer_norm``: the norm in front of a linear layer, with or without the residual
                    stream's addition; few rows is decoding
norm_backward       ``ops.layer_norm_backward`` from the norm's input, held in full or as an 8-bit
                    checkpoint, with the gradients of its weight and bias
norm_step           both, as a training step has them: forward with a checkpoint of the sum, backward from it
checkpoint          ``ops.checkpoint_activation`` and ``ops.restore_activation``: to 8 bits and back
weight_gradient     ``ops.weight_gradient``: checkpoint^T @ gradient of a linear layer, on top of what earlier
                    micro-batches have summed
==================  ====================================================================================

An 8-bit checkpoint of a (rows, cols) tensor: blocks of 8 rows x 128 columns, each with a scale 2^e, e the smallest whole
number (not under -117) with max|x| <= 448 * 2^e over the block's finite values; a value is held as e4m3(x / 2^e), rounded
to nearest even, what is not finite as NaN.  ``values`` (uint8) is [row block][column][row in block], the columns filled up
with zeros to whole blocks; ``scales`` (uint8) is [column block][row block], e + 127, its rows filled up to whole 16 bytes.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZES = {"f16": 2, "bf16": 2, "f32": 4}
_ROWS, _COLS, _EPS = 8, 128, 1e-5


def listed():
    return [
        # One decoding step of a batch of 16: the call itself counts.
        {"name": "norm decode", "kind": "norm", "rows": 16, "cols": 4096, "dtype": "bf16", "residual": True, "affine": "same"},
        # A long prompt or a training batch.
        {"name": "norm prompt", "kind": "norm", "rows": 8192, "cols": 4096, "dtype": "bf16", "residual": False, "affine": "same"},
        # Nothing divides, rows start anywhere; 32-bit activations.
        {"name": "norm ragged", "kind": "norm", "rows": 1000, "cols": 1003, "dtype": "f32", "residual": True, "affine": "f32"},
        # The backward pass of the smallest benchmark configuration's rows.
        {"name": "norm backward small", "kind": "norm_backward", "rows": 512, "cols": 512, "dtype": "f16", "residual": False, "affine": "same", "held": "full"},
        # The last row block and the last column block are part of one.
        {"name": "norm backward ragged", "kind": "norm_backward", "rows": 1003, "cols": 1000, "dtype": "bf16", "residual": True, "affine": "f32", "held": "8bit"},
        # A long batch of a training step.
        {"name": "norm backward long", "kind": "norm_backward", "rows": 16384, "cols": 4096, "dtype": "bf16", "residual": True, "affine": "same", "held": "full"},
        # Forward and backward of one norm of a training step that keeps 8 bits of its input.
        {"name": "norm step", "kind": "norm_step", "rows": 8192, "cols": 4096, "dtype": "bf16", "residual": True, "affine": "same"},
        # A small activation to 8 bits and back.
        {"name": "checkpoint small", "kind": "checkpoint", "rows": 512, "cols": 512, "dtype": "f16"},
        # The input of a large linear layer.
        {"name": "checkpoint batch", "kind": "checkpoint", "rows": 16384, "cols": 4096, "dtype": "bf16"},
        # Many tokens, a narrow layer: few outputs, a long sum.
        {"name": "weight gradient narrow", "kind": "weight_gradient", "rows": 16384, "cols": 1024, "outputs": 512, "dtype": "f16", "out": "f32", "layout": "kn", "add": False},
        # The linear layer of a training step, summed over micro-batches in fp32; the largest case.
        {"name": "weight gradient batch", "kind": "weight_gradient", "rows": 8192, "cols": 4096, "outputs": 4096, "dtype": "bf16", "out": "f32", "layout": "kn", "add": True},
        # Nothing divides; the weight is held as (outputs, inputs).
        {"name": "weight gradient ragged", "kind": "weight_gradient", "rows": 1003, "cols": 1000, "outputs": 2064, "dtype": "bf16", "out": "bf16", "layout": "nk", "add": False},
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], evenly spread over the logarithm."""
    value = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step, max(-(-lo // step), round(value / step))) * step


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    largest = max(_cost(c) for c in listed())
    while True:
        case = _draw_one(rng)
        if _cost(case) <= largest:
            return case


def _draw_one(rng):
    kind = rng.choice(("norm", "norm_backward", "norm_step", "checkpoint", "weight_gradient"))
    case = {"kind": kind, "rows": _spread(rng, 1, 16384), "cols": _spread(rng, 64, 16384, rng.choice((1, 8, 128)))}
    if kind == "norm":
        case["dtype"] = rng.choice(("bf16", "bf16", "f16", "f32"))
    elif kind == "norm_backward":
        case["held"] = rng.choice(("full", "8bit"))
        case["dtype"] = rng.choice(("bf16", "f16") if case["held"] == "8bit" else ("bf16", "f16", "f32"))
    else:
        case["dtype"] = rng.choice(("bf16", "f16"))
    if kind.startswith("norm"):
        case["residual"] = rng.random() < 0.5
        case["affine"] = rng.choice(("same", "f32"))
    if kind == "weight_gradient":
        case["cols"] = _spread(rng, 64, 8192, rng.choice((1, 8, 128)))
        case["outputs"] = _spread(rng, 64, 8192, rng.choice((1, 8, 128)))
        case["out"] = rng.choice(("f32", case["dtype"]))
        case["layout"] = rng.choice(("kn", "nk"))
        case["add"] = rng.random() < 0.5
    return case


def work(case):
    kind, rows, cols = case["kind"], case["rows"], case["cols"]
    size, n = _SIZES[case["dtype"]], rows * cols
    held = n + rows * cols // (_ROWS * _COLS)
    more = 1 if case.get("residual") else 0
    affine = 2 * cols * (4 if case.get("affine") == "f32" else size)
    if kind == "norm":
        return {"bytes": n * size * (2 + 2 * more) + affine + 8 * rows, "flops": 8 * n}
    if kind == "norm_backward":
        return {"bytes": n * size * (2 + more) + (held if case["held"] == "8bit" else n * size) + affine // 2 + 8 * cols + 8 * rows, "flops": 14 * n}
    if kind == "norm_step":
        return {"bytes": n * size * (4 + 3 * more) + 2 * held + affine + affine // 2 + 8 * cols + 16 * rows, "flops": 24 * n}
    if kind == "checkpoint":
        return {"bytes": 2 * (n * size + held), "flops": 4 * n}
    outputs = case["outputs"]
    out = cols * outputs * _SIZES[case["out"]]
    return {"bytes": held + rows * outputs * size + out * (2 if case["add"] else 1), "flops": 2 * n * outputs}


# ---- inputs --------------------------------------------------------------------------------------


def _activation(gen, rows, cols, dtype):
    """Normal values with an offset and a spread of each column's own, as a residual stream has them: a few columns
    in a thousand are twenty times as large."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    spread = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
    spread = torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.003, 20.0 * spread, spread)
    x *= spread
    x += 0.3 * torch.randn(cols, generator=gen, device="cuda")
    return x.to(dtype)


def _gradient(gen, rows, cols, dtype):
    """Normal values, each row of a size of its own: tokens count differently in a loss."""
    g = torch.randn(rows, cols, generator=gen, device="cuda")
    g *= 0.05 * torch.exp(0.7 * torch.randn(rows, 1, generator=gen, device="cuda"))
    return g.to(dtype)


def _blocks(x):
    """A (rows, cols) tensor as (row blocks, 8, column blocks, 128), zeros beyond it."""
    rows, cols = x.shape
    rb, cb = -(-rows // _ROWS), -(-cols // _COLS)
    full = torch.zeros(rb * _ROWS, cb * _COLS, dtype=x.dtype, device=x.device)
    full[:rows, :cols] = x
    return full.view(rb, _ROWS, cb, _COLS)


def _quantised(x):
    """(e4m3 values as blocks, exponents (row blocks, column blocks)) of a tensor, in 32 bits."""
    b = _blocks(x).float()
    finite = torch.isfinite(b)
    amax = torch.where(finite, b.abs(), torch.zeros_like(b)).amax(dim=(1, 3))
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -117)).clamp(min=-117)
    scaled = torch.ldexp(b, -e[:, None, :, None])
    q = torch.where(finite, scaled, torch.full_like(b, math.nan)).to(torch.float8_e4m3fn)
    return q, e


def _held(x):
    """(values, scales) of an 8-bit checkpoint of ``x``, laid out as the module's text says."""
    q, e = _quantised(x)
    rb, _, cb, _ = q.shape
    values = q.view(torch.uint8).permute(0, 2, 3, 1).reshape(rb, cb * _COLS, _ROWS).contiguous()
    scales = torch.full((cb, -(-rb // 16) * 16), 127, dtype=torch.uint8, device=x.device)
    scales[:, :rb] = (e + 127).t().to(torch.uint8)
    return values, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, rows, cols, dtype = case["kind"], case["rows"], case["cols"], _DTYPES[case["dtype"]]
    state = {"case": case}
    if kind == "weight_gradient":
        outputs, out = case["outputs"], _DTYPES[case["out"]]
        # The input of the layer: what a norm has left, held in 8 bits.
        state["values"], state["scales"] = _held(torch.randn(rows, cols, generator=gen, device="cuda").to(dtype))
        state["grad"] = _gradient(gen, rows, outputs, dtype)
        shape = (cols, outputs) if case["layout"] == "kn" else (outputs, cols)
        state["sum"] = torch.randn(shape, generator=gen, device="cuda").to(out) if case["add"] else None
        return state
    x = _activation(gen, rows, cols, dtype)
    if kind == "checkpoint":
        return {**state, "x": x}
    affine = torch.float32 if case["affine"] == "f32" else dtype
    state["weight"] = (1.0 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(affine)
    state["bias"] = (0.1 * torch.randn(cols, generator=gen, device="cuda")).to(affine)
    if kind == "norm_backward":
        centred = x.double()
        mean = centred.mean(dim=1)
        centred -= mean[:, None]
        state["mean"], state["rstd"] = mean.float(), ((centred * centred).mean(dim=1) + _EPS).rsqrt().float()
        if case["held"] == "8bit":
            state["values"], state["scales"] = _held(x)
        else:
            state["x"] = x
    else:
        state["x"] = x
        state["residual"] = _activation(gen, rows, cols, dtype) if case["residual"] else None
    if kind != "norm":
        state["grad"] = _gradient(gen, rows, cols, dtype)
        # What reaches the norm's input past the norm, along the residual stream.
        state["grad_summed"] = _gradient(gen, rows, cols, dtype) if case["residual"] else None
    return state


# ---- one pass -------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from tileccl_amd import ops

    case = state["case"]
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    if kind == "norm":
        r = ops.layer_norm(state["x"], state["weight"], state["bias"], eps=_EPS, residual=state["residual"])
        return {"out": r.out, "mean": r.mean, "rstd": r.rstd, "summed": r.summed}
    if kind == "norm_step":
        r = ops.layer_norm(state["x"], state["weight"], state["bias"], eps=_EPS, residual=state["residual"], checkpoint=True)
        d = ops.layer_norm_backward(state["grad"], r.checkpoint, r.mean, r.rstd, state["weight"], grad_summed=state["grad_summed"])
        return {"out": r.out, "mean": r.mean, "rstd": r.rstd, "summed": r.summed, "dx": d.x, "dweight": d.weight, "dbias": d.bias}
    if kind == "norm_backward":
        x = state["x"] if case["held"] == "full" else ops.ActivationCheckpoint(state["values"], state["scales"], case["rows"], case["cols"], dtype)
        d = ops.layer_norm_backward(state["grad"], x, state["mean"], state["rstd"], state["weight"], grad_summed=state["grad_summed"])
        return {"dx": d.x, "dweight": d.weight, "dbias": d.bias}
    if kind == "checkpoint":
        return ops.restore_activation(ops.checkpoint_activation(state["x"]))
    x = ops.ActivationCheckpoint(state["values"], state["scales"], case["rows"], case["cols"], dtype)
    return ops.weight_gradient(x, state["grad"], out_dtype=_DTYPES[case["out"]], layout=case["layout"], add=state["sum"])


def _restored(values, scales, rows, cols):
    """The values that a checkpoint stands for, in 32 bits."""
    rb, width, _ = values.shape
    q = values.view(torch.float8_e4m3fn).float().view(rb, width // _COLS, _COLS, _ROWS)
    e = scales[:, :rb].t().to(torch.int32) - 127
    return torch.ldexp(q, e[:, :, None, None]).permute(0, 3, 1, 2).reshape(rb * _ROWS, width)[:rows, :cols]


def _plain_forward(state):
    x, residual = state["x"], state["residual"]
    summed = None if residual is None else (x.float() + residual.float()).to(x.dtype)
    s = (x if summed is None else summed).float()
    mean = s.mean(dim=1)
    centred = s - mean[:, None]
    rstd = torch.rsqrt((centred * centred).mean(dim=1) + _EPS)
    out = centred * rstd[:, None] * state["weight"].float() + state["bias"].float()
    return s, {"out": out.to(x.dtype), "mean": mean, "rstd": rstd, "summed": summed}


def _plain_backward(state, s, mean, rstd):
    dy, further = state["grad"].float(), state["grad_summed"]
    normed = (s - mean[:, None]) * rstd[:, None]
    g = dy * state["weight"].float()
    along = (g * normed).mean(dim=1, keepdim=True)
    dx = rstd[:, None] * (g - g.mean(dim=1, keepdim=True) - normed * along)
    if further is not None:
        dx = dx + further.float()
    return {"dx": dx.to(state["grad"].dtype), "dweight": (dy * normed).sum(dim=0), "dbias": dy.sum(dim=0)}


def _plain(state):
    case = state["case"]
    kind, rows, cols, dtype = case["kind"], case["rows"], case["cols"], _DTYPES[case["dtype"]]
    if kind == "norm":
        return _plain_forward(state)[1]
    if kind == "norm_step":
        s, outs = _plain_forward(state)
        s = _restored(*_held(s), rows, cols)
        return {**outs, **_plain_backward(state, s, outs["mean"], outs["rstd"])}
    if kind == "norm_backward":
        s = state["x"].float() if case["held"] == "full" else _restored(state["values"], state["scales"], rows, cols)
        return _plain_backward(state, s, state["mean"], state["rstd"])
    if kind == "checkpoint":
        return _restored(*_held(state["x"]), rows, cols).to(dtype)
    x, dy = _restored(state["values"], state["scales"], rows, cols), state["grad"].float()
    dw = x.t() @ dy if case["layout"] == "kn" else dy.t() @ x
    if state["sum"] is not None:
        dw = dw + state["sum"].float()
    return dw.to(_DTYPES[case["out"]])


# ---- the definitions in 64 bits --------------------------------------------------------------------


def _exact_checkpoint(x):
    """What an 8-bit checkpoint of ``x`` stands for: every step of it is exact in 64 bits."""
    rows, cols = x.shape
    b = _blocks(x.double())
    amax = b.abs().amax(dim=(1, 3), keepdim=True)
    floor = torch.full_like(amax, -117.0)
    e = torch.where(amax > 0, torch.ceil(torch.log2(amax.clamp(min=2.0**-160) / 448.0)), floor)
    e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)  # a logarithm that was rounded
    e = torch.where((amax > 0) & (amax <= 448.0 * torch.exp2(e - 1)), e - 1, e)
    e = torch.maximum(e, floor)
    v = b / torch.exp2(e)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0**-30))), min=-6.0) - 3.0)
    v = torch.round(v / step) * step  # to even
    return (v * torch.exp2(e)).reshape(b.shape[0] * _ROWS, b.shape[2] * _COLS)[:rows, :cols]


def _exact_values(state):
    """The values of the checkpoint in ``state``, read byte by byte."""
    case = state["case"]
    code = state["values"].to(torch.int64)
    sign = 1.0 - 2.0 * (code >> 7).double()
    power, fraction = (code >> 3) & 15, (code & 7).double()
    v = torch.where(power > 0, (8.0 + fraction) * torch.exp2(power.double() - 10.0), fraction * 2.0**-9) * sign
    scale = torch.exp2(state["scales"].double() - 127.0)[:, : v.shape[0]]
    v = v * scale.t().repeat_interleave(_COLS, dim=1)[:, :, None]
    return v.transpose(1, 2).reshape(-1, v.shape[1])[: case["rows"], : case["cols"]]


def _exact_forward(state):
    s = state["x"].double()
    summed = None
    if state["residual"] is not None:
        # The sum as it is stored is the operator's definition of it: one rounding of the exact sum.
        summed = s + state["residual"].double()
        s = summed.to(state["x"].dtype).double() if state["x"].dtype != torch.float32 else summed.float().double()
    mean = s.sum(dim=1) / s.shape[1]
    variance = ((s - mean[:, None]) ** 2).sum(dim=1) / s.shape[1]
    rstd = 1.0 / torch.sqrt(variance + _EPS)
    out = (s - mean[:, None]) * rstd[:, None] * state["weight"].double() + state["bias"].double()
    return s, {"out": out, "mean": mean, "rstd": rstd, "summed": summed}


def _exact_backward(state, s, mean, rstd):
    dy, columns = state["grad"].double(), s.shape[1]
    normed = (s - mean[:, None]) * rstd[:, None]
    g = dy * state["weight"].double()
    dx = g - g.sum(dim=1, keepdim=True) / columns - normed * ((g * normed).sum(dim=1, keepdim=True) / columns)
    dx = dx * rstd[:, None]
    if state["grad_summed"] is not None:
        dx = dx + state["grad_summed"].double()
    return {"dx": dx, "dweight": (dy * normed).sum(dim=0), "dbias": dy.sum(dim=0)}


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return _exact_forward(state)[1]
    if kind == "norm_step":
        s, outs = _exact_forward(state)
        stored = s.to(state["x"].dtype)  # exact: the sum has this type
        return {**outs, **_exact_backward(state, _exact_checkpoint(stored), outs["mean"], outs["rstd"])}
    if kind == "norm_backward":
        s = state["x"].double() if case["held"] == "full" else _exact_values(state)
        return _exact_backward(state, s, state["mean"].double(), state["rstd"].double())
    if kind == "checkpoint":
        return _exact_checkpoint(state["x"])
    dw = _exact_values(state).t().contiguous() @ state["grad"].double()
    if case["layout"] == "nk":
        dw = dw.t()
    return dw if state["sum"] is None else dw + state["sum"].double()
