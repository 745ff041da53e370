"""A gated feed-forward layer of a training step or of a decoder, and the update of its weights, as cases that can be timed.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges.  ``prepare(case, seed)`` makes what a
program holds before the call, ``run(state)`` is one pass: the operators of ``tileccl_amd.ops`` where ``own`` is true,
elementary torch operations in 32 bits where it is not.  ``work(case)`` is what one pass cannot do without, and
``exact(case, seed)`` the outputs by their definition in 64 bits.

The kinds of case (``kind``) and what each stands for:

==================  ====================================================================================
gated               ``ops.gated_linear``: both projections of a gated feed-forward layer, the activation and the
                    product; few rows is decoding
gated_backward      ``ops.gated_linear_backward``: from the gradient of that product the gradients of the two
                    projections, of the layer's input and of its weight; the projections are kept or computed again
gated_step          both, as a training step has them
weight_gradient     ``ops.weight_gradient`` from a linear layer's input in full
adamw               ``ops.adamw_step``: the update of all weights, moments in 32 or in 8 bits
==================  ====================================================================================

``weight`` is (inputs, 2 * outputs): the gate's columns, then the other projection's.  ``layout`` says how it lies in
memory: ``kn`` row by row, ``nk`` as the ``.t()`` view of a (2 * outputs, inputs) tensor.

Moments of AdamW in 8 bits lie one tensor behind another, each from a multiple of 128 elements on, with a scale 2^e for every
128 elements (a byte, e + 127), and are rounded up or down at random, so that a held value is on average the one that it was
made of: a value y / 2^e that lies the fraction f of a step above the held value under it becomes the next one where
f + u >= 1.  u is 16 bits of a hash of the element's place and the step's number (``_noise``): the lower ones for the first
moment, the upper ones for the second.

* first moment: e4m3, e the smallest whole number (not under -117) with max|m| <= 448 * 2^e over the block's finite values;
* second moment: code 0 is 0, code c from 1 to 254 is (1 + ((c - 1) % 8) / 8) * 2^((c - 1) // 8 - 30); e = floor(log2(max v)), in
  -90 .. 127; what is positive is never held as less than code 1.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZES = {"f16": 2, "bf16": 2, "f32": 4}
_BLOCK = 128
_BETAS, _EPS, _DECAY, _LR = (0.9, 0.999), 1e-8, 0.01, 3e-4


def listed():
    return [
        # One token of one sequence: two weights are read, and next to nothing is computed.
        {"name": "gated token", "kind": "gated", "rows": 1, "inputs": 4096, "outputs": 8192, "dtype": "bf16", "layout": "nk", "activation": "silu", "keep": False},
        # One step of a batch that is no round number, a weight that lies row by row.
        {"name": "gated decode", "kind": "gated", "rows": 13, "inputs": 4096, "outputs": 4096, "dtype": "f16", "layout": "kn", "activation": "gelu_tanh", "keep": False},
        # Nothing divides anything.
        {"name": "gated ragged", "kind": "gated", "rows": 1003, "inputs": 1001, "outputs": 1035, "dtype": "bf16", "layout": "kn", "activation": "gelu", "keep": True},
        # A long prompt; the largest case.
        {"name": "gated prompt", "kind": "gated", "rows": 8192, "inputs": 4096, "outputs": 8192, "dtype": "bf16", "layout": "nk", "activation": "silu", "keep": False},
        # The backward pass of a small batch.
        {"name": "gated backward", "kind": "gated_backward", "rows": 2048, "inputs": 2048, "outputs": 4096, "dtype": "f16", "layout": "kn", "activation": "gelu_tanh", "kept": True, "add": False},
        # Nothing was kept, sums over micro-batches go on, nothing is a multiple of a tile.
        {"name": "gated backward ragged", "kind": "gated_backward", "rows": 999, "inputs": 1000, "outputs": 1544, "dtype": "bf16", "layout": "nk", "activation": "silu", "kept": False, "add": True},
        # A layer of a training step, forward and backward.
        {"name": "gated step", "kind": "gated_step", "rows": 4096, "inputs": 4096, "outputs": 4096, "dtype": "bf16", "layout": "kn", "activation": "silu", "kept": True, "add": False},
        # Many tokens, a narrow layer: few outputs, a long sum.
        {"name": "weight gradient narrow", "kind": "weight_gradient", "rows": 16384, "inputs": 1024, "outputs": 512, "dtype": "f16", "out": "f32", "layout": "kn", "add": False},
        # The second linear layer of a block, summed over micro-batches, its weight held as (outputs, inputs).
        {"name": "weight gradient batch", "kind": "weight_gradient", "rows": 4096, "inputs": 8192, "outputs": 4096, "dtype": "bf16", "out": "f32", "layout": "nk", "add": True},
        # A few small weights: the call itself counts.
        {"name": "adamw few", "kind": "adamw", "tensors": 6, "most": 262144, "sizes": 1, "dtype": "f32", "grad": "f32", "bits": 32, "master": False, "step": 10},
        # A block's weights in 16 bits beside a copy in 32, gradients as the weight gradients leave them.
        {"name": "adamw block", "kind": "adamw", "tensors": 12, "most": 67108864, "sizes": 2, "dtype": "bf16", "grad": "f32", "bits": 32, "master": True, "step": 1000},
        # Many tensors of any size, moments in 8 bits.
        {"name": "adamw 8 bits", "kind": "adamw", "tensors": 150, "most": 16777216, "sizes": 3, "dtype": "bf16", "grad": "bf16", "bits": 8, "master": True, "step": 300},
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
    kind = rng.choice(("gated", "gated", "gated_backward", "gated_step", "weight_gradient", "adamw"))
    if kind == "adamw":
        dtype, grad = rng.choice((("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32")))
        return {"kind": kind, "tensors": _spread(rng, 1, 300), "most": _spread(rng, 1, 1 << 26), "sizes": rng.randrange(1 << 30), "dtype": dtype, "grad": grad,
                "bits": rng.choice((8, 32)), "master": dtype != "f32" and rng.random() < 0.6, "step": _spread(rng, 1, 100000)}
    odd = rng.choice((1, 8, 128))
    case = {"kind": kind, "rows": _spread(rng, 1, 16384), "inputs": _spread(rng, 64, 8192, odd), "outputs": _spread(rng, 64, 8192, odd),
            "dtype": rng.choice(("bf16", "f16")), "layout": rng.choice(("kn", "nk"))}
    if kind == "weight_gradient":
        return {**case, "out": rng.choice(("f32", case["dtype"])), "add": rng.random() < 0.5}
    case["activation"] = rng.choice(("silu", "gelu", "gelu_tanh", "relu"))
    if kind == "gated":
        return {**case, "keep": rng.random() < 0.5}
    # A projection that is computed again may have its last bit another way, and relu's derivative jumps at 0.
    if kind == "gated_step" and case["activation"] == "relu":
        case["activation"] = "silu"
    case["kept"] = rng.random() < 0.6 or case["activation"] == "relu"
    return {**case, "add": rng.random() < 0.5}


def _tensor_sizes(case):
    """How many elements each tensor has: from 1 to ``most``, the first one ``most``, and where each starts in flat memory."""
    rng = random.Random(case["sizes"])
    sizes = [case["most"]] + [_spread(rng, 1, case["most"]) for _ in range(case["tensors"] - 1)]
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // _BLOCK) * _BLOCK
    return sizes, starts, at


def work(case):
    kind = case["kind"]
    if kind == "adamw":
        n, p, g = sum(_tensor_sizes(case)[0]), _SIZES[case["dtype"]], _SIZES[case["grad"]]
        each = g + (8 + p if case["master"] else 2 * p)  # a copy in 32 bits is read and written, its 16 bits are written
        # Moments are read and written; those in 8 bits come back as the 16-bit values that they stand for.
        each += 16 if case["bits"] == 32 else 4 * (1 + 1 / _BLOCK) + 2 * (1 + 1 / _BLOCK) + 4
        return {"bytes": int(n * each), "flops": 15 * n}
    rows, inputs, outputs, e = case["rows"], case["inputs"], case["outputs"], _SIZES[case["dtype"]]
    if kind == "weight_gradient":
        out = inputs * outputs * _SIZES[case["out"]]
        return {"bytes": e * rows * (inputs + outputs) + out * (2 if case["add"] else 1), "flops": 2 * rows * inputs * outputs}
    x, w, h = e * rows * inputs, e * 2 * inputs * outputs, e * rows * outputs
    product = 4 * rows * inputs * outputs
    if kind == "gated":
        return {"bytes": x + w + h * (3 if case["keep"] else 1), "flops": product}
    dw = e * 2 * inputs * outputs
    back = {"bytes": h + (2 * h if case["kept"] else 0) + x + w + 2 * h + x + dw * (2 if case["add"] else 1), "flops": product * (2 if case["kept"] else 3)}
    if kind == "gated_step":
        back["bytes"] += x + w + h * (3 if case["kept"] else 1)
        back["flops"] += product
    return back


# ---- inputs --------------------------------------------------------------------------------------


def _gradient(gen, rows, cols, dtype):
    """Normal values, each row of a size of its own: tokens count differently in a loss."""
    g = torch.randn(rows, cols, generator=gen, device="cuda")
    g *= 0.05 * torch.exp(0.7 * torch.randn(rows, 1, generator=gen, device="cuda"))
    return g.to(dtype)


def _weight(gen, inputs, columns, dtype, layout):
    w = torch.randn((inputs, columns) if layout == "kn" else (columns, inputs), generator=gen, device="cuda")
    w *= 1.2 * inputs**-0.5
    w = w.to(dtype)
    return w if layout == "kn" else w.t()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    if kind == "adamw":
        return _prepare_adamw(case, gen)
    rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
    # What a norm has left.
    state = {"case": case, "x": torch.randn(rows, inputs, generator=gen, device="cuda").to(dtype)}
    if kind == "weight_gradient":
        state["grad"] = _gradient(gen, rows, outputs, dtype)
        shape = (inputs, outputs) if case["layout"] == "kn" else (outputs, inputs)
        state["sum"] = torch.randn(shape, generator=gen, device="cuda").to(_DTYPES[case["out"]]) if case["add"] else None
        return state
    state["weight"] = _weight(gen, inputs, 2 * outputs, dtype, case["layout"])
    if kind != "gated":
        state["grad"] = _gradient(gen, rows, outputs, dtype)
        # The weight's gradient has the weight's type here: it is that of values that were rounded once already.
        if case["add"]:
            state["sum"] = torch.randn((inputs, 2 * outputs) if case["layout"] == "kn" else (2 * outputs, inputs), generator=gen, device="cuda").to(dtype)
            state["sum"] = state["sum"] if case["layout"] == "kn" else state["sum"].t()
        else:
            state["sum"] = None
    if kind == "gated_backward":
        # The projections as the forward pass has kept them.
        state["kept"] = (state["x"].float() @ state["weight"].float()).to(dtype) if case["kept"] else None
    return state


def _prepare_adamw(case, gen):
    sizes, starts, total = _tensor_sizes(case)
    dtype, grad = _DTYPES[case["dtype"]], _DTYPES[case["grad"]]
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    # Elements that no gradient has reached yet are 0 in both moments: rows of a table that no token has had.
    spread = torch.exp(1.5 * torch.randn(total // _BLOCK, generator=gen, device="cuda")).repeat_interleave(_BLOCK)
    for n, at in zip(sizes, starts):
        used[at : at + n] = True
    spread *= used
    rand = lambda: torch.randn(total, generator=gen, device="cuda")  # noqa: E731
    scale = 256.0 if case["grad"] == "f16" else 1.0
    flat = {"params": 0.02 * rand() * used, "grads": (1e-3 * scale * rand() * spread).to(grad)}
    flat["params"], master = flat["params"].to(dtype), flat["params"]
    if case["master"]:
        flat["master"] = master
    first, second = 3e-4 * rand() * spread, (0.9e-3 * spread) ** 2 * torch.exp(0.5 * rand())
    never = torch.rand(total // _BLOCK, generator=gen, device="cuda").lt(0.02).repeat_interleave(_BLOCK)
    first.masked_fill_(never, 0.0)
    second.masked_fill_(never, 0.0)
    if case["bits"] == 8:
        zero = torch.zeros((), device="cuda")
        flat["first"], flat["first_scales"] = _first_codes(first, zero)
        flat["second"], flat["second_scales"] = _second_codes(second, zero)
    else:
        flat["first"], flat["second"] = first, second
    views = lambda t: [t[at : at + n] for n, at in zip(sizes, starts)]  # noqa: E731
    return {"case": case, "flat": flat, "params": views(flat["params"]), "grads": views(flat["grads"]), "sizes": tuple(sizes), "grad_scale": 1.0 / scale}


# ---- one pass -------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from tileccl_amd import ops

    case = state["case"]
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    if kind == "adamw":
        flat = state["flat"]
        held = ops.AdamWState(flat["first"], flat["second"], flat.get("first_scales"), flat.get("second_scales"), flat.get("master"), state["sizes"])
        ops.adamw_step(state["params"], state["grads"], held, step=case["step"], lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_DECAY, grad_scale=state["grad_scale"])
        first, second = ops.adamw_moments(held)
        return {"params": flat["params"], "master": flat.get("master"), "first": first, "second": second}
    if kind == "weight_gradient":
        return ops.weight_gradient(state["x"], state["grad"], out_dtype=_DTYPES[case["out"]], layout=case["layout"], add=state["sum"])
    outs, kept = {}, state.get("kept")
    if kind != "gated_backward":
        r = ops.gated_linear(state["x"], state["weight"], activation=case["activation"], keep=case["keep"] if kind == "gated" else case["kept"])
        outs, kept = {"out": r.out, "kept": r.kept}, r.kept
    if kind != "gated":
        d = ops.gated_linear_backward(state["grad"], kept, state["x"], state["weight"], activation=case["activation"], out_dtype=dtype, add=state["sum"])
        outs = {**outs, "inner": d.inner, "dx": d.x, "dweight": d.weight}
    return outs


def _activated(g, activation):
    """The activation of ``g`` and its derivative, in ``g``'s type."""
    if activation == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if activation == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * (c * (1.0 + 3 * 0.044715 * g * g))


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "adamw":
        return _plain_adamw(state)
    x = state["x"].float()
    if kind == "weight_gradient":
        dy = state["grad"].float()
        dw = x.t() @ dy if case["layout"] == "kn" else dy.t() @ x
        if state["sum"] is not None:
            dw = dw + state["sum"].float()
        return dw.to(_DTYPES[case["out"]])
    dtype, n = state["x"].dtype, case["outputs"]
    w = state["weight"].float()
    outs, kept = {}, state.get("kept")
    if kind != "gated_backward":
        z = x @ w
        keep = case["keep"] if kind == "gated" else case["kept"]
        kept = z.to(dtype) if keep else None
        outs = {"out": (_activated(z[:, :n], case["activation"])[0] * z[:, n:]).to(dtype), "kept": kept}
    if kind != "gated":
        z = kept.float() if kept is not None else x @ w
        dh = state["grad"].float()
        a, slope = _activated(z[:, :n], case["activation"])
        inner = torch.cat([dh * z[:, n:] * slope, dh * a], dim=1).to(dtype)
        d = inner.float()
        dw = x.t() @ d
        if state["sum"] is not None:
            dw = dw + state["sum"].float()
        outs = {**outs, "inner": inner, "dx": (d @ w.t()).to(dtype), "dweight": dw.to(dtype)}
    return outs


# -- AdamW


def _noise(total, step, device):
    """32 bits for each place in flat memory, another pattern for every step.  (Whole numbers below 2^32, held in 64 bits.)"""
    most = 0xFFFFFFFF
    place = torch.arange(total, device=device, dtype=torch.int64)
    key = (step * 0x9E3779B9 + (place >> 32) * 0xBB67AE85) & most
    h = (place & most) ^ key
    h = ((h ^ (h >> 16)) * 0x6A09E667) & most
    h = ((h ^ (h >> 15)) * 0x3C6EF373) & most
    return h ^ (h >> 16)


def _finite_max(blocks):
    return torch.where(torch.isfinite(blocks), blocks.abs(), torch.zeros_like(blocks)).amax(dim=1)


def _first_codes(m, u):
    """(codes, scales) of first moments; ``u``: what is added to the fraction of a step."""
    b = m.view(-1, _BLOCK)
    amax = _finite_max(b)
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -117)).clamp(min=-117)
    y = torch.ldexp(b.abs(), -e[:, None])
    step = torch.ldexp(torch.ones_like(y), torch.clamp(torch.frexp(y)[1] - 1, min=-6) - 3)
    q = torch.floor(y / step + (u.view(-1, _BLOCK) if u.dim() else u)) * step
    q = torch.where(torch.isfinite(b), torch.copysign(q, b), torch.full_like(b, math.nan))
    return q.to(torch.float8_e4m3fn).view(torch.uint8).view(-1), (e + 127).to(torch.uint8)


def _second_codes(v, u):
    b = v.view(-1, _BLOCK)
    amax = _finite_max(b)
    e = (torch.frexp(amax)[1] - 1).clamp(-90, 127)
    e = torch.where(amax > 0, e, torch.full_like(e, -90))
    y = torch.ldexp(b, -e[:, None])
    mantissa, exponent = torch.frexp(y)  # y = 2 mantissa * 2^(exponent - 1)
    steps = torch.floor(16.0 * mantissa + (u.view(-1, _BLOCK) if u.dim() else u)).to(torch.int32)  # 8 .. 16
    code = torch.clamp(8 * (exponent - 1 + 30) + steps - 8 + 1, min=1)
    code = torch.where(y > 0, code, torch.zeros_like(code))
    code = torch.where(torch.isfinite(b), code, torch.full_like(code, 255))
    return code.to(torch.uint8).view(-1), (e + 127).to(torch.uint8)


def _first_values(codes, scales):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float().view(-1, _BLOCK), scales.to(torch.int32)[:, None] - 127).view(-1)


def _second_values(codes, scales):
    c = codes.view(-1, _BLOCK).to(torch.int32) - 1
    v = torch.ldexp(1.0 + (c & 7).float() / 8.0, (c >> 3) - 30 + scales.to(torch.int32)[:, None] - 127)
    v = torch.where(c < 0, torch.zeros_like(v), v)
    return torch.where(c == 254, torch.full_like(v, math.nan), v).view(-1)


def _plain_adamw(state):
    case, flat = state["case"], state["flat"]
    (b1, b2), t = _BETAS, case["step"]
    eight = case["bits"] == 8
    m = _first_values(flat["first"], flat["first_scales"]) if eight else flat["first"]
    v = _second_values(flat["second"], flat["second_scales"]) if eight else flat["second"]
    g = flat["grads"].float() * state["grad_scale"]
    m = b1 * m + (1.0 - b1) * g
    v = b2 * v + (1.0 - b2) * (g * g)
    p = flat["master"] if case["master"] else flat["params"].float()
    p = p * (1.0 - _LR * _DECAY) - (_LR / (1.0 - b1**t)) * m / (torch.sqrt(v) * (1.0 / math.sqrt(1.0 - b2**t)) + _EPS)
    if case["master"]:
        flat["master"].copy_(p)
    flat["params"].copy_(p)
    if not eight:
        flat["first"].copy_(m)
        flat["second"].copy_(v)
        return {"params": flat["params"], "master": flat.get("master"), "first": flat["first"], "second": flat["second"]}
    noise = _noise(m.numel(), t, m.device)
    codes, scales = _first_codes(m, (noise & 0xFFFF).float() / 65536.0)
    flat["first"].copy_(codes)
    flat["first_scales"].copy_(scales)
    codes, scales = _second_codes(v, (noise >> 16).float() / 65536.0)
    flat["second"].copy_(codes)
    flat["second_scales"].copy_(scales)
    # The values that the codes stand for: they are exact in bfloat16.
    first, second = _first_values(flat["first"], flat["first_scales"]), _second_values(flat["second"], flat["second_scales"])
    return {"params": flat["params"], "master": flat.get("master"), "first": first.bfloat16(), "second": second.bfloat16()}


# ---- the definitions in 64 bits --------------------------------------------------------------------


def _exact_activation(g, activation):
    if activation == "silu":
        return g * torch.special.expit(g), torch.special.expit(g) + g * torch.special.expit(g) * torch.special.expit(-g)
    if activation == "gelu":
        cdf = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2.0 * math.pi)
    if activation == "relu":
        return torch.clamp(g, min=0.0), torch.where(g > 0, torch.ones_like(g), torch.zeros_like(g))
    # 0.5 (1 + tanh(z)) is the logistic function of 2 z.
    z = 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g**3)
    s = torch.special.expit(z)
    return g * s, s + g * s * torch.special.expit(-z) * (2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * g**2))


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "adamw":
        return _exact_adamw(state)
    x = state["x"].double()
    if kind == "weight_gradient":
        dw = x.t().contiguous() @ state["grad"].double()
        if case["layout"] == "nk":
            dw = dw.t()
        return dw if state["sum"] is None else dw + state["sum"].double()
    half, dtype = case["outputs"], state["x"].dtype
    gate, up = (w.double() for w in state["weight"].split(half, dim=1))
    outs, kept = {}, state.get("kept")
    if kind == "gated_backward" and kept is not None:
        g, u = kept[:, :half].double(), kept[:, half:].double()
    else:
        g, u = x @ gate, x @ up
    if kind != "gated_backward":
        outs["out"] = _exact_activation(g, case["activation"])[0] * u
        if case["keep"] if kind == "gated" else case["kept"]:
            outs["kept"] = torch.cat([g, u], dim=1)
            # What is kept is rounded once, and the backward pass starts from that.
            g, u = g.to(dtype).double(), u.to(dtype).double()
        else:
            outs["kept"] = None
    if kind != "gated":
        a, slope = _exact_activation(g, case["activation"])
        dg, du = state["grad"].double() * u * slope, state["grad"].double() * a
        outs["inner"] = torch.cat([dg, du], dim=1)
        # The products take the gradients as they are stored.
        dg, du = dg.to(dtype).double(), du.to(dtype).double()
        outs["dx"] = dg @ gate.t().contiguous() + du @ up.t().contiguous()
        dw = torch.cat([x.t() @ dg, x.t() @ du], dim=1)
        outs["dweight"] = dw if state["sum"] is None else dw + state["sum"].double()
    return outs


def _exact_held(y, power, bits, u):
    """``y`` between multiples of 2^(power - bits), the upper one where the fraction and u reach 1."""
    step = torch.exp2((power - bits).double())
    low = torch.floor(y / step)
    return (low + (y / step - low + u >= 1.0)) * step


def _exact_adamw(state):
    case, flat = state["case"], state["flat"]
    t = case["step"]
    if case["bits"] == 8:
        code = flat["first"].to(torch.int64)
        power, fraction = (code >> 3) & 15, (code & 7).double()
        m = torch.where(power > 0, (8.0 + fraction) * torch.exp2(power.double() - 10.0), fraction * 2.0**-9) * (1.0 - 2.0 * (code >> 7).double())
        m = m * torch.exp2(flat["first_scales"].double() - 127.0).repeat_interleave(_BLOCK)
        code = flat["second"].to(torch.int64)
        v = torch.where(code > 0, (8.0 + ((code + 7) & 7).double()) * torch.exp2(((code - 1) >> 3).double() - 33.0), torch.zeros_like(m))
        v = v * torch.exp2(flat["second_scales"].double() - 127.0).repeat_interleave(_BLOCK)
    else:
        m, v = flat["first"].double(), flat["second"].double()
    g = flat["grads"].double() * state["grad_scale"]
    m = m + (1.0 - _BETAS[0]) * (g - m)
    v = v + (1.0 - _BETAS[1]) * (g * g - v)
    p = (flat["master"] if case["master"] else flat["params"]).double()
    p = p - _LR * _DECAY * p - _LR * (m / (1.0 - _BETAS[0] ** t)) / ((v / (1.0 - _BETAS[1] ** t)).sqrt() + _EPS)
    if case["bits"] == 8:
        noise = _noise(m.numel(), t, m.device)
        amax = m.abs().view(-1, _BLOCK).amax(dim=1)
        e = torch.ceil(torch.log2(amax.clamp(min=2.0**-140) / 448.0))
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)  # a logarithm that was rounded
        e = torch.where(amax <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(min=-117).repeat_interleave(_BLOCK)
        y = m.abs() / torch.exp2(e)
        power = torch.clamp(_floor_log2(y), min=-6.0)
        m = torch.sign(m) * _exact_held(y, power, 3, (noise & 0xFFFF).double() / 65536.0) * torch.exp2(e)
        e = torch.clamp(_floor_log2(v.view(-1, _BLOCK).amax(dim=1)), -90, 127).repeat_interleave(_BLOCK)
        y = v / torch.exp2(e)
        held = torch.clamp(_exact_held(y, _floor_log2(y), 3, (noise >> 16).double() / 65536.0), min=2.0**-30)
        v = torch.where(v > 0, held, torch.zeros_like(held)) * torch.exp2(e)
    return {"params": p, "master": p if case["master"] else None, "first": m, "second": v}


def _floor_log2(y):
    power = torch.floor(torch.log2(y.clamp(min=2.0**-200)))
    power = torch.where(torch.exp2(power) > y, power - 1, power)  # a logarithm that was rounded
    return torch.where(torch.exp2(power + 1) <= y, power + 1, power)
