"""What the tests of the gated layer, of the weight gradient from an input in full and of AdamW measure with.

Sums of n products.  A product of two 16-bit values is exact in fp32, and whatever the order of the additions, each of them
(an MFMA's own may cut off instead of rounding) is off by at most 2^-23 of a partial sum, which is at most the sum S of the
magnitudes: n 2^-23 S in all.

Activations.  |act'| <= 1.13 and |act''| <= 1.2 for every one of them but relu's jump (gelu: 1.129 and 0.798, silu 1.10 and 0.5,
gelu_tanh 1.129 and 0.80), so an error of g reaches act(g) and act'(g) at most so large.  Their own fp32 evaluation: an exponential whose
argument has a rounding of |arg| 2^-24 next to a handful of other roundings; g times what is off by |g| s(g) 2^-22 has a maximum of
g^2 s(g) <= 0.54 at that, so 2^-20 (|g| + 1) covers act, 2^-19 covers act' (its terms are at most 1.2 and g s(-g) <= 0.28).
"""

import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
BITS = {BF16: 8, F16: 11, F32: 24}                  # of the significand
LOWEST = {BF16: -126, F16: -14, F32: -126}          # exponent of the smallest normal value


def rand(shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def placed(t, pitch=None, offset=0):
    """``t`` on the GPU with rows of ``pitch`` elements, ``offset`` elements behind an allocation's start; NaN around it."""
    rows, cols = t.shape
    pitch = cols if pitch is None else pitch
    memory = torch.full((rows * pitch + offset + 64,), float("nan"), dtype=t.dtype, device="cuda")
    view = memory[offset:].as_strided((rows, cols), (pitch, 1))
    view.copy_(t)
    return view


def half(size, dtype):
    """Half the spacing of ``dtype`` at values up to ``size`` (in [2^(k-1), 2^k) neighbours are 2^(k - bits) apart)."""
    _, k = torch.frexp(size.double())
    return torch.ldexp(torch.ones_like(size, dtype=torch.float64), torch.clamp(k, min=LOWEST[dtype] + 1) - BITS[dtype] - 1)


def rounded(want, error, dtype):
    """The bound of a value that is off by ``error`` and then rounded once."""
    return error + half(want.abs() + error, dtype)


def within(got, want, bound, name):
    got, want = got.detach().cpu().double(), want.double()
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{name}: NaN where there is none, or none where there is"
    off = torch.where(nan | (got == want), 0.0, (got - want).abs() - bound.nan_to_num(0.0))
    assert bool((off <= 0).all()), f"{name}: off by {float(off.max()):.3g} more than its bound, at {int(off.argmax())} of {tuple(off.shape)}"


SUM = 2.0**-23


def gated_bounds(g, u, s, k, dtype, name):
    """(out, its bound) from the 64-bit projections and the sums of magnitudes ``s`` over ``k`` products."""
    from oracle import layers as ref

    n = g.shape[1]
    eg, eu = k * SUM * s[:, :n], k * SUM * s[:, n:]
    a, _ = ref.activation(g, name)
    error = (1.13 * eg + 2.0**-20 * (g.abs() + 1)) * (u.abs() + eu) + a.abs() * eu
    return a * u, rounded(a * u, error, dtype)


def inner_bounds(dh, g, u, eg, eu, dtype, name):
    """(inner, its bound) from projections that are off by at most ``eg`` and ``eu``."""
    from oracle import layers as ref

    a, slope = ref.activation(g.double(), name)
    dh, u = dh.double(), u.double()
    want = torch.cat([dh * u * slope, dh * a], dim=1)
    dg = dh.abs() * ((slope.abs() + 1.2 * eg + 2.0**-19) * eu + u.abs() * (1.2 * eg + 2.0**-19))
    du = dh.abs() * (1.13 * eg + 2.0**-20 * (g.double().abs() + 1))
    error = torch.cat([dg, du], dim=1) + 2.0**-22 * want.abs()
    return want, rounded(want, error, dtype)
