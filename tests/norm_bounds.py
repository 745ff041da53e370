"""How far a layer norm in 32 bits may be from its definition, by the magnitudes of each row.

E = 32 * 2^-24 covers a chain of fp32 operations: sums are trees over a thread's vectors, lanes and wavefronts of fewer than 30
levels, with a handful of products around them.  For a row s with largest magnitude t and variance v:

* the mean is off by E t;
* each wavefront sums squares around its own mean, and the wavefronts' means are off by E t, their distances from the row's (whose
  squares sum up to no more than v) by 2 E t: v is off by E v + 4 E t sqrt(v) + 4 (E t)^2.  A difference of sums would be off by
  E t^2;
* rstd is off by what that makes of 1 / sqrt(v + eps), and E of itself;
* out is off by the error of the mean and of rstd in (s - mean) rstd, and E of itself and the bias, before it is rounded.

The backward pass is given mean and rstd: (s - mean) rstd is off by a few roundings of itself, whatever the mean."""

import torch

from oracle import training as ref

E = 32 * 2.0**-24
BITS = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}
LOWEST = {torch.bfloat16: -126, torch.float16: -14, torch.float32: -126}


def half(size, dtype):
    """Half the spacing of ``dtype`` at values up to ``size``."""
    _, k = torch.frexp(size.double())
    return torch.ldexp(torch.ones_like(size, dtype=torch.float64), torch.clamp(k, min=LOWEST[dtype] + 1) - BITS[dtype] - 1)


def within(got, want, bound, name):
    got = got.detach().cpu()
    # A value beyond the output's type is an infinity of its sign (16-bit gradients of a constant row whose 8-bit values are not).
    top = torch.finfo(got.dtype).max
    beyond = (want.abs() + bound > top) & torch.isinf(got) & (got.sign() == want.sign())
    off = torch.where(beyond, 0.0, (got.double() - want).abs() - bound)
    assert bool((off <= 0).all()), f"{name}: off by {float(off.max()):.3g} more than its bound, at {int(off.argmax())}"


def forward(out, mean, rstd, s, weight, bias, eps=1e-5):
    want, m, r = ref.layer_norm(s, weight, bias, eps)
    top, v = s.double().abs().amax(1), 1 / r**2 - eps
    v = v.clamp(min=0.0)
    off_v = E * v + 4 * E * top * v.sqrt() + 4 * (E * top) ** 2
    most, least = ((v - off_v).clamp(min=0.0) + eps) ** -0.5, (v + off_v + eps) ** -0.5
    off_r = torch.maximum(most - r, r - least) + E * most
    within(mean, m, E * top, "mean")
    within(rstd, r, off_r, "rstd")
    w, b = weight.double().abs(), bias.double().abs()
    centred = (s.double() - m[:, None]).abs()
    chain = w * ((E * top * most)[:, None] + centred * off_r[:, None] + E * centred * r[:, None]) + E * (want.abs() + b)
    within(out, want, half(want.abs() + chain, s.dtype) + chain, "out")


def backward(dx, dweight, dbias, dy, s, mean, rstd, weight, dtype):
    mean, rstd = mean.cpu(), rstd.cpu()
    want, dw, db = ref.layer_norm_backward(dy, s, mean, rstd, weight)
    normed = (s.double() - mean.double()[:, None]) * rstd.double()[:, None]
    g = dy.double() * weight.double()
    parts = g.abs() + g.abs().mean(1, keepdim=True) + normed.abs() * (g * normed).abs().mean(1, keepdim=True)
    chain = 2 * E * rstd.double()[:, None] * parts
    within(dx, want, half(want.abs() + chain, dtype) + chain, "dx")
    more = 1 + dy.shape[0] / 1024  # rows that a thread adds up one after the other: 32 of 1024
    within(dweight, dw, more * E * (dy.double() * normed).abs().sum(0), "dweight")
    within(dbias, db, more * E * dy.double().abs().sum(0), "dbias")


def rows_with_means(rows, cols, dtype, seed):
    """Rows by turns around 0, with means far larger than their spread (as far as ``dtype`` can hold the spread), with one wide
    step, and constant."""
    g = torch.Generator().manual_seed(seed)
    far = {torch.float32: 4096.0, torch.float16: 64.0, torch.bfloat16: 8.0}[dtype]
    s = torch.randn(rows, cols, generator=g)
    s[1::5] += far
    s[2::5] = 1000.0 * s[2::5] - 200.0 * far
    s[3::5, cols // 2:] += far / 4
    s[4::5] = 100.0
    return s.to(dtype)
