"""CPU restatement of the training operators in 64 bits (test infrastructure only).

Each function is the operator's definition, written with elementary operations on float64 tensors; nothing here is
shared with the package.  The reference has no counterpart of these operators.
"""

from __future__ import annotations

import torch

ROWS, COLS, LOWEST = 8, 128, -117  # a block of the 8-bit layout; the lowest exponent of a scale


def exponents(x: torch.Tensor) -> torch.Tensor:
    """int64 (row blocks, column blocks): the smallest e >= -117 with max|x| <= 448 * 2**e over a block's finite values."""
    rows, cols = x.shape
    out = torch.empty(-(-rows // ROWS), -(-cols // COLS), dtype=torch.int64)
    for i in range(out.shape[0]):
        for j in range(out.shape[1]):
            block = x[i * ROWS:(i + 1) * ROWS, j * COLS:(j + 1) * COLS].double()
            finite = block[torch.isfinite(block)].abs()
            top = finite.max().item() if finite.numel() else 0.0
            e = LOWEST
            while top > 448.0 * 2.0**e:
                e += 1
            out[i, j] = e
    return out


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value of each element (ties to even), by its spacing; |v| <= 448."""
    _, power = torch.frexp(v.abs().clamp(min=2.0**-40))  # v in [2**(power - 1), 2**power)
    spacing = torch.ldexp(torch.ones_like(v), torch.clamp(power - 1, min=-6) - 3)
    return torch.round(v / spacing) * spacing


def held(x: torch.Tensor) -> torch.Tensor:
    """The values that the 8-bit checkpoint of ``x`` stands for (float64)."""
    e = exponents(x)
    scale = torch.ldexp(torch.ones(e.shape, dtype=torch.float64), e)
    scale = scale.repeat_interleave(ROWS, 0)[: x.shape[0]].repeat_interleave(COLS, 1)[:, : x.shape[1]]
    v = x.double()
    finite = torch.isfinite(v)
    q = e4m3(torch.where(finite, v, 0.0) / scale)
    # Rounded past the largest value of the type: the e4m3 below (240 is the neighbour of 256).
    q = torch.where((q * scale).abs() > torch.finfo(x.dtype).max, q.sign() * 240.0, q)
    return torch.where(finite, q * scale, float("nan"))


def layer_norm(s: torch.Tensor, weight=None, bias=None, eps: float = 1e-5):
    """(out, mean, rstd) in float64 of the norm's input ``s``."""
    s = s.double()
    mean = s.sum(1) / s.shape[1]
    centred = s - mean[:, None]
    rstd = 1.0 / torch.sqrt((centred * centred).sum(1) / s.shape[1] + eps)
    out = centred * rstd[:, None]
    if weight is not None:
        out = out * weight.double()
    if bias is not None:
        out = out + bias.double()
    return out, mean, rstd


def layer_norm_backward(grad, s, mean, rstd, weight=None, grad_summed=None):
    """(dx, dweight, dbias) in float64 by the formula, with the given statistics."""
    dy, s, mean, rstd = grad.double(), s.double(), mean.double(), rstd.double()
    normed = (s - mean[:, None]) * rstd[:, None]
    g = dy if weight is None else dy * weight.double()
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - normed * (g * normed).mean(1, keepdim=True))
    if grad_summed is not None:
        dx = dx + grad_summed.double()
    return dx, (dy * normed).sum(0), dy.sum(0)


def weight_gradient(x: torch.Tensor, grad: torch.Tensor, add=None) -> torch.Tensor:
    """(columns, outputs) in float64 from the values that are held."""
    w = x.double().t() @ grad.double()
    return w if add is None else w + add.double()
