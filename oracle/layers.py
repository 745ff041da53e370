"""CPU restatement of the gated linear layer and of AdamW in 64 bits (test infrastructure only).

Each function is the operator's definition, written with elementary operations on float64 tensors; nothing here is
shared with the package.  The reference has no counterpart of these operators.
"""

from __future__ import annotations

import math

import torch

BLOCK = 128  # moments that share a scale


def activation(g: torch.Tensor, name: str) -> tuple[torch.Tensor, torch.Tensor]:
    """(act(g), act'(g)) of a float64 tensor."""
    if name == "silu":
        s = torch.special.expit(g)
        return g * s, s + g * s * torch.special.expit(-g)
    if name == "gelu":
        cdf = torch.special.erfc(-g / math.sqrt(2.0)) / 2
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        z = math.sqrt(2.0 / math.pi) * (g + 0.044715 * g**3)
        t = torch.tanh(z)
        return g * (1 + t) / 2, (1 + t) / 2 + g / 2 * (1 - t * t) * math.sqrt(2.0 / math.pi) * (1 + 3 * 0.044715 * g * g)
    assert name == "relu"
    return torch.clamp(g, min=0.0), (g > 0).double()


def projections(x: torch.Tensor, weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """g and u of ``x @ weight`` and, of the same shape as that, the sums of the products' magnitudes."""
    x, weight = x.double(), weight.double()
    z = x @ weight
    half = weight.shape[1] // 2
    return z[:, :half], z[:, half:], x.abs() @ weight.abs()


def gated_gradient(dh: torch.Tensor, g: torch.Tensor, u: torch.Tensor, name: str) -> torch.Tensor:
    a, slope = activation(g.double(), name)
    dh = dh.double()
    return torch.cat([dh * u.double() * slope, dh * a], dim=1)


# ---- AdamW ----------------------------------------------------------------------------------------


def adamw(p, g, m, v, *, step, lr, betas, eps, weight_decay, grad_scale):
    """(p, m, v) behind a step, all float64."""
    b1, b2 = betas
    p, g, m, v = p.double(), g.double() * grad_scale, m.double(), v.double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * weight_decay) - lr * (m / (1 - b1**step)) / ((v / (1 - b2**step)).sqrt() + eps), m, v


def noise(place: int, step: int) -> int:
    """The 32 random bits of an element and a step, with whole numbers of any size."""
    most = 2**32 - 1
    h = (place & most) ^ ((step * 0x9E3779B9 + (place >> 32) * 0xBB67AE85) & most)
    h = (h ^ (h >> 16)) * 0x6A09E667 & most
    h = (h ^ (h >> 15)) * 0x3C6EF373 & most
    return h ^ (h >> 16)


def uniforms(total: int, step: int) -> tuple[torch.Tensor, torch.Tensor]:
    """What the first and the second moment of every place are rounded with, in [0, 1)."""
    h = [noise(i, step) for i in range(total)]
    return torch.tensor([x & 0xFFFF for x in h], dtype=torch.float64) / 65536, torch.tensor([x >> 16 for x in h], dtype=torch.float64) / 65536


def first_value(code: int) -> float:
    """An e4m3 code's value."""
    power, fraction = code >> 3 & 15, code & 7
    v = (8 + fraction) * 2.0 ** (power - 10) if power else fraction * 2.0**-9
    v = math.nan if code & 127 == 127 else v
    return -v if code & 128 else v


def second_value(code: int) -> float:
    if code in (0, 255):
        return math.nan if code else 0.0
    return (1 + (code - 1) % 8 / 8) * 2.0 ** ((code - 1) // 8 - 30)


FIRST = torch.tensor([first_value(c) for c in range(256)], dtype=torch.float64)
SECOND = torch.tensor([second_value(c) for c in range(256)], dtype=torch.float64)


def values(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """What flat codes stand for."""
    n = codes.numel() // BLOCK
    return (table[codes.long()].view(n, BLOCK) * torch.exp2(scales[:n].double() - 127)[:, None]).view(-1)


def first_exponent(top: float) -> int:
    e = -117
    while top > 448 * 2.0**e:
        e += 1
    return e


def second_exponent(top: float) -> int:
    return min(127, max(-90, math.frexp(top)[1] - 1)) if top else -90


def neighbours(y: torch.Tensor, table: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The held magnitudes on either side of ``y`` (the same one twice where y is one; ``y`` at most the largest)."""
    grid = torch.unique(table[torch.isfinite(table)].abs())
    at = torch.searchsorted(grid, y, right=True) - 1
    low = grid[at.clamp(min=0)]
    return low, torch.where(low == y, low, grid[(at + 1).clamp(max=len(grid) - 1)])
