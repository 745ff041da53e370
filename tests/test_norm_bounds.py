"""That the bounds of ``norm_bounds.py`` tell a sound norm in 32 bits from others."""

import pytest
import torch

from oracle import training as ref
from tests import norm_bounds

F32 = torch.float32


def inputs(cols=1003):
    s = norm_bounds.rows_with_means(40, cols, F32, 1)
    g = torch.Generator().manual_seed(2)
    return s, 1 + 0.2 * torch.randn(cols, generator=g), 0.3 * torch.randn(cols, generator=g), torch.randn(40, cols, generator=g)


def two_passes(s, w, b, eps=1e-5):
    mean = s.mean(1)
    centred = s - mean[:, None]
    rstd = ((centred * centred).mean(1) + eps).rsqrt()
    return centred * rstd[:, None] * w + b, mean, rstd


def one_pass(s, w, b, eps=1e-5):
    mean = s.mean(1)
    rstd = (((s * s).mean(1) - mean * mean).clamp(min=0.0) + eps).rsqrt()
    return (s - mean[:, None]) * rstd[:, None] * w + b, mean, rstd


@pytest.mark.parametrize("cols", [7, 300, 1003, 20000])
def test_squares_around_the_mean_are_taken(cols):
    s, w, b, _ = inputs(cols)
    norm_bounds.forward(*two_passes(s, w, b), s, w, b)


@pytest.mark.parametrize("cols", [300, 1003, 20000])
def test_a_difference_of_sums_is_not(cols):
    s, w, b, _ = inputs(cols)
    out, mean, rstd = one_pass(s, w, b)
    far = slice(1, None, 5)
    with pytest.raises(AssertionError, match="rstd"):
        norm_bounds.forward(out[far], mean[far], rstd[far], s[far], w, b)
    good = two_passes(s, w, b)
    with pytest.raises(AssertionError, match="out"):
        norm_bounds.forward(out[far], good[1][far], good[2][far], s[far], w, b)


@pytest.mark.parametrize("row", range(5))
def test_zeros_and_wrong_statistics_are_not(row):
    s, w, b, dy = inputs()
    out, mean, rstd = two_passes(s, w, b)
    some = slice(row, None, 5)
    s, dy, out, mean, rstd = s[some], dy[some], out[some], mean[some], rstd[some]
    norm_bounds.forward(out, mean, rstd, s, w, b)
    for got in ((out, mean, 0 * rstd), (out, mean + 1e-2 * s.abs().amax(1), rstd), (out, mean, 2 * rstd), (out + 1.0, mean, rstd)):
        with pytest.raises(AssertionError):
            norm_bounds.forward(*got, s, w, b)
    dx, dw, db = (t.float() for t in ref.layer_norm_backward(dy, s, mean, rstd, w))
    norm_bounds.backward(dx, dw, db, dy, s, mean, rstd, w, F32)
    for got in ((0 * dx, dw, db), (dx, dw + 1.0, db), (dx, dw, 0 * db), (dx + 1e-3 * rstd[:, None], dw, db)):
        with pytest.raises(AssertionError):
            norm_bounds.backward(*got, dy, s, mean, rstd, w, F32)


def test_infinities_stand_for_what_the_type_cannot_hold():
    got, want = torch.tensor([float("inf"), -float("inf"), 1.0]).half(), torch.tensor([7e4, -1e9, 1.0], dtype=torch.float64)
    norm_bounds.within(got, want, torch.tensor(32.0), "x")
    for other in ((-got, want), (got, torch.tensor([6e4, -1e9, 1.0], dtype=torch.float64)), (torch.tensor([65504.0, -65504.0, 1.0]).half(), want)):
        with pytest.raises(AssertionError):
            norm_bounds.within(*other, torch.tensor(32.0), "x")
