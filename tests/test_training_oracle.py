"""What holds the 64-bit restatement of the training operators in place: closed forms, another library's cast, and
gradients against differences."""

import pytest
import torch

from oracle import training as ref


def test_e4m3_is_the_type_torch_has():
    g = torch.Generator().manual_seed(1)
    v = torch.cat([torch.randn(4000, generator=g) * 100, torch.randn(4000, generator=g) * 0.01, torch.tensor([448.0, 447.9, 2.0**-9, 2.0**-10, 3 * 2.0**-10, 0.0, 17.0, 19.0])])
    v = v.clamp(-448, 448)
    assert torch.equal(ref.e4m3(v.double()), v.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("top, e", [(448.0, 0), (448.0001, 1), (1.75, -8), (1.76, -7), (224.0, -1), (0.0, -117), (2.0**-130, -117), (65504.0, 8)])
def test_exponents_by_hand(top, e):
    x = torch.zeros(8, 128, dtype=torch.float64)
    x[3, 77] = -top
    assert ref.exponents(x).tolist() == [[e]]


def test_blocks_are_8_by_128_and_what_is_not_finite_has_no_part():
    x = torch.full((9, 129), 448.0)
    x[8, 128] = 2.0
    x[0, 0], x[0, 1] = float("inf"), float("nan")
    assert ref.exponents(x).tolist() == [[0, 0], [0, -7]]
    h = ref.held(x)
    assert torch.isnan(h[0, :2]).all() and torch.equal(h[0, 2:], x[0, 2:].double()) and h[8, 128] == 2.0


def test_held_values_are_within_half_a_spacing():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, 300, generator=g).bfloat16()
    err = (ref.held(x) - x.double()).abs()
    top = torch.ldexp(torch.ones(ref.exponents(x).shape, dtype=torch.float64), ref.exponents(x)).repeat_interleave(8, 0)[:40].repeat_interleave(128, 1)[:, :300]
    assert bool((err <= torch.maximum(x.double().abs() / 16, top * 2.0**-10)).all())


@pytest.mark.parametrize("dtype, most", [(torch.float16, 61440.0), (torch.bfloat16, 240.0 * 2.0**120)])
def test_the_largest_values_stay_finite(dtype, most):
    x = torch.full((1, 3), torch.finfo(dtype).max, dtype=dtype)
    x[0, 1] = -x[0, 1]
    x[0, 2] = 1.0
    assert ref.held(x)[0, :2].tolist() == [most, -most] and bool(torch.isfinite(ref.held(x).to(dtype)).all())


def test_norm_closed_form():
    out, mean, rstd = ref.layer_norm(torch.tensor([[1.0, 3.0], [5.0, 5.0]]), torch.tensor([2.0, 1.0]), torch.tensor([0.0, 10.0]), eps=0.25)
    assert mean.tolist() == [2.0, 5.0] and torch.allclose(rstd, torch.tensor([1.25**-0.5, 2.0], dtype=torch.float64))
    assert torch.allclose(out, torch.tensor([[-2.0 * 1.25**-0.5, 10.0 + 1.25**-0.5], [0.0, 10.0]], dtype=torch.float64))


@pytest.mark.parametrize("affine", [False, True])
def test_gradients_are_those_of_differences(affine):
    g = torch.Generator().manual_seed(3)
    s, dy, more = (torch.randn(3, 7, generator=g, dtype=torch.float64) for _ in range(3))
    w = torch.randn(7, generator=g, dtype=torch.float64) if affine else torch.ones(7, dtype=torch.float64)
    b = torch.randn(7, generator=g, dtype=torch.float64)
    _, mean, rstd = ref.layer_norm(s, w, b)
    dx, dw, db = ref.layer_norm_backward(dy, s, mean, rstd, w if affine else None, more)

    def loss(s, w, b):
        return float((ref.layer_norm(s, w, b)[0] * dy).sum() + (s * more).sum())

    for t, d in ((s, dx), (w, dw), (b, db)):
        for i in range(t.numel()):
            h = torch.zeros_like(t).reshape(-1)
            h[i] = 1e-6
            h = h.view_as(t)
            args = [(u + h, u - h) if u is t else (u, u) for u in (s, w, b)]
            slope = (loss(*(a[0] for a in args)) - loss(*(a[1] for a in args))) / 2e-6
            assert abs(slope - float(d.reshape(-1)[i])) < 1e-7 * (1 + abs(slope))


def test_weight_gradient_is_that_of_differences():
    g = torch.Generator().manual_seed(4)
    x, dy, w = torch.randn(5, 3, generator=g, dtype=torch.float64), torch.randn(5, 4, generator=g, dtype=torch.float64), torch.randn(3, 4, generator=g, dtype=torch.float64)
    dw = ref.weight_gradient(x, dy)
    for i in range(3):
        for j in range(4):
            h = torch.zeros(3, 4, dtype=torch.float64)
            h[i, j] = 0.5  # linear in w: the step does not matter
            assert abs(float((x @ (w + h) * dy).sum() - (x @ (w - h) * dy).sum()) - float(dw[i, j])) < 1e-12
