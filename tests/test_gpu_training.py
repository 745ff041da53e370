"""Layer norm, activations in 8 bits and weight gradients on the GPU against their definitions in 64 bits.

Tolerances.  half() is half a spacing of the output's type at a value: what one rounding costs.
E = 64 * 2^-24 covers every chain of fp32 operations here: sums are trees of at most 24 levels over lanes, wavefronts and
vectors, with a handful of products and a reciprocal root around them.  What E multiplies is a bound on the magnitudes that
enter: for (s - mean) * rstd that is max|s| * rstd over the row, since the error of the mean is relative to the values.
"""

import pytest
import torch

from oracle import training as ref
from tileccl_amd import _launch, ops

pytestmark = pytest.mark.gpu

BITS = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}  # of the significand
LOWEST = {torch.bfloat16: -126, torch.float16: -14, torch.float32: -126}  # exponent of the smallest normal value
E = 64 * 2.0**-24
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rand(shape, seed, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def placed(t, pitch=None, offset=0):
    """``t`` on the GPU with rows of ``pitch`` elements, ``offset`` elements behind an allocation's start; NaN around it."""
    rows, cols = t.shape
    pitch = cols if pitch is None else pitch
    memory = torch.full((rows * pitch + offset + 64,), float("nan"), dtype=t.dtype, device="cuda")
    view = memory[offset:].as_strided((rows, cols), (pitch, 1))
    view.copy_(t)
    return view


def within(got, want, bound, name):
    got, want, bound = got.detach().cpu().double(), want.double(), torch.as_tensor(bound, dtype=torch.float64)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{name}: NaN where there is none, or none where there is"
    off = torch.where(nan, 0.0, (got - want).abs()) - bound.expand_as(want).nan_to_num(0.0)
    assert bool((off <= 0).all()), f"{name}: off by {float(off.max()):.3g} more than its bound, at {int(off.argmax())}"


def half(size, dtype):
    """Half the spacing of ``dtype`` at values up to ``size`` (in [2^(k-1), 2^k) neighbours are 2^(k - bits) apart)."""
    _, k = torch.frexp(size.double())
    return torch.ldexp(torch.ones_like(size, dtype=torch.float64), torch.clamp(k, min=LOWEST[dtype] + 1) - BITS[dtype] - 1)


def check_forward(r, s, weight, bias, eps=1e-5):
    out, mean, rstd = ref.layer_norm(s, weight, bias, eps)
    top = s.double().abs().amax(1)
    within(r.mean, mean, E * top, "mean")
    within(r.rstd, rstd, E * rstd * (1 + (top * rstd) ** 2), "rstd")
    w = torch.ones(s.shape[1], dtype=torch.float64) if weight is None else weight.double().abs()
    b = torch.zeros_like(w) if bias is None else bias.double().abs()
    chain = E * (((top * rstd) * (1 + (top * rstd) ** 2) + 1)[:, None] * w + b)
    within(r.out, out, half(out.abs() + chain, s.dtype) + chain, "out")


def check_backward(d, dy, s, mean, rstd, weight, more):
    """``mean``, ``rstd``: what the operator was given; ``s``: the values it was given (a checkpoint's, if that)."""
    mean, rstd = mean.cpu(), rstd.cpu()
    dx, dw, db = ref.layer_norm_backward(dy, s, mean, rstd, weight, more)
    top = (s.double().abs().amax(1) * rstd.double().abs()).clamp(min=1.0)  # of (s - mean) * rstd and its parts
    w = torch.ones(s.shape[1], dtype=torch.float64) if weight is None else weight.double().abs()
    g = (dy.double().abs() * w).amax(1)
    chain = E * 4 * rstd.double() * g * (1 + top * top) + E * (0 if more is None else more.double().abs().amax(1))
    within(d.x, dx, half(dx.abs() + chain[:, None], dy.dtype) + chain[:, None], "dx")
    if d.weight is not None:
        within(d.weight, dw, E * 4 * (dy.double().abs() * top[:, None]).sum(0), "dweight")
        within(d.bias, db, E * dy.double().abs().sum(0), "dbias")


FORWARD = [
    # rows, cols, type, affine, residual: one token, one column, around vectors, wavefronts, row groups and blocks
    (1, 4096, BF16, "same", True), (1, 1, F32, None, False), (3, 1, F16, "f32", True), (5, 7, BF16, "same", False),
    (2, 8, F16, "same", True), (9, 9, F32, "f32", True), (64, 127, BF16, "f32", True), (65, 128, F16, "same", False),
    (63, 129, BF16, "same", True), (17, 511, F32, "f32", False), (33, 512, BF16, "same", True), (300, 513, F16, "f32", True),
    (1000, 1003, BF16, "f32", True), (2100, 264, F16, "same", False), (4100, 72, BF16, "same", True), (7, 4097, F16, "same", True),
    (130, 8192, BF16, "same", False), (5, 8193, BF16, "f32", True), (3, 16384, F16, "same", True), (3, 16390, BF16, "same", False),
    (2, 32768, BF16, "f32", True), (2, 32765, F32, "f32", True), (1200, 2048, F32, "f32", False), (6000, 1536, BF16, "same", True),
]


WITH_AND_WITHOUT_8_BITS = [(*c, held) for held in (False, True) for c in FORWARD if not held or c[2] != F32]


@pytest.mark.parametrize("rows, cols, dtype, affine, residual, checkpoint", WITH_AND_WITHOUT_8_BITS)
def test_forward(lib, rows, cols, dtype, affine, residual, checkpoint):
    x, more = rand((rows, cols), 1, dtype, 2.0, 0.5), rand((rows, cols), 2, dtype) if residual else None
    at = F32 if affine == "f32" else dtype
    weight, bias = (None, None) if affine is None else (rand((cols,), 3, at, 0.2, 1.0), rand((cols,), 4, at, 0.3))
    r = ops.layer_norm(x.cuda(), None if weight is None else weight.cuda(), None if bias is None else bias.cuda(),
                       residual=None if more is None else more.cuda(), checkpoint=checkpoint)
    s = x if more is None else (x.float() + more.float()).to(dtype)
    if residual:
        assert torch.equal(r.summed.cpu(), s)
    else:
        assert r.summed is None
    check_forward(r, s, weight, bias)
    if checkpoint:
        assert torch.equal(ops.restore_activation(r.checkpoint).cpu().double(), ref.held(s))
    else:
        assert r.checkpoint is None


@pytest.mark.parametrize("rows, cols, pitches, offset", [(37, 1000, (1003, 1001, 1009), 1), (37, 1003, (1003, 1008, 1016), 3), (8, 520, (528, 1040, 520), 0), (600, 64, (67, 65, 71), 5)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rows_of_any_pitch_and_start(lib, rows, cols, pitches, offset, dtype):
    x, more, w, b = rand((rows, cols), 1, dtype), rand((rows, cols), 2, dtype), rand((cols,), 3, dtype), rand((cols,), 4, dtype)
    s = (x.float() + more.float()).to(dtype)
    out = placed(torch.zeros(rows, cols, dtype=dtype), pitches[2], offset)
    r = ops.layer_norm(placed(x, pitches[0], offset), w.cuda(), b.cuda(), residual=placed(more, pitches[1], offset), out=out, checkpoint=dtype != F32)
    assert r.out is out
    check_forward(r, s, w, b)
    full = out.as_strided(((rows - 1) * pitches[2] + cols + offset + 64,), (1,), 0).cpu()
    outside = torch.ones_like(full, dtype=torch.bool)
    outside.as_strided((rows, cols), (pitches[2], 1), offset).fill_(False)
    assert bool(torch.isnan(full[outside]).all()), "written outside the rows"
    dy = rand((rows, cols), 5, dtype)
    dx = placed(torch.zeros(rows, cols, dtype=dtype), pitches[1], offset)
    for held in (placed(s, pitches[2], offset), r.checkpoint):
        if held is None:
            continue
        d = ops.layer_norm_backward(placed(dy, pitches[0], offset), held, r.mean, r.rstd, w.cuda(), grad_summed=placed(more, pitches[1], offset), out=dx)
        check_backward(d, dy, s if isinstance(held, torch.Tensor) else ref.held(s), r.mean, r.rstd, w, more)
    if dtype != F32:
        held = ops.checkpoint_activation(placed(x, pitches[0], offset))
        back = ops.restore_activation(held, out=placed(torch.zeros(rows, cols, dtype=dtype), pitches[1], offset))
        assert torch.equal(back.cpu().double(), ref.held(x))


@pytest.mark.parametrize("rows, cols, dtype, affine, more, held", WITH_AND_WITHOUT_8_BITS)
def test_backward(lib, rows, cols, dtype, affine, more, held):
    s, dy = rand((rows, cols), 1, dtype, 2.0, 0.5), rand((rows, cols), 2, dtype, 0.1)
    more = rand((rows, cols), 3, dtype, 0.1) if more else None
    at = F32 if affine == "f32" else dtype
    weight = None if affine is None else rand((cols,), 4, at, 0.2, 1.0)
    _, mean, rstd = ref.layer_norm(s)
    mean, rstd = mean.float().cuda(), rstd.float().cuda()
    x = ops.checkpoint_activation(s.cuda()) if held else s.cuda()
    args = (dy.cuda(), x, mean, rstd, None if weight is None else weight.cuda())
    d = ops.layer_norm_backward(*args, grad_summed=None if more is None else more.cuda())
    check_backward(d, dy, ref.held(s) if held else s, mean, rstd, weight, more)
    again = ops.layer_norm_backward(*args, grad_summed=None if more is None else more.cuda())
    assert all(torch.equal(a, b) for a, b in zip(d, again)), "the same inputs gave other bits"
    only = ops.layer_norm_backward(*args, grad_summed=None if more is None else more.cuda(), affine=False)
    assert torch.equal(only.x, d.x) and only.weight is None and only.bias is None


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows, cols", [(1025, 5), (1030, 100), (9000, 1003), (5001, 2052), (3000, 4096), (1100, 4100), (2500, 6001), (1027, 8190), (1026, 8200), (1100, 16383), (1030, 16400)])
def test_backward_of_many_rows(lib, rows, cols, dtype):
    """Workgroups that take several groups of rows, with rows that end inside a vector; dx in the place of either gradient."""
    s, dy, more = rand((rows, cols), 1, dtype, 2.0, 0.5), rand((rows, cols), 2, dtype, 0.1), rand((rows, cols), 3, dtype, 0.1)
    weight = rand((cols,), 4, dtype, 0.2, 1.0)
    _, mean, rstd = ref.layer_norm(s)
    mean, rstd = mean.float().cuda(), rstd.float().cuda()
    d = ops.layer_norm_backward(dy.cuda(), s.cuda(), mean, rstd, weight.cuda(), grad_summed=more.cuda())
    check_backward(d, dy, s, mean, rstd, weight, more)
    for place in (0, 1):
        g, m = dy.cuda(), more.cuda()
        there = ops.layer_norm_backward(g, s.cuda(), mean, rstd, weight.cuda(), grad_summed=m, out=(g, m)[place])
        assert torch.equal(there.x, d.x) and torch.equal(there.weight, d.weight) and torch.equal(there.bias, d.bias)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows, cols", [(1025, 5), (1027, 100), (1030, 4096), (9001, 1003), (5006, 2052), (2500, 4100)])
def test_backward_of_many_rows_from_8_bits(lib, rows, cols, dtype):
    """Blocks with scales of their own, the last of them cut in its first or second half."""
    s, dy, more = rand((rows, cols), 1, dtype, 0.1, 0.1), rand((rows, cols), 2, dtype, 0.1), rand((rows, cols), 3, dtype, 0.1)
    s *= torch.exp2(((torch.arange(rows) // 8)[:, None] * 7 + (torch.arange(cols) // 128)[None] * 3) % 5).to(dtype)
    _, mean, rstd = ref.layer_norm(s)
    mean, rstd = mean.float().cuda(), rstd.float().cuda()
    held = ops.checkpoint_activation(s.cuda())
    d = ops.layer_norm_backward(dy.cuda(), held, mean, rstd, grad_summed=more.cuda())
    check_backward(d, dy, ref.held(s), mean, rstd, None, more)
    m = more.cuda()
    there = ops.layer_norm_backward(dy.cuda(), held, mean, rstd, grad_summed=m, out=m)
    assert torch.equal(there.x, d.x) and torch.equal(there.weight, d.weight) and torch.equal(there.bias, d.bias)


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("rows, cols", [(16, 16384), (60, 12001), (250, 2056), (257, 2056), (1000, 260), (1024, 9)])
def test_sums_of_few_rows(lib, rows, cols, held):
    """Column sums by workgroups of their own: wide and narrow ones, one pass over the rows and several, part of a vector at the end."""
    s, dy = rand((rows, cols), 1, BF16, 2.0, 0.5), rand((rows, cols), 2, BF16, 0.1)
    _, mean, rstd = ref.layer_norm(s)
    mean, rstd = mean.float().cuda(), rstd.float().cuda()
    x = ops.checkpoint_activation(s.cuda()) if held else s.cuda()
    check_backward(ops.layer_norm_backward(dy.cuda(), x, mean, rstd), dy, ref.held(s) if held else s, mean, rstd, None, None)


def test_backward_against_differences(lib):
    """The gradients of the forward kernel itself, in fp32: its outputs are some 1e-7 of themselves off, so differences
    over steps of 2^-6 are about 2^6 * 48 * 4e-7 = 1.3e-3 off, and the terms of second order in the step 2^-12 * 10 = 2.5e-3."""
    s, dy, w, b = rand((2, 24), 1), rand((2, 24), 2), rand((24,), 3, F32, 0.2, 1.0).cuda(), rand((24,), 4).cuda()
    r = ops.layer_norm(s.cuda(), w, b)
    d = ops.layer_norm_backward(dy.cuda(), s.cuda(), r.mean, r.rstd, w)

    def loss(x):
        return float((ops.layer_norm(x.cuda(), w, b).out.double().cpu() * dy.double()).sum())

    for i in range(48):
        h = torch.zeros(48)
        h[i] = 2.0**-6
        h = h.view(2, 24)
        slope = (loss(s + h) - loss(s - h)) / 2.0**-5
        assert abs(slope - float(d.x.reshape(-1)[i])) < 4e-3


def test_rows_that_are_constant_large_or_not_finite(lib):
    x = rand((12, 300), 1)
    x[0] = 0.0
    x[1] = 1000.0
    x[2] += 1000.0            # a mean a thousand times the spread
    x[3] *= 1e18              # squares that overflow
    x[4] *= 1e-20
    x[5, 17] = float("nan")
    x[6, 299] = float("inf")
    x[7, 0] = -float("inf")
    r = ops.layer_norm(x.cuda())
    good = [0, 1, 2, 4, 8, 9, 10, 11]
    check_forward(type(r)(r.out[good], r.mean[good], r.rstd[good], None, None), x[good], None, None)
    assert bool(torch.isnan(r.out[5:8]).all()) and bool(torch.isfinite(r.out[good]).all())
    dy = rand((12, 300), 2)
    d = ops.layer_norm_backward(dy.cuda(), x.cuda(), r.mean, r.rstd)
    check_backward(type(d)(d.x[good], None, None), dy[good], x[good], r.mean[good], r.rstd[good], None, None)
    assert bool(torch.isnan(d.x[5:8]).all()) and bool(torch.isnan(d.weight).all()) and bool(torch.isfinite(d.bias).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows, cols", [(1, 1), (8, 128), (7, 127), (9, 129), (64, 513), (1003, 1000), (16, 2049), (3, 40000)])
def test_checkpoint_bytes(lib, rows, cols, dtype):
    """Codes and scales, bit for bit, with every kind of block: empty, tiny, huge, spread over the whole range."""
    x = rand((rows, cols), 5, F32)
    x *= torch.exp2(torch.randint(-30, 12, (-(-rows // 8), -(-cols // 128)), generator=torch.Generator().manual_seed(6)).float()).repeat_interleave(8, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    x = x.to(dtype)
    if rows >= 16 and cols >= 257:
        x[:8, :128] = 0
        x[8:16, :128] = torch.finfo(dtype).max
        x[:8, 128:256] = torch.finfo(dtype).smallest_normal
        x[8:16, 128:256] = rand((8, 128), 7, F32, 1.0).sign().to(dtype) * 2.0**-24
        x[0, 256], x[1, 256], x[2, 256] = float("nan"), float("inf"), -float("inf")
    held = ops.checkpoint_activation(x.cuda())
    e = ref.exponents(x)
    assert torch.equal(held.scales[:, : e.shape[0]].cpu().long(), e.t() + 127)
    values = held.values.cpu().view(torch.float8_e4m3fn).double()  # row block, column, row
    assert bool((values.transpose(1, 2).reshape(-1, values.shape[1])[rows:] == 0).all()) and bool((values[:, cols:] == 0).all())
    want = ref.held(x)
    back = ops.restore_activation(held).cpu().double()
    assert torch.equal(torch.isnan(back), torch.isnan(want)) and torch.equal(back.nan_to_num(0.0), want.nan_to_num(0.0))


GRADIENT = [
    # tokens, inputs, outputs, type, result, layout, add
    (1, 1, 1, BF16, F32, "kn", False), (1, 128, 8, F16, F16, "nk", True), (8, 64, 16, BF16, BF16, "kn", True), (63, 129, 130, F16, F32, "nk", False),
    (64, 128, 128, BF16, F32, "kn", False), (65, 127, 136, BF16, BF16, "nk", True), (200, 300, 257, F16, F16, "kn", False), (1003, 1000, 2064, BF16, BF16, "nk", False),
    (4096, 136, 72, F16, F32, "kn", True), (5000, 100, 100, BF16, F32, "nk", True), (129, 4096, 264, F16, F32, "nk", False), (512, 512, 256, F16, F16, "kn", True),
    (700, 2500, 2600, BF16, F32, "kn", True), (700, 2600, 2504, F16, F16, "nk", True), (320, 4104, 1300, BF16, F32, "nk", False),
]


def check_weight(w, held, dy, add, dtype):
    """Products of an e4m3 and a 16-bit value are exact in fp32; at most tokens / 8 + 64 additions meet in one sum (a
    matrix instruction takes 32 tokens, the splits are added one by one), each off by a spacing at most."""
    want, size = ref.weight_gradient(held, dy, add), ref.weight_gradient(held.abs(), dy.abs())
    if add is not None:
        size = size + add.double().abs()
    chain = (dy.shape[0] / 8 + 64) * 2.0**-23 * size
    within(w, want, half(want.abs() + chain, dtype) + chain, "weight gradient")


@pytest.mark.parametrize("rows, cols, outputs, dtype, result, layout, add", GRADIENT)
def test_weight_gradient(lib, rows, cols, outputs, dtype, result, layout, add):
    x, dy = rand((rows, cols), 1, dtype), rand((rows, outputs), 2, dtype, 0.1)
    held = ops.checkpoint_activation(x.cuda())
    earlier = rand((cols, outputs), 3, result) if add else None
    given = None if earlier is None else (earlier if layout == "kn" else earlier.t()).contiguous().cuda()
    w = ops.weight_gradient(held, dy.cuda(), layout=layout, out_dtype=result, add=given)
    assert w.dtype == result and tuple(w.shape) == ((cols, outputs) if layout == "kn" else (outputs, cols))
    check_weight(w if layout == "kn" else w.t(), ref.held(x), dy, earlier, result)
    again = ops.weight_gradient(held, dy.cuda(), layout=layout, out_dtype=result, add=given)
    assert torch.equal(w, again), "the same inputs gave other bits"
    if given is not None:
        there = ops.weight_gradient(held, dy.cuda(), layout=layout, out_dtype=result, add=given, out=given)
        assert there is given and torch.equal(given, w)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("pitch, offset, out_pitch", [(264, 8, 263), (257, 0, 300), (262, 3, 261)])
def test_weight_gradient_of_any_pitch_and_start(lib, layout, pitch, offset, out_pitch):
    rows, cols, outputs = 150, 260, 256
    x, dy = rand((rows, cols), 1, BF16), rand((rows, outputs), 2, BF16)
    held = ops.checkpoint_activation(x.cuda())
    shape = (cols, outputs) if layout == "kn" else (outputs, cols)
    out = placed(torch.zeros(shape), max(out_pitch, shape[1]), offset)
    ops.weight_gradient(held, placed(dy, pitch, offset), layout=layout, out=out)
    check_weight(out if layout == "kn" else out.t(), ref.held(x), dy, None, F32)


@pytest.mark.parametrize("rows, cols, outputs", [(100, 128, 64), (190, 256, 136), (1090, 64, 264), (9000, 64, 64), (9000, 512, 384)])
def test_weight_gradient_of_blocks_with_scales_of_their_own(lib, rows, cols, outputs):
    """Neighbouring blocks' scales differ by up to 2^10; the tokens are cut at odd and even steps of 64."""
    x, dy = rand((rows, cols), 1, BF16), rand((rows, outputs), 2, BF16)
    x *= torch.exp2(((torch.arange(rows) // 8)[:, None] * 7 + (torch.arange(cols) // 128)[None] * 3) % 11 - 5).to(BF16)
    held = ops.checkpoint_activation(x.cuda())
    check_weight(ops.weight_gradient(held, dy.cuda()), ref.held(x), dy, None, F32)


@pytest.mark.parametrize("rows, cols, outputs", [(1, 8192, 8192), (65, 8192, 264), (100, 8192, 264), (100, 264, 8192)])
def test_weight_gradient_of_fewer_steps_than_stages(lib, rows, cols, outputs):
    """Few tokens of wide layers: what the pipeline would load next, and the last scales of a cut at an odd step, lie behind the operands."""
    x, dy = rand((rows, cols), 1, BF16), rand((rows, outputs), 2, BF16)
    held = ops.checkpoint_activation(x.cuda())
    check_weight(ops.weight_gradient(held, dy.cuda()), ref.held(x), dy, None, F32)


def test_what_is_not_finite_stays_in_its_row_and_column(lib):
    """NaN and infinities beside and behind the operands (the memory around them is NaN) and in them."""
    rows, cols, outputs = 100, 200, 136
    x, dy = rand((rows, cols), 1, BF16), rand((rows, outputs), 2, BF16)
    x[99, 199] = float("nan")
    dy[7, 5] = float("inf")
    w = ops.weight_gradient(ops.checkpoint_activation(placed(x, 208)), placed(dy, 144)).cpu()
    bad = torch.zeros(cols, outputs, dtype=torch.bool)
    bad[199], bad[:, 5] = True, True
    assert bool((~torch.isfinite(w[bad])).all()) and bool(torch.isfinite(w[~bad]).all())


def test_no_rows(lib):
    x = torch.empty(0, 96, dtype=BF16, device="cuda")
    r = ops.layer_norm(x, checkpoint=True)
    assert r.out.shape == (0, 96) and r.mean.shape == (0,)
    for held in (x, r.checkpoint):
        d = ops.layer_norm_backward(x, held, r.mean, r.rstd)
        assert d.x.shape == (0, 96) and not d.weight.any() and not d.bias.any()
    assert ops.restore_activation(ops.checkpoint_activation(x)).shape == (0, 96)
    dy, add = torch.empty(0, 40, dtype=BF16, device="cuda"), rand((96, 40), 1).cuda()
    assert not ops.weight_gradient(r.checkpoint, dy).any()
    assert torch.equal(ops.weight_gradient(r.checkpoint, dy, add=add), add)


def test_in_place(lib):
    x, more, w = rand((50, 300), 1, BF16).cuda(), rand((50, 300), 2, BF16).cuda(), rand((300,), 3, BF16).cuda()
    want = ops.layer_norm(x, w, residual=more)
    for name in ("x", "residual"):
        a, b = x.clone(), more.clone()
        assert torch.equal(ops.layer_norm(a, w, residual=b, out=a if name == "x" else b).out, want.out)
    d = ops.layer_norm_backward(x, want.summed, want.mean, want.rstd, w, grad_summed=more)
    for name in ("grad", "summed"):
        a, b = x.clone(), more.clone()
        assert torch.equal(ops.layer_norm_backward(a, want.summed, want.mean, want.rstd, w, grad_summed=b, out=a if name == "grad" else b).x, d.x)


def test_refusals(lib):
    x = torch.zeros(16, 64, dtype=BF16, device="cuda")
    mean = torch.zeros(16, device="cuda")
    held = ops.checkpoint_activation(x)
    cases = [
        ("contiguous rows", lambda: ops.layer_norm(x.t())),
        ("has no columns", lambda: ops.layer_norm(x[:, :0])),
        ("rows overlap", lambda: ops.layer_norm(x.as_strided((16, 64), (32, 1)))),
        ("must be float16, bfloat16 or float32", lambda: ops.layer_norm(x.double())),
        ("weight must be a contiguous vector of 64", lambda: ops.layer_norm(x, mean)),
        ("weight must be a contiguous vector of 64", lambda: ops.layer_norm(x, torch.ones(64, dtype=F16, device="cuda"))),
        ("share one dtype", lambda: ops.layer_norm(x, torch.ones(64, device="cuda"), torch.ones(64, dtype=BF16, device="cuda"))),
        ("residual must have shape", lambda: ops.layer_norm(x, residual=x[:8])),
        ("residual must have dtype", lambda: ops.layer_norm(x, residual=x.half())),
        ("out overlaps an input", lambda: ops.layer_norm(x[:8], out=x.view(-1)[32:544].view(8, 64))),
        ("a checkpoint holds", lambda: ops.layer_norm(x.float(), checkpoint=True)),
        ("at most 32768", lambda: ops.layer_norm(torch.zeros(1, 32769, dtype=F16, device="cuda"))),
        ("x must have shape", lambda: ops.layer_norm_backward(x, x[:8], mean, mean)),
        ("the checkpoint is of", lambda: ops.layer_norm_backward(x.half(), held, mean, mean)),
        ("mean must be a contiguous vector of 16", lambda: ops.layer_norm_backward(x, x, mean[:8], mean)),
        ("rstd must be a contiguous vector of 16", lambda: ops.layer_norm_backward(x, x, mean, mean.double())),
        ("x must be float16 or bfloat16", lambda: ops.checkpoint_activation(x.float())),
        ("out must have shape", lambda: ops.restore_activation(held, out=x[:8])),
        ("contiguous uint8 of shape", lambda: ops.restore_activation(ops.ActivationCheckpoint(held.values[:1], held.scales, 16, 64, BF16))),
        ("layout must be", lambda: ops.weight_gradient(held, x, layout="mn")),
        ("the checkpoint is of", lambda: ops.weight_gradient(held, x[:8])),
        ("the checkpoint is of", lambda: ops.weight_gradient(held, x.half())),
        ("the result must be", lambda: ops.weight_gradient(held, x, out_dtype=F16)),
        ("add must have shape", lambda: ops.weight_gradient(held, x, add=mean.view(1, 16))),
        ("add must have dtype", lambda: ops.weight_gradient(held, x, add=torch.zeros(64, 64, device="cuda"), out=torch.zeros(64, 64, dtype=BF16, device="cuda"))),
        ("the result must be", lambda: ops.weight_gradient(held, x, out=torch.zeros(64, 64, device="cuda").double())),
    ]
    for text, call in cases:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(ValueError, match="workspace has"):
        from tileccl_amd import _lib
        import ctypes as C

        d = _lib.NormGradDesc(grad=x.data_ptr(), x=x.data_ptr(), dx=x.data_ptr(), mean=mean.data_ptr(), rstd=mean.data_ptr(), ld_grad=64, ld_x=64, ld_dx=64, rows=16, cols=64,
                              dtype=_lib.BF16, affine_dtype=_lib.BF16)
        _lib.check(lib.tccl_layer_norm_grad(C.byref(d), None), "tccl_layer_norm_grad")


def step(x, more, w, b, dy, dz):
    r = ops.layer_norm(x, w, b, residual=more, checkpoint=True)
    kept = ops.checkpoint_activation(r.out)
    d = ops.layer_norm_backward(dy, r.checkpoint, r.mean, r.rstd, w, grad_summed=more)
    return (r.out, r.mean, r.rstd, r.summed, r.checkpoint.values, d.x, d.weight, d.bias, ops.restore_activation(kept), ops.weight_gradient(kept, dz), ops.weight_gradient(kept, dz[:, :100].contiguous(), layout="nk"))


def inputs(seed):
    return [rand((1000, 520), seed, BF16).cuda(), rand((1000, 520), seed + 1, BF16).cuda(), rand((520,), seed + 2, BF16).cuda(), rand((520,), seed + 3, BF16).cuda(),
            rand((1000, 520), seed + 4, BF16).cuda(), rand((1000, 264), seed + 5, BF16).cuda()]


def test_on_another_stream(lib):
    args = inputs(1)
    want = step(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step(*args)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_recorded_into_a_graph(lib):
    """Replays with other inputs in the same memory, eager work between them, each against the eager result."""
    args = inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step(*args)
    for seed in (11, 21, 31):
        for a, b in zip(args, inputs(seed)):
            a.copy_(b)
        want = [t.clone() for t in step(*args)]
        for t in recorded:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(recorded, want):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(lib):
    """More than 4 GiB of activations, and of their 8-bit values; the last rows against the definition."""
    rows, cols, last = 140_001, 32768, 9
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    tail = rand((last, cols), 1, BF16)
    x[-last:] = tail.cuda()
    held = ops.checkpoint_activation(x)
    back = ops.restore_activation(held)
    start = (rows - last) // 8 * 8  # the first row of the block that the tail begins in
    want = ref.held(torch.cat([torch.zeros(rows - last - start, cols, dtype=BF16), tail]))[rows - last - start:]
    assert torch.equal(back[-last:].cpu().double(), want) and not back[: rows - last].any()
    del back
    r = ops.layer_norm(x, out=x)
    check_forward(type(r)(r.out[-last:], r.mean[-last:], r.rstd[-last:], None, None), tail, None, None)
    dy = rand((last, cols), 2, BF16, 0.1)
    x.zero_()
    x[-last:] = dy.cuda()
    d = ops.layer_norm_backward(x, held, r.mean, r.rstd, out=x)
    check_backward(type(d)(d.x[-last:], d.weight, d.bias), dy, want, r.mean[-last:], r.rstd[-last:], None, None)
    del x, d, held
    rows, cols, outputs = 270_000, 72, 8200
    x, dy = torch.zeros(rows, cols, dtype=BF16, device="cuda"), torch.zeros(rows, outputs, dtype=BF16, device="cuda")
    x[-last:], dy[-last:] = rand((last, cols), 3, BF16).cuda(), rand((last, outputs), 4, BF16).cuda()
    x[0], dy[0] = 1.0, 2.0
    held = ops.checkpoint_activation(x)
    few = ops.restore_activation(held)[-last:].cpu().double()
    w = ops.weight_gradient(held, dy).cpu().double()
    want = ref.weight_gradient(few, dy[-last:].cpu()) + 2.0
    size = ref.weight_gradient(few.abs(), dy[-last:].cpu().abs()) + 2.0
    assert bool(((w - want).abs() <= 64 * 2.0**-23 * size).all())


def test_tensors_on_a_heap(lib):
    from tileccl_amd import v2

    heaps = v2.SymmetricHeap.create_all(16 << 20, 2)
    try:
        x = rand((64, 256), 1, F16)
        a, out = heaps[1].allocate_tensor((64, 256), F16), heaps[1].allocate_tensor((64, 256), F16)
        a.copy_(x)
        check_forward(ops.layer_norm(a, out=out), x, None, None)
    finally:
        for h in heaps:
            h.cleanup()
