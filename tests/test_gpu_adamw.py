"""AdamW on the GPU against its definition in 64 bits.

fp32 roundings are 2^-24 of a value each.  m: two products, a sum, the scaled gradient and two constants: 6 roundings of
|b1 m| + |(1 - b1) g|.  v likewise, 8.  The step lr / c1 * m / (sqrt(v / c2) + eps): 20 roundings of it (the reciprocal is good to one unit,
constants are rounded once, m and v as above), and p's own: 4 of |p|.
Held in 8 bits a value is one of the two around it, which one is known but where the fraction and u meet 1 within the fp32 error of
the value, in steps: 2^-24 * 8 * 16 is less than 2^-16.
"""

import pytest
import torch

from oracle import layers as ref
from tests.layer_bounds import BF16, F16, F32, rand, rounded, within
from tileccl_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0**-24
HOW = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
TYPES = [(F32, F32, False), (BF16, F32, True), (BF16, BF16, True), (F16, F32, False), (F16, F16, True), (BF16, BF16, False)]


def flat_of(tensors, state, dtype=torch.float64):
    """Tensors as they lie in flat memory, zeros between them."""
    at = ops.AdamWState.offsets(state.sizes)
    out = torch.zeros(at[-1], dtype=dtype)
    for t, start, n in zip(tensors, at, state.sizes):
        out[start:start + n] = t.detach().reshape(-1).cpu().to(dtype)
    return out


def used(state):
    return flat_of([torch.ones(n) for n in state.sizes], state).bool()


def check_step(params, grads, state, before, want_m, want_v, want_p, grad_scale, how):
    """Everything but the held moments: ``before`` is (p, m, v) in 64 bits."""
    p0, m0, v0 = before
    g = (flat_of(grads, state) * grad_scale).abs()
    b1, b2 = how["betas"]
    mask = used(state)
    step = (want_p - p0 * (1 - how["lr"] * how["weight_decay"])).abs()
    error = 4 * U * p0.abs() + 24 * U * step
    # the step follows errors of m and of sqrt(v): relative to them
    m_error, v_error = 6 * U * (b1 * m0.abs() + (1 - b1) * g), 8 * U * (b2 * v0 + (1 - b2) * g * g)
    error = error + torch.where(want_m != 0, step * m_error / want_m.abs().clamp(min=1e-300), 0.0)
    master = state.master
    if master is not None:
        within(master.cpu()[mask], want_p[mask], (error + 2.0**-149)[mask], "master")
    dtype = params[0].dtype
    got = flat_of(params, state, torch.float64)
    within(got[mask], want_p[mask], rounded(want_p, error, dtype)[mask] if dtype != F32 else (error + 2.0**-149)[mask], "params")
    if master is not None:
        assert torch.equal(flat_of(params, state, dtype)[mask], master.cpu().to(dtype)[mask]), "params are the master's rounded values"
    return mask, m_error, v_error


SIZES = [(1,), (7, 128), (129,), (64, 2), (4096,), (5000,), (3, 5, 7), (12288,), (20001,), (8,)]


def make(types, sizes, bits, seed, scale=1.0):
    p_type, g_type, master = types
    params = [rand(s, seed + i, p_type, 0.5).cuda() for i, s in enumerate(sizes)]
    grads = [rand(s, seed + 100 + i, F32, 0.1 * (1 + i % 4)).mul(scale).to(g_type).cuda() for i, s in enumerate(sizes)]
    return params, grads, ops.AdamWState.zeros(params, bits=bits, master=master)


@pytest.mark.parametrize("types", TYPES)
def test_three_steps_in_32_bits(types):
    params, grads, state = make(types, SIZES, 32, 1)
    for step in (1, 2, 3):
        p0 = state.master.cpu().double() if state.master is not None else flat_of(params, state)
        before = p0, state.first.cpu().double(), state.second.cpu().double()
        g = flat_of(grads, state)
        want_p, want_m, want_v = ref.adamw(p0, g, *before[1:], step=step, grad_scale=0.25, **HOW)
        ops.adamw_step(params, grads, state, step=step, grad_scale=0.25, **HOW)
        mask, m_error, v_error = check_step(params, grads, state, before, want_m, want_v, want_p, 0.25, HOW)
        within(state.first, want_m, m_error, "first")
        within(state.second, want_v, v_error, "second")
        assert not state.first.cpu()[~mask].any() and not state.second.cpu()[~mask].any()


def check_held(codes, scales, y, u, table, exponent, lowest, name, mask):
    """Every block's scale and every code, from the exact values ``y`` and the random numbers ``u``."""
    n = y.numel() // ref.BLOCK
    y, u = y.view(n, ref.BLOCK), u.view(n, ref.BLOCK)
    got = ref.values(codes, scales, table).view(n, ref.BLOCK)
    mask = mask.view(n, ref.BLOCK)
    for b in range(n):
        fine = y[b][torch.isfinite(y[b])].abs()
        top = float(fine.max()) if fine.numel() else 0.0
        e = int(scales[b]) - 127
        assert e in {exponent(top * (1 - 16 * U)), exponent(top * (1 + 16 * U))}, f"{name}: scale of block {b}"
        z = y[b].abs() / 2.0**e
        low, high = ref.neighbours(z, table)
        low = torch.where(z > 0, low.clamp(min=lowest), low)
        high = torch.maximum(high, low)
        f = torch.where(high > low, (z - low) / (high - low).clamp(min=1e-300), 0.0) + u[b]
        want = torch.where(f >= 1, high, low) * torch.sign(y[b])
        have = got[b] / 2.0**e
        close = (f - 1).abs() < 2.0**-16
        # a value of which z is within rounding of being one of the codes may have that one, too
        near = ((z - low).abs() < 16 * U * z) & (have.abs() == low) | ((z - high).abs() < 16 * U * z) & (have.abs() == high)
        ok = (have == want) | (close & ((have.abs() == low) | (have.abs() == high))) | near | ~torch.isfinite(y[b]) & torch.isnan(have)
        assert bool(ok[mask[b]].all()), f"{name}: block {b}, element {int((~ok & mask[b]).nonzero()[0])}"
        assert not bool(got[b][~mask[b]].any())


@pytest.mark.parametrize("types", TYPES)
def test_three_steps_in_8_bits(types):
    sizes = [(1,), (130,), (3, 100), (5000,), (17,)]
    params, grads, state = make(types, sizes, 8, 2)
    # magnitudes over many octaves within a block; nothing at all in a part of one
    grads[3].mul_(torch.exp2(torch.linspace(-14, 2, 5000, device="cuda")).to(grads[3].dtype))
    grads[3][1000:1300] = 0.0
    for step in (1, 2, 30):
        p0 = state.master.cpu().double() if state.master is not None else flat_of(params, state)
        m0 = ref.values(state.first.cpu(), state.first_scales.cpu(), ref.FIRST)
        v0 = ref.values(state.second.cpu(), state.second_scales.cpu(), ref.SECOND)
        want_p, want_m, want_v = ref.adamw(p0, flat_of(grads, state), m0, v0, step=step, grad_scale=1.0, **HOW)
        ops.adamw_step(params, grads, state, step=step, **HOW)
        mask, _, _ = check_step(params, grads, state, (p0, m0, v0), want_m, want_v, want_p, 1.0, HOW)
        um, uv = ref.uniforms(want_m.numel(), step)
        check_held(state.first.cpu(), state.first_scales.cpu(), want_m, um, ref.FIRST, ref.first_exponent, 0.0, "first", mask)
        check_held(state.second.cpu(), state.second_scales.cpu(), want_v, uv, ref.SECOND, ref.second_exponent, 2.0**-30, "second", mask)
        first, second = ops.adamw_moments(state)
        assert first.dtype == second.dtype == BF16
        assert torch.equal(first.cpu().double(), ref.values(state.first.cpu(), state.first_scales.cpu(), ref.FIRST))
        assert torch.equal(second.cpu().double(), ref.values(state.second.cpu(), state.second_scales.cpu(), ref.SECOND))


def test_held_moments_are_right_on_average():
    """Constant gradients: after many steps m is g and v is g * g, also where a step moves v by a hundredth of what is between two codes."""
    n = 1 << 14
    g = torch.full((n,), 0.25, device="cuda")
    p = torch.zeros(n, device="cuda")
    state = ops.AdamWState.zeros([p], bits=8)
    b2 = 0.99
    for step in range(1, 401):
        ops.adamw_step([p], [g], state, step=step, lr=0.0, betas=(0.9, b2), weight_decay=0.0)
    first, second = (t.double() for t in ops.adamw_moments(state))
    # v's spread: a step's variance is at most 0.01 of v times an eighth of it, and 50 of them add up: 0.0625 v^2; the mean of 16384
    # independent elements is within 6 * 0.25 / 128 of it, and 1 - b2^400 = 0.982.
    assert abs(float(second.mean()) / 0.0625 - 0.982) < 6 * 0.25 / 128
    assert abs(float(first.mean()) / 0.25 - 1) < 6 * 0.25 / 128


def test_many_tensors_take_several_launches():
    sizes = [(1 + 37 * i % 400,) for i in range(230)]
    params, grads, state = make((F32, F32, False), sizes, 32, 3)
    p0 = flat_of(params, state)
    want_p, want_m, want_v = ref.adamw(p0, flat_of(grads, state), torch.zeros_like(p0), torch.zeros_like(p0), step=1, grad_scale=1.0, **HOW)
    ops.adamw_step(params, grads, state, step=1, **HOW)
    check_step(params, grads, state, (p0, torch.zeros_like(p0), torch.zeros_like(p0)), want_m, want_v, want_p, 1.0, HOW)
    assert all(p._version == 1 for p in params)


def test_no_tensors_and_empty_ones():
    ops.adamw_step([], [], ops.AdamWState.zeros([]), step=1)
    empty = torch.empty(0, 5, device="cuda")
    p, g = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    state = ops.AdamWState.zeros([empty, p, empty])
    ops.adamw_step([empty, p, empty], [empty, g, empty], state, step=1, lr=0.5, weight_decay=0.0)
    assert torch.allclose(p, torch.full_like(p, 0.5))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_anywhere(bits):
    """Addresses of no particular alignment, and nothing beside them written."""
    memory = torch.full((4001,), 7.0, dtype=BF16, device="cuda")
    grads_at = rand((4001,), 5, BF16).cuda()
    spans = [(1, 700), (705, 300), (1400, 1), (1403, 2001)]
    params, grads = [memory[a:a + n] for a, n in spans], [grads_at[a + 1:a + 1 + n] for a, n in spans]
    state = ops.AdamWState.zeros(params, bits=bits, master=True)
    ops.adamw_step(params, grads, state, step=1, lr=0.5, weight_decay=0.0)
    for (a, n), g in zip(spans, grads):
        want = 7.0 - 0.5 * torch.sign(g.float())
        assert torch.equal(memory[a:a + n].float(), want.to(BF16).float())
        memory[a:a + n] = 7.0
    assert bool((memory == 7.0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite(bits):
    p = torch.ones(300, device="cuda")
    g = torch.full((300,), 0.5, device="cuda")
    g[3], g[200] = float("nan"), float("inf")
    state = ops.AdamWState.zeros([p], bits=bits)
    ops.adamw_step([p], [g], state, step=1)
    bad = torch.isnan(p).nonzero().flatten().tolist()
    assert bad == [3, 200]
    first, second = ops.adamw_moments(state)
    if bits == 8:
        assert torch.isnan(first).nonzero().flatten().tolist() == [3, 200] == torch.isnan(second).nonzero().flatten().tolist()
        fine = torch.ones(384, dtype=torch.bool, device="cuda")
        fine[3] = fine[200] = False
        assert bool((first[:300][fine[:300]] > 0.04).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_steps_count_on(bits):
    """step, lr and grad_scale as device words: a graph's replays are the eager steps of the same numbers."""
    sizes = [(1000,), (333,), (64, 65)]
    params, grads, state = make((BF16, F32, True), sizes, bits, 7)
    other, _, other_state = make((BF16, F32, True), sizes, bits, 7)
    step, lr, scale = torch.ones(1, dtype=torch.int32, device="cuda"), torch.full((1,), 1e-2, device="cuda"), torch.full((), 0.5, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adamw_step(params, grads, state, step=step, lr=lr, grad_scale=scale, weight_decay=0.1)
        step.add_(1)
    for k in range(1, 5):
        lr.fill_(1e-2 / k)
        graph.replay()
        torch.cuda.synchronize()
        assert int(step) == k + 1
        ops.adamw_step(other, grads, other_state, step=k, lr=float(lr), grad_scale=0.5, weight_decay=0.1)
        # the constants of a step are made in 64 bits here and in 32 there: 4 roundings of a step of at most lr * 4
        near = (state.master - other_state.master).abs()
        assert float(near.max()) <= k * 2.0**-20 * 1e-2 * 4 + 2.0**-22
        if bits == 32:
            assert torch.equal(state.first, other_state.first) and torch.equal(state.second, other_state.second)
        else:
            assert torch.equal(state.first, other_state.first) and torch.equal(state.second_scales, other_state.second_scales)
        for mine, theirs in zip(state[:5], other_state[:5]):
            if mine is not None:
                theirs.copy_(mine)
        for mine, theirs in zip(params, other):
            theirs.copy_(mine)


def test_another_stream():
    params, grads, state = make((F32, F32, False), [(70000,), (3,)], 8, 9)
    same, _, same_state = make((F32, F32, False), [(70000,), (3,)], 8, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.adamw_step(params, grads, state, step=5)
    torch.cuda.current_stream().wait_stream(side)
    ops.adamw_step(same, grads, same_state, step=5)
    assert all(torch.equal(a, b) for a, b in zip(params, same)) and all(torch.equal(a, b) for a, b in zip(state[:4], same_state[:4]))
