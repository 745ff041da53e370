"""The weight gradient's large tiles, and the small ones over many steps, against the definition in 64 bits.

Every block of 8 x 128 has a scale of its own, neighbours' up to 2^10 apart.  The 64-bit products run on the GPU (one matrix
product of float64 tensors); the bounds are ``check_weight``'s of ``test_gpu_training.py``: products are exact in fp32, and at most
tokens / 8 + 64 additions meet in one sum, each off by a spacing at most."""

import pytest
import torch

from tests.test_gpu_training import BF16, F16, F32, half
from tests.weight_shapes import CUTS, cut
from tileccl_amd import _lib, ops

pytestmark = pytest.mark.gpu

# shape, type, result, layout, add
CASES = [
    ((64, 8192, 4096), BF16, F32, "kn", True), ((64, 8192, 4096), F16, F16, "nk", False),
    ((128, 4096, 8192), F16, F32, "nk", True), ((128, 4096, 8192), BF16, BF16, "kn", True),
    ((200, 8192, 4096), F16, F32, "kn", False), ((200, 8192, 4096), BF16, F32, "nk", True),
    ((700, 8000, 4000), BF16, F32, "kn", True), ((700, 8000, 4000), F16, F32, "nk", True),
    ((700, 8000, 4000), F16, F16, "kn", True), ((700, 8000, 4000), BF16, BF16, "nk", False),
    ((1100, 4096, 4096), BF16, F32, "kn", True), ((1100, 4096, 4096), F16, F32, "nk", True), ((1100, 4096, 4096), F16, F32, "kn", False),
    ((8300, 4096, 4096), BF16, F32, "kn", True), ((8300, 4096, 4096), F16, F16, "nk", True),
    ((9000, 2050, 2300), BF16, F32, "nk", True), ((9000, 2050, 2300), F16, F16, "kn", True), ((9000, 4096, 1100), BF16, BF16, "kn", False),
    ((9000, 4104, 4090), BF16, F32, "kn", True), ((9000, 4104, 4090), F16, F32, "nk", False), ((560000, 256, 256), F16, F32, "kn", True),
]


def device_units(lib):
    import ctypes as C

    info = _lib.DeviceInfo()
    _lib.check(lib.tccl_device_query(-1, C.byref(info)), "tccl_device_query")
    return info.compute_units


def on_gpu(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def test_cases_reach_every_kernel():
    assert {c[0] for c in CASES} == set(CUTS)


@pytest.mark.parametrize("shape, dtype, result, layout, add", CASES)
def test_tiles(lib, shape, dtype, result, layout, add):
    units = device_units(lib)
    if units == 256:
        assert cut(lib, shape, units) == CUTS[shape]
    rows, cols, outputs = shape
    x, dy = on_gpu((rows, cols), 1, dtype), on_gpu((rows, outputs), 2, dtype, 0.1)
    x *= torch.exp2(((torch.arange(rows, device="cuda") // 8)[:, None] * 7 + (torch.arange(cols, device="cuda") // 128)[None] * 3) % 11 - 5).to(dtype)
    held = ops.checkpoint_activation(x)
    values, grad = ops.restore_activation(held).double(), dy.double()
    earlier = on_gpu((cols, outputs), 3, result, 4.0) if add else None
    want, size = values.t() @ grad, values.abs().t() @ grad.abs()
    if add:
        want, size = want + earlier.double(), size + earlier.double().abs()
    chain = (rows / 8 + 64) * 2.0**-23 * size
    bound = half((want.abs() + chain).cpu(), result).cuda() + chain
    given = None if earlier is None else (earlier if layout == "kn" else earlier.t()).contiguous()
    w = ops.weight_gradient(held, dy, layout=layout, out_dtype=result, add=given)
    off = ((w if layout == "kn" else w.t()).double() - want).abs() - bound
    assert bool((off <= 0).all()), f"off by {float(off.max()):.3g} more than its bound, at {int(off.argmax())}"
    assert torch.equal(ops.weight_gradient(held, dy, layout=layout, out_dtype=result, add=given), w), "the same inputs gave other bits"
    if add:
        there = ops.weight_gradient(held, dy, layout=layout, add=given, out=given)
        assert there is given and torch.equal(given, w)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("pitch, offset", [(4100, 0), (4099, 0), (4096, 1)])
def test_large_tiles_on_top_of_a_sum_of_any_pitch_and_start(lib, layout, pitch, offset):
    """Rows of the sum and the result on 16 bytes (through LDS) and off them."""
    rows, cols, outputs = 1100, 4096, 4096
    x, dy = on_gpu((rows, cols), 1, BF16), on_gpu((rows, outputs), 2, BF16, 0.1)
    held = ops.checkpoint_activation(x)
    memory = torch.full((cols * pitch + 64,), float("nan"), device="cuda")
    given = memory[offset:].as_strided((cols, outputs), (pitch, 1))
    given.copy_(on_gpu((cols, outputs), 3, F32))
    want = ops.weight_gradient(held, dy, layout=layout).double() + given.double()
    got = ops.weight_gradient(held, dy, layout=layout, add=given, out=given)
    # The sum without it is stored as it was accumulated: one addition more, rounded once.
    assert got is given and bool(((given.double() - want).abs() <= 2.0**-24 * want.abs()).all())
    outside = torch.ones_like(memory, dtype=torch.bool)
    outside[offset:].as_strided((cols, outputs), (pitch, 1)).fill_(False)
    assert bool(torch.isnan(memory[outside]).all()), "written outside the rows"
