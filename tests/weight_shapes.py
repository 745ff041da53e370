"""Sizes of weight gradients by the kernel that takes them, shared by the CPU test of that choice and the GPU test of the kernels."""

import ctypes as C

# tokens, inputs, outputs -> edge of a tile, groups, splits, steps of a split (256 compute units)
CUTS = {
    (64, 8192, 4096): (256, 1, 1, 1),      # one step, two, four: fewer than the stages, and one more
    (128, 4096, 8192): (256, 1, 1, 2),
    (200, 8192, 4096): (256, 1, 1, 4),
    (700, 8000, 4000): (256, 1, 1, 11),    # tiles cut at both edges, and rows of tiles
    (1100, 4096, 4096): (256, 1, 1, 18),   # whole tiles only
    (8300, 4096, 4096): (256, 1, 1, 130),  # scales are read again behind 128 steps
    (9000, 2050, 2300): (256, 1, 3, 47),   # partial sums of three splits, which begin at odd steps
    (9000, 4096, 1100): (256, 1, 3, 47),
    (9000, 4104, 4090): (128, 1, 1, 141),  # the small tiles behind 128 steps
    (560000, 256, 256): (128, 2, 32, 274),  # two groups, each behind 128 steps
}


def cut(lib, shape, compute_units):
    got = [C.c_int32() for _ in range(4)]
    assert lib.tccl_weight_gradient_cut(*shape, compute_units, *map(C.byref, got)) == 0
    return tuple(v.value for v in got)
