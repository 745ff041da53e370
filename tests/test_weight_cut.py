"""How the weight gradient is cut into tiles and splits, on the host."""

import ctypes as C
import random

import pytest

from tests.weight_shapes import CUTS, cut
from tileccl_amd import _lib


@pytest.mark.parametrize("shape", CUTS)
def test_the_tested_shapes_reach_the_kernels_that_they_are_for(lib, shape):
    assert cut(lib, shape, 256) == CUTS[shape]


def test_every_cut_covers_the_rows(lib):
    rng = random.Random(3)
    seen = set()
    for _ in range(2000):
        shape = tuple(int(2 ** rng.uniform(0, top)) for top in (16, 14, 14))
        edge, groups, splits, steps = cut(lib, shape, rng.choice((64, 256, 304)))
        total = -(-shape[0] // 64)
        assert (edge, groups) in ((256, 1), (128, 1), (128, 2))
        assert splits * steps >= total > (splits - 1) * steps, "a split without rows, or rows without a split"
        seen.add((edge, groups, splits > 1))
    assert len(seen) == 6


def test_no_rows_is_one_split_without_steps(lib):
    assert cut(lib, (0, 100, 100), 256)[2:] == (1, 0)


def test_refusals(lib):
    out = [C.c_int32() for _ in range(4)]
    assert lib.tccl_weight_gradient_cut(1, 1, 1, 0, *map(C.byref, out)) == _lib.ERR_INVALID
    assert lib.tccl_weight_gradient_cut(1, 1, 1, 256, *map(C.byref, out[:3]), None) == _lib.ERR_INVALID
    assert lib.tccl_weight_gradient_cut(1, 0, 1, 256, *map(C.byref, out)) == _lib.ERR_INVALID
