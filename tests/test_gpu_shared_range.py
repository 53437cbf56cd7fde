"""Decode attention over shared prefixes where sizes are extreme: scores next to 0 or past f32's
range, values that are all zeros or far smaller than others."""
from __future__ import annotations

import math

import numpy as np
import pytest

from test_gpu_shared import Batch

pytestmark = pytest.mark.gpu

SHAPES = [([200], [[40, 0, 3]], 16, 8, 128), ([100, 30], [[70], [1]], 8, 4, 64)]


@pytest.mark.parametrize("q_scale,k_scale", [(0.0, 1.0), (0.0, 1e-8), (0.0, 1e-30), (1e-20, 1e-20),
                                             (1e-37, 1e-30), (1e-30, 1e-37)])
@pytest.mark.parametrize("shape", SHAPES)
def test_scores_next_to_zero(shape, q_scale, k_scale, rng):
    """Weights that are all the same, of key counts that fill no tile: the mean of the values."""
    Batch(rng, *shape, q_scale=q_scale, k_scale=k_scale).check()


@pytest.mark.parametrize("size", [1e18, 1e25, 1e37])
@pytest.mark.parametrize("shape", SHAPES)
def test_huge_rows_that_do_not_meet(shape, size, rng):
    """q has even dims alone and the keys odd ones: every score is 0, whatever the sizes."""
    batch = Batch(rng, *shape, q_scale=size, k_scale=size)
    batch.q[..., 1::2] = 0
    batch.k[..., ::2] *= 0  # (rows that nobody sees stay NaN)
    batch.check()


@pytest.mark.parametrize("H,d,tile", [(64, 64, 64), (64, 128, 32)])
def test_values_that_begin_with_zeros(H, d, tile, rng):
    """Prefixes of large values and, behind each in the same run, one whose first tile of values
    is zeros and the second tiny: a run holds two chains (64 kv heads have 8 runs each, and a
    chain of two tiles counts as three)."""
    batch = Batch(rng, [2 * tile] * 16, [[0]] * 16, H, 64, d)
    for g, at in enumerate(batch.prefix_row):
        if g % 2 == 0:
            batch.v[at:at + 2 * tile] *= np.float32(2.0 ** 90)
        else:
            batch.v[at:at + tile] = 0
            batch.v[at + tile:at + 2 * tile] *= np.float32(2.0 ** (-100 if g % 4 == 1 else 100))
    batch.check()
