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
