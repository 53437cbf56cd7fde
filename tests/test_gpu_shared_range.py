"""Decode attention over shared prefixes where sizes are extreme: scores next to 0 or past f32's
range, values that are all zeros or far smaller than others."""
from __future__ import annotations

import math

import numpy as np
import pytest

from test_gpu_shared import SHAPES as ATTENTION, Batch

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


def two_norms(got, o):
    return np.linalg.norm(got - o, axis=-1), np.linalg.norm(o, axis=-1)


@pytest.mark.parametrize("i", range(len(ATTENTION)))
def test_rows_in_the_2_norm(i, rng):
    """Ordinary rows are as exact as f32 products make them: a score (some 2 nats, of products
    that are off by 2^-22 each with either sign) is off by 2^-21 or so, its weight by as much of
    itself, values by 2^-22; the errors of a row's weights have either sign, so that the row's is
    theirs. 2^-18 is eight times that, and a thirtieth of what a lost second part (2^-11 to 2^-13)
    makes of any of the four operands."""
    prefix, own, H, G, d = ATTENTION[i]
    batch = Batch(rng, prefix, own, H, G, d, q_scale=2.0)
    o, _ = batch.want()
    off, size = two_norms(batch.run(), o)
    assert (off <= 2.0 ** -18 * size).all(), (off / size).max()


def sink(batch, at, gap, rng):
    """Row `at` of the caches takes `gap` nats more than other keys on average, and has no
    values."""
    G, d = batch.G, batch.d
    u = rng.standard_normal((G, d)).astype(np.float32)
    u /= np.linalg.norm(u, axis=-1, keepdims=True)
    batch.k -= (batch.k * u).sum(-1, keepdims=True) * u
    heads = np.repeat(u, batch.H // G, axis=0)
    batch.q += 16 * heads
    batch.k[at] = u * np.float32(gap * math.sqrt(d) / 16)
    batch.v[at] = 0


@pytest.mark.parametrize("gap", [8, 15, 20, 25, 35])
@pytest.mark.parametrize("P,own,H,G,d,at", [
    (513, [9, 0], 16, 8, 128, 0), (513, [9, 0], 32, 8, 64, 0),
    (9000, [3] * 5, 4, 2, 128, 0), (9000, [40], 4, 4, 64, 4321), (200, [70, 900], 16, 8, 128, 150),
])
def test_a_key_that_takes_the_weight_and_has_no_values(P, own, H, G, d, at, gap, rng):
    """What is left of the row is as exact, of its own size, as without that key: as in
    test_rows_in_the_2_norm, and the score of that key (all others' share hangs on it), a sum
    of 24 products in f32 whose roundings are 2^-24 of it each, 2^-22 in all where half of
    them agree."""
    batch = Batch(rng, [P], [own], H, G, d, q_scale=2.0)
    sink(batch, batch.prefix_row[0] + at, gap, rng)
    o, _ = batch.want()
    off, size = two_norms(batch.run(), o)
    print(gap, (off / size).max(), flush=True)
    assert (off <= (2.0 ** -18 + 1.5 * gap * 2.0 ** -22) * size).all(), (off / size).max()


def test_many_keys_that_take_the_weight(rng):
    """The same with such a key in every group's prefix and every sequence's own keys, which lie in
    few runs (64 kv heads have 8 runs each)."""
    batch = Batch(rng, [300] * 12, [[200, 33]] * 12, 64, 64, 64, q_scale=2.0)
    k, q, v = batch.k, batch.q, batch.v
    u = np.zeros((64, 64), np.float32)
    u[:, 0] = 1
    k[..., 0] = np.where(np.isnan(k[..., 0]), k[..., 0], 0)
    q += 16 * u
    for i, at in enumerate(batch.prefix_row + batch.own_row):
        k[at + i % 30, :, 0] += 10 + i % 3 * 4
        v[at + i % 30] = 0
    o, _ = batch.want()
    off, size = two_norms(batch.run(), o)
    assert (off <= (2.0 ** -18 + 60 * 2.0 ** -22) * size).all(), (off / size).max()


@pytest.mark.parametrize("H,G,d", [(16, 8, 128), (8, 4, 64)])
def test_scores_past_the_range_of_f32(H, G, d, rng):
    """Scores of -infinity have no weight beside others (of the prefix or own), and a row with
    none else is NaN, as one with a score of +infinity is."""
    batch = Batch(rng, [70, 70], [[40, 3], [5, 90]], H, G, d, q_scale=0.0)
    batch.q[:] = 1e20
    for g, size in ((0, -1e20), (1, 1e-21)):
        at = batch.prefix_row[g]
        batch.k[at:at + 70] = np.float32(size)
    for b, size in enumerate((-1e20, 1e-21, -1e20, 1e20)):
        at = batch.own_row[b]
        batch.k[at:at + batch.n_keys[b]] = np.float32(size)
    got = batch.run()
    assert np.isnan(got[[0, 3]]).all()
    for b, row, n in ((1, batch.own_row[1], 3), (2, batch.prefix_row[1], 70)):
        batch.rows = lambda _: list(range(row, row + n))
        o, tol = batch.want([b])
        assert (np.abs(got[b] - o[b]) <= tol[b]).all()


@pytest.mark.parametrize("size", [0.3, 0.02, 1e-3])
@pytest.mark.parametrize("spread", [2.0, 8.0])
@pytest.mark.parametrize("H,G,d", [(16, 8, 128), (32, 8, 64)])
def test_a_key_that_takes_the_weight_and_has_small_values(H, G, d, spread, size, rng):
    """The same with values of a part of the others' size, also where scores lie far apart (a sum
    of more products in turn: scores up to 4 spread, and the gap)."""
    batch = Batch(rng, [2900], [[40, 200, 0]], H, G, d, q_scale=spread)
    at = batch.prefix_row[0]
    v = batch.v[at].copy()
    sink(batch, at, 20, rng)
    batch.v[at] = v * np.float32(size)
    o, _ = batch.want()
    off, norm = two_norms(batch.run(), o)
    print(size, (off / norm).max(), flush=True)
    assert (off <= (2.0 ** -18 + 1.5 * (20 + 4 * spread) * 2.0 ** -22) * norm).all()


@pytest.mark.parametrize("H,G,d", [(16, 8, 128), (32, 8, 64)])
@pytest.mark.parametrize("v_scale", [1e-30, 1e30])
@pytest.mark.parametrize("part", [0.0, 0.01])
def test_a_key_that_takes_the_weight_of_huge_or_tiny_values(H, G, d, v_scale, part, rng):
    """References that have fallen leave large sums, beside values near either end of f32. Results
    below 2^-126 (of 1e-30, and a share of e^-27) are multiples of 2^-149: the partial results of up
    to 64 runs, their sum's steps and the result itself are off by half of that each."""
    batch = Batch(rng, [1300], [[40, 700]], H, G, d, q_scale=2.0, v_scale=v_scale)
    at = batch.prefix_row[0]
    v = batch.v[at].copy()
    sink(batch, at, 30, rng)
    batch.k[batch.own_row[1] + 3] = batch.k[at] * np.float32(0.8)
    batch.v[batch.own_row[1] + 3] = 0
    batch.v[at] = v * np.float32(part)
    o, _ = batch.want()
    off, size = (x / v_scale for x in two_norms(batch.run().astype(np.float64), o))
    least = (64 + 2) * 2.0 ** -150 * math.sqrt(d) / v_scale
    assert (off <= (2.0 ** -18 + 45 * 2.0 ** -22) * size + least).all(), (off / size).max()
