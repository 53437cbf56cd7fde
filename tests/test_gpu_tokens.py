"""Log probabilities, alternatives and sampling on the GPU, through the C ABI, against 64
bits."""
from __future__ import annotations

import math

import numpy as np
import pytest

from flock_amd import ops

pytestmark = pytest.mark.gpu
B = ops.DeviceBuffer
INF, NAN = float("inf"), float("nan")
NONE = 0xffffffff


def dev(a, dtype=np.float32):
    return B.from_array(np.ascontiguousarray(a, dtype).ravel())


def place(x, pad=0, shift=0):
    """Rows x on the device, `pad` floats apart, `shift` floats behind an aligned address;
    what lies between holds infinities."""
    n, V = x.shape
    wide = np.full((n, V + pad), INF, np.float32)
    wide[:, :V] = x
    flat = np.concatenate([np.full(shift, INF, np.float32), wide.ravel(),
                           np.full(64, INF, np.float32)])
    buf = dev(flat)
    return buf, buf.ptr + 4 * shift, V + pad


def workspace(n, V, k):
    return B(max(256, ops.tokens_ws_bytes(n, V, k)))


def score(x, tokens=None, k=0, entropy=True, pad=0, shift=0):
    n, V = x.shape
    buf, at, ld = place(x, pad, shift)
    lp = dev(np.full(n, 7)) if tokens is not None else None
    ent = dev(np.full(n, 7)) if entropy else None
    ids = dev(np.full(n * k, 7), np.uint32) if k else None
    tops = dev(np.full(n * k, 7)) if k else None
    ops.token_logprobs(at, None if tokens is None else dev(tokens, np.uint32), lp, n, V,
                       workspace(n, V, k), entropy=ent, n_top=k, top_ids=ids, top_logprobs=tops,
                       ld=ld if pad else 0)
    ops.sync()
    return (None if lp is None else lp.download(n), None if ent is None else ent.download(n),
            ids.download(n * k, np.uint32).reshape(n, k) if k else None,
            tops.download(n * k).reshape(n, k) if k else None)


def order(row, k):
    """Ids of the k largest, ties by the lowest id; no -infinity, no NaN."""
    ids = np.flatnonzero(row > -INF)
    return ids[np.argsort(-row[ids], kind="stable")][:k]


def want(row, k):
    """(log probabilities, entropy, top ids, top log probabilities) in 64 bits."""
    x = row.astype(np.float64)
    ids = np.full(k, NONE, np.uint32)
    best = order(row, k)
    ids[:len(best)] = best
    if np.isnan(x).any() or not (x.max() < INF) or not (x.max() > -INF):
        lp, ent = np.full(x.size, NAN), NAN
    else:
        lp = x - x.max()
        lp = lp - np.log(np.exp(lp).sum())
        p = np.exp(lp)
        ent = -(p[p > 0] * lp[p > 0]).sum()
    top = np.full(k, -INF)
    top[:len(best)] = lp[best]
    return lp, ent, ids, top


def slack(V):
    """How far a row's sum may be off, relative to it: a weight's exponential by 2^-21 (its
    argument, a rounded difference of up to 100, by 100 * 2^-24 more where weights still
    count), and fewer than V / 256 + 64 rounded additions in turn."""
    return 2.0 ** -21 + 100 * 2.0 ** -24 + (V / 256 + 64) * 2.0 ** -24


def check(x, tokens=None, k=0, **kw):
    n, V = x.shape
    got = score(x, tokens, k, **kw)
    eps = slack(V)
    for r in range(n):
        lp, ent, ids, top = want(x[r], k)
        if tokens is not None:
            w = lp[tokens[r]] if tokens[r] < V else NAN
            close(got[0][r], w, eps + 2.0 ** -23 * abs(w))
        if got[1] is not None:
            close(got[1][r], ent, 4 * eps * (1 + ent))
        if k:
            assert np.array_equal(got[2][r], ids), (r, got[2][r], ids)
            for a, b in zip(got[3][r], top):
                close(a, b, eps + 2.0 ** -23 * abs(b))
    return got


def close(a, b, tol):
    if np.isnan(b):
        assert np.isnan(a), (a, b)
    elif np.isinf(b):
        assert a == b
    else:
        assert abs(float(a) - b) <= tol, (a, b, tol)


def language(rng, n, V):
    x = rng.standard_normal((n, V), np.float32) * np.float32(2.5)
    for r in range(n):
        x[r, rng.integers(0, V, min(12, V))] += 8
        if r % 3 == 0:
            x[r, rng.integers(0, V)] += 20
    return x


# -------------------------------------------------------------------- scores --
@pytest.mark.parametrize("n,V,k,pad,shift", [
    (1, 1, 1, 0, 0), (1, 2, 5, 0, 1), (3, 3, 64, 2, 3), (2, 63, 64, 0, 0), (5, 64, 64, 1, 2),
    (4, 65, 7, 0, 0), (2, 255, 1, 5, 1), (3, 1000, 20, 0, 0), (2, 4097, 64, 3, 1),
    (1, 32003, 64, 0, 3), (300, 1025, 5, 0, 0), (1, 151936, 5, 0, 0), (1, 151936, 0, 0, 0),
    (7, 151936, 20, 0, 0), (3, 200001, 64, 1, 0), (600, 5000, 0, 62, 0), (2100, 400, 3, 0, 0)])
def test_scores(n, V, k, pad, shift, rng):
    print(n, V, k, pad, shift, flush=True)
    x = language(rng, n, V)
    tokens = rng.integers(0, V, n)
    tokens[::2] = x[::2].argmax(1)
    a = check(x, tokens, k, pad=pad, shift=shift)
    b = score(x, tokens, k, pad=pad, shift=shift)
    assert all(p is None or np.array_equal(p, q) for p, q in zip(a, b))


def test_outputs_are_optional(rng):
    x = language(rng, 4, 3001)
    t = x.argmax(1)
    full = check(x, t, 5)
    assert np.array_equal(score(x, t, 0, entropy=False)[0], full[0])
    assert np.array_equal(score(x)[1], full[1])
    only = score(x, None, 5, entropy=False)
    assert np.array_equal(only[2], full[2]) and np.array_equal(only[3], full[3])


@pytest.mark.parametrize("V", [100, 5000, 151936])
def test_orders_that_are_hard(V, rng):
    """Rising, falling, all equal, two values, blocks of ties, and the largest at each end."""
    i = np.arange(V, dtype=np.float32)
    rows = [i * np.float32(1e-4), -i * np.float32(1e-4), np.zeros(V), np.where(i % 7 == 3, 1, -1),
            (i // 40) % 50, np.where(i == V - 1, 9, 0), np.where(i == 0, 9, 0),
            np.where(i % 2 == 0, 0.0, -0.0)]
    x = np.stack([np.asarray(r, np.float32) for r in rows])
    for k in (1, 20, 64):
        check(x, np.full(len(x), V - 1), k)


@pytest.mark.parametrize("n,V", [(256, 170001), (520, 90001)])
def test_rows_that_waves_take_in_segments(n, V, rng):
    """Many long rows: a workgroup each, whose waves look for alternatives more than once.
    Some rows are checked, hard ones among them."""
    x = rng.standard_normal((1, V), np.float32).repeat(n, 0) + np.arange(n, dtype=np.float32)[:, None]
    i = np.arange(V, dtype=np.float32)
    x[3], x[4], x[5], x[6] = i, -i, 2.5, (i // 1000) % 7
    x[7, 100:] = -INF
    x[8, :-40] = -INF
    rows = [0, 3, 4, 5, 6, 7, 8, n // 2, n - 1]
    buf = dev(x)
    tokens = np.full(n, V - 1)
    for k in (1, 64):
        lp, ids, tops = B(4 * n), B(4 * n * k), B(4 * n * k)
        ops.token_logprobs(buf, dev(tokens, np.uint32), lp, n, V, workspace(n, V, k), n_top=k,
                           top_ids=ids, top_logprobs=tops)
        ops.sync()
        got = ids.download(n * k, np.uint32).reshape(n, k)
        values, logs = tops.download(n * k).reshape(n, k), lp.download(n)
        for r in rows:
            l, _, w, top = want(x[r], k)
            assert np.array_equal(got[r], w), r
            close(logs[r], l[-1], slack(V) + 2.0 ** -23 * abs(l[-1]))
            for a, b in zip(values[r], top):
                close(a, b, slack(V) + 2.0 ** -23 * abs(b))


def test_masks_and_what_is_not_finite(rng):
    V = 3000
    x = language(rng, 10, V)
    x[0, 17:] = -INF                       # few alternatives
    x[1] = -INF                            # none
    x[2] = -INF
    x[2, 2999] = -5.0                      # one
    x[3, 100] = NAN
    x[4, 2000] = INF
    x[5, rng.permutation(V)[:2900]] = -INF
    x[6] = NAN
    x[7, :] = -3.4028235e38                # the type's lowest value is a logit
    x[8, ::2] = -3.4028235e38
    x[9, :] = 3.0e38
    check(x, np.array([3, 0, 2999, 5, 2000, int(np.flatnonzero(x[5] == -INF)[0]), 1, 2, 0, 9]), 64)


def test_ids_outside_the_vocabulary(rng):
    x = language(rng, 4, 500)
    check(x, np.array([499, 500, NONE, 0], np.uint64), 1, pad=12)


def test_a_nearly_sure_row_keeps_its_small_logarithm():
    """One id 30 above the others: log p = -log(1 + R), R = 999 exp(-30): relative to R,
    not to 1."""
    x = np.zeros((1, 1000), np.float32)
    x[0, 77] = 30
    lp, ent, _, _ = score(x, np.array([77]))
    R = 999 * math.exp(-30)
    assert abs(lp[0] + math.log1p(R)) <= slack(1000) * R
    H = math.log1p(R) + R * 30 / (1 + R)
    assert abs(ent[0] - H) <= 4 * slack(1000) * H


# ------------------------------------------------------------------ sampling --
def choose(row, u, t=1.0, k=64, top_p=1.0, min_p=0.0):
    ids = order(row, k)
    if not len(ids) or not (0 <= t < INF and 1 <= k and top_p > 0 and 0 <= min_p <= 1 and 0 <= u < 1):
        return NONE
    if t == 0:
        return int(ids[0])
    x = row[ids].astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / np.float64(t)))
    before = np.concatenate([[0], np.cumsum(w)[:-1]])
    n = 0
    while n < len(w) and before[n] < top_p * w.sum() and w[n] >= min_p and w[n] > 0:
        n += 1
    c = np.cumsum(w[:n])
    return int(ids[min(np.searchsorted(c, u * c[-1], side="right"), n - 1)])


def draw(x, u, max_k, t=None, k=None, top_p=None, min_p=None, pad=0, shift=0):
    n, V = x.shape
    buf, at, ld = place(x, pad, shift)
    token, lp = dev(np.full(n, 7), np.uint32), dev(np.full(n, 7))

    def opt(a, dtype=np.float32):
        return None if a is None else dev(np.broadcast_to(np.asarray(a, dtype), (n,)), dtype)

    ops.sample(at, opt(u), token, n, V, max_k, workspace(n, V, max_k), temperature=opt(t),
               top_k=opt(k, np.uint32), top_p=opt(top_p), min_p=opt(min_p), logprob=lp,
               ld=ld if pad else 0)
    ops.sync()
    return token.download(n, np.uint32), lp.download(n)


def check_draw(x, u, max_k, t=None, k=None, top_p=None, min_p=None, **kw):
    n, V = x.shape
    token, lp = draw(x, u, max_k, t, k, top_p, min_p, **kw)

    def at(a, r, default, dtype=np.float32):
        return default if a is None else dtype(np.broadcast_to(np.asarray(a, dtype), (n,))[r])

    for r in range(n):
        w = choose(x[r], float(at(u, r, 0)), float(at(t, r, 1.0)),
                   int(at(k, r, max_k, np.uint32)) if int(at(k, r, 1, np.uint32)) <= max_k else 0,
                   float(at(top_p, r, 1.0)), float(at(min_p, r, 0.0)))
        assert token[r] == w, (r, token[r], w)
        value = want(x[r], 1)[0][w] if w != NONE else NAN
        close(lp[r], value, slack(V) + 2.0 ** -23 * abs(value))
    return token


@pytest.mark.parametrize("n,V,max_k,pad,shift", [
    (1, 1, 1, 0, 0), (64, 2, 64, 1, 1), (100, 50, 20, 0, 0), (40, 3000, 64, 5, 3),
    (3, 151936, 20, 0, 0), (200, 2501, 50, 0, 0), (9, 70001, 64, 2, 0), (1, 151936, 64, 0, 1)])
def test_samples(n, V, max_k, pad, shift, rng):
    x = language(rng, n, V)
    u = rng.random(n, np.float32)
    u[0] = 0
    u[-1] = np.float32(1 - 2.0 ** -24)
    kw = dict(pad=pad, shift=shift)
    check_draw(x, u, max_k, **kw)
    check_draw(x, u, max_k, t=rng.uniform(0.2, 1.5, n), k=rng.integers(1, max_k + 1, n),
               top_p=rng.uniform(0.3, 1, n), min_p=rng.uniform(0, 0.2, n), **kw)
    check_draw(x, u, max_k, t=np.where(rng.random(n) < 0.5, 0, 1), **kw)


def test_uniform_numbers_pick_equal_weights_in_turn(rng):
    """Four ids of equal logits far above the rest: u * 4, without a rounding."""
    x = np.full((64, 500), -1e4, np.float32)
    x[:, [7, 90, 200, 499]] = 3.0
    u = np.arange(64) / 64
    assert check_draw(x, u, 4).tolist() == [(7, 90, 200, 499)[i // 16] for i in range(64)]
    assert check_draw(x, u, 64).tolist() == [(7, 90, 200, 499)[i // 16] for i in range(64)]
    # top_p = 1/2 is reached by the second, 1/2 + 2^-24 only by the third.
    assert set(check_draw(x, u, 64, top_p=0.5)) == {7, 90}
    assert set(check_draw(x, u, 64, top_p=0.5 + 2.0 ** -23)) == {7, 90, 200}


def test_masks_extremes_and_rows_without_an_alternative(rng):
    V = 800
    x = language(rng, 9, V)
    x[0] = -INF
    x[1] = NAN
    x[2, 5:] = -INF
    x[3, 9] = NAN                  # never chosen; the distribution is gone
    x[4, [8, 70]] = INF            # these two, in equal parts
    x[5, 1:] = -INF
    x[6] = 0
    for u in (0.0, 0.3, 0.9):
        check_draw(x, u, 64)
        check_draw(x, u, 64, t=1e-30)
        check_draw(x, u, 64, t=1e30)
        check_draw(x, u, 64, t=INF)
        check_draw(x, u, 64, min_p=1.0, top_p=1e-30)


def test_settings_out_of_range_are_refused(rng):
    x = language(rng, 14, 300)
    u = np.array([0.5] * 5 + [1.0, -0.1, NAN] + [0.5] * 6, np.float32)
    t = np.array([-1, NAN] + [1] * 12, np.float32)
    k = np.array([5, 5, 0, 21, NONE] + [5] * 9, np.uint64)
    top_p = np.array([1] * 8 + [0, -1, NAN, 1, 1, 1], np.float32)
    min_p = np.array([0] * 11 + [-0.1, 1.1, NAN], np.float32)
    token, lp = draw(x, u, 20, t, k, top_p, min_p)
    assert (token == NONE).all() and np.isnan(lp).all()


def test_logprob_may_be_left_out(rng):
    x = language(rng, 5, 2000)
    u = rng.random(5, np.float32)
    token = dev(np.zeros(5), np.uint32)
    ops.sample(dev(x), dev(u), token, 5, 2000, 20, workspace(5, 2000, 20))
    ops.sync()
    assert np.array_equal(token.download(5, np.uint32), draw(x, u, 20)[0])


# -------------------------------------------------------------------- graphs --
def test_captured_calls_replayed_on_new_logits(rng):
    """Scores and samples captured on one workspace, replayed with eager work between."""
    for n, V, k in ((1, 151936, 20), (70, 3001, 64)):
        x = [language(rng, n, V) for _ in range(3)]
        logits, u = dev(x[0]), dev(np.zeros(n))
        token, lp, ent = dev(np.zeros(n), np.uint32), dev(np.zeros(n)), dev(np.zeros(n))
        ids, tops = dev(np.zeros(n * k), np.uint32), dev(np.zeros(n * k))
        ws = workspace(n, V, k)
        stream = ops.Stream()
        ops.set_stream(stream)
        with ops.Graph() as g:
            ops.sample(logits, u, token, n, V, k, ws)
            ops.token_logprobs(logits, token, lp, n, V, ws, entropy=ent, n_top=k, top_ids=ids,
                               top_logprobs=tops)
        for y in x + x[:1]:
            number = rng.random(n, np.float32)
            logits.upload(y)
            u.upload(number)
            g.launch()
            ops.sync()
            t = token.download(n, np.uint32)
            got = (lp.download(n), ent.download(n), ids.download(n * k, np.uint32).reshape(n, k),
                   tops.download(n * k).reshape(n, k))
            assert np.array_equal(t, check_draw(y, number, k))
            for a, b in zip(got, check(y, t, k)):
                assert np.array_equal(a, b)
        ops.set_stream(None)
        g.free()
        stream.free()


def test_rows_behind_four_gigabytes(rng):
    """Rows whose stride puts them past 2^32 bytes."""
    V, ld, n = 1000, (1 << 29) + 1, 3
    x = language(rng, n, V)
    big = B(4 * ((n - 1) * ld + V))
    for r in range(n):
        big.upload(x[r], 4 * r * ld)
    lp, ids, tops = B(4 * n), B(4 * n * 5), B(4 * n * 5)
    t = x.argmax(1)
    ops.token_logprobs(big, dev(t, np.uint32), lp, n, V, workspace(n, V, 5), n_top=5, top_ids=ids,
                       top_logprobs=tops, ld=ld)
    ops.sync()
    full = check(x, t, 5)
    assert np.array_equal(lp.download(n), full[0])
    assert np.array_equal(ids.download(5 * n, np.uint32).reshape(n, 5), full[2])
    big.free()
