"""The paged 4-bit cache on the GPU, through the C ABI: plans and codes equal to
the reference's, attention against 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest

import kv4_ref as ref
import oracle
from flock_amd import ops
from flock_amd._lib import FlockError

pytestmark = pytest.mark.gpu
B = ops.DeviceBuffer
EPS = 9.999999974752427e-7


def u32(a):
    return B.from_array(np.ascontiguousarray(a, np.uint32).ravel())


def filled(n, value=7.0):
    return B.from_array(np.full(max(n, 1), value, np.float32))


# ---------------------------------------------------------------------- plan --
def run_plan(n_keys, n_new, table, free, max_tokens, n_pages, page, window, sinks, in_place=False):
    S, M = table.shape
    f = np.zeros(1 + n_pages, np.uint32)
    f[0] = len(free)
    f[1:1 + len(free)] = free
    t_in = u32(table)
    t_out = t_in if in_place else u32(np.full(S * M, 5))
    f_in, f_out = u32(f), u32(np.zeros(1 + n_pages))
    q_off, lost = u32(np.zeros(S + 1)), u32([99])
    pos, slots = u32(np.full(max_tokens, 9)), u32(np.full(max_tokens, 9))
    ws = B(ops.kv4_plan_ws_bytes(S))
    ops.kv4_plan(u32(n_keys), u32(n_new), t_in, t_out, f_in, f_out, q_off, pos, slots, lost, S, M,
                 n_pages, max_tokens, page, window, sinks, ws)
    ops.sync()
    got = f_out.download(1 + n_pages, np.uint32)
    return (t_out.download(S * M, np.uint32).reshape(S, M), got[1:1 + got[0]].tolist(),
            q_off.download(S + 1, np.uint32).tolist(), pos.download(max_tokens, np.uint32).tolist(),
            slots.download(max_tokens, np.uint32).tolist(), int(lost.download(1, np.uint32)[0]))


def check_plan(*args, **kw):
    got, want = run_plan(*args, **kw), ref.plan(*args)
    np.testing.assert_array_equal(got[0], want[0])
    assert got[1:] == tuple(want[1:])
    return got


@pytest.mark.parametrize("S,M,page,window,sinks,seed", [
    (1, 1, 32, 0, 0, 0), (3, 5, 32, 0, 0, 1), (16, 70, 64, 0, 0, 2), (17, 64, 32, 100, 4, 3),
    (40, 130, 32, 33, 40, 4), (300, 9, 256, 300, 1, 5), (33, 65, 128, 1, 0, 6)])
def test_plan_steps_equal_the_reference(S, M, page, window, sinks, seed):
    """A few steps in a row: prompts, single tokens, ends, tokens taken back, idle
    sequences; the table and the free list of one step feed the next."""
    rng = np.random.default_rng(seed)
    n_pages = S * M // 2 + 3
    table = np.full((S, M), ref.NONE, np.uint32)
    free = rng.permutation(n_pages).tolist()
    keys = np.zeros(S, np.int64)
    for step in range(5):
        new = rng.choice([0, 1, 3, page, M * page // 3], S)
        what = rng.random(S)
        keys = np.where(what < 0.1, 0, np.where(what < 0.2, keys // 2, keys + new))
        keys = np.minimum(keys, M * page + 5)  # a few past the table
        new = np.minimum(new, keys)
        max_tokens = max(1, int(new.sum()) + (step % 3 - 1) * 7)
        table, free, *_ = check_plan(keys, new, table, free, max_tokens, n_pages, page, window,
                                     sinks, in_place=step % 2 == 1)


def test_plan_without_free_pages_and_again_with_some():
    table = np.full((2, 4), ref.NONE, np.uint32)
    t, free, _, _, slots, lost = check_plan([100, 60], [100, 60], table, [3, 1], 160, 8, 32, 0, 0)
    assert lost == 160 - 64 and free == []
    t, free, _, _, _, lost = check_plan([100, 60], [100, 60], t, [0, 2, 4, 5, 6], 160, 8, 32, 0, 0)
    assert lost == 0 and len(free) == 1


def test_plan_takes_more_new_tokens_than_keys_as_all():
    t, *_ = check_plan([5], [9], np.full((1, 2), ref.NONE, np.uint32), [0, 1], 9, 2, 32, 0, 0)


# ------------------------------------------------------------- append, read --
def read_back(pool, slots, n, G, D, n_pages, page):
    k, v = filled(n * G * D), filled(n * G * D)
    ops.kv4_read(pool, slots, k, v, n, G, D, n_pages, page)
    ops.sync()
    return (x.download(n * G * D).reshape(n, G, D) for x in (k, v))


def rows_like_caches(rng, n, G, D):
    """Normal rows, and rows that reach the format's edges."""
    x = rng.standard_normal((n, G, D)).astype(np.float32)
    x[0::7] *= np.float32(1e-7)           # scales below f16's normal numbers
    x[1::7] *= np.float32(3e4)            # some past the largest value
    x[2::7] = np.rint(x[2::7] * 2) / 2    # ties
    x[3::7, :, :32] = 0                   # a block of zeros
    if n > 4:
        x[4, 0, 5] = np.nan
        x[4, -1, D - 1] = -np.inf
        x[4, 0, 40:42] = [3, -3]          # the largest twice, with both signs
    return x


@pytest.mark.parametrize("n,G,D,page", [(1, 1, 128, 32), (40, 8, 128, 64), (67, 3, 64, 128),
                                        (33, 5, 64, 32), (300, 2, 128, 256)])
def test_append_and_read_equal_the_reference(n, G, D, page, rng):
    k, v = rows_like_caches(rng, n, G, D), rows_like_caches(rng, n, G, D)[::-1].copy()
    n_pages = -(-n // page) + 2
    slots = rng.permutation(n_pages * page)[:n].astype(np.uint32)
    slots[n // 2:n // 2 + 1] = ref.NONE
    start = rng.integers(0, 256, (n_pages, G, page // 32, 36 * D), dtype=np.uint8)
    want = start.copy()
    ref.store(want, slots, k, v, page)
    pool, sl = B.from_array(start), u32(slots)
    ops.kv4_append(B.from_array(k), B.from_array(v), sl, pool, n, G, D, n_pages, page)
    ops.sync()
    np.testing.assert_array_equal(pool.download(want.size, np.uint8), want.ravel())
    rk, rv = ref.load(want, page)
    gk, gv = read_back(pool, sl, n, G, D, n_pages, page)
    for got, whole in ((gk, rk), (gv, rv)):
        for i, s in enumerate(slots):
            np.testing.assert_array_equal(got[i], 0 if s == ref.NONE else whole[s])


@pytest.mark.parametrize("n,H,G,D,page,pairing,stacked", [
    (1, 16, 8, 128, 64, "neox", False), (37, 16, 8, 128, 32, "norm", True),
    (70, 20, 4, 64, 128, "neox", True), (9, 8, 1, 64, 64, "norm", False),
    (130, 40, 5, 128, 256, "neox", False)])
def test_prologue_stores_the_f32_prologues_rows(n, H, G, D, page, pairing, stacked, rng):
    """q equals qk_prologue's bits; K and V the codes of its rows."""
    q, k, v = (rng.standard_normal((n, h * D)).astype(np.float32) for h in (H, G, G))
    gq, gk = (rng.normal(1, 0.1, D).astype(np.float32) for _ in range(2))
    inv = oracle.rope_inv_freq(D, 1e6)
    pos0 = 1000
    n_pages = -(-n // page) + 1
    slots = rng.permutation(n_pages * page)[:n].astype(np.uint32)
    pool = B.from_array(np.zeros(n_pages * ops.kv4_page_bytes(G, D, page), np.uint8))
    dev = [B.from_array(x) for x in (gq, gk, inv)]
    raw = [B.from_array(x) for x in (q, k, v)]
    qn = filled(n * H * D)
    args = raw
    if stacked:
        whole = B.from_array(np.concatenate([q, k, v], 1))
        args = [whole.ptr, whole.ptr + 4 * H * D, whole.ptr + 4 * (H + G) * D]
    sl = u32(slots)
    ops.kv4_prologue(*args, *dev, EPS, pairing, u32(pos0 + np.arange(n)), sl, qn, pool, n, H, G, D,
                     n_pages, page, in_stride=(H + 2 * G) * D if stacked else 0)
    rows = pos0 + n
    qw, kc, vc = filled(n * H * D), B(4 * rows * G * D), B(4 * rows * G * D)
    ops.qk_prologue(*raw, *dev, EPS, pairing, qw, kc, vc, n, pos0, H, G, D, rows)
    ops.sync()
    np.testing.assert_array_equal(qn.download(n * H * D), qw.download(n * H * D))
    for got, cache in zip(read_back(pool, sl, n, G, D, n_pages, page), (kc, vc)):
        x = cache.download(n * G * D, offset_bytes=4 * pos0 * G * D).reshape(n, G, D)
        np.testing.assert_array_equal(got, ref.values(*ref.quantise(x)))


# ----------------------------------------------------------------- attention --
class Batch:
    """Sequences of n_keys[b] keys with their pages dealt out at random, and q rows
    for the last n_new[b] of them. Pages that no visible key needs have no entry;
    what the table's last pages hold behind a sequence is NaN, infinities and scales whose
    products with codes are infinite."""

    def __init__(self, rng, n_keys, n_new, H, G, D, page, window=0, sinks=0, k=None, v=None):
        self.shape = (H, G, D, page, window, sinks)
        self.n_keys, self.n_new = list(n_keys), list(n_new)
        S, M = len(n_keys), max(1, -(-max(n_keys) // page))
        self.S, self.M = S, M
        table, self.q_off = ref.dealt(n_keys, n_new, M, page, window, sinks)
        ids = rng.permutation(S * M).astype(np.uint32)
        self.table = np.where(table < S * M, ids[np.minimum(table, S * M - 1)], ref.NONE)
        self.P = S * M
        self.pool = rng.integers(0, 256, (self.P, G, page // 32, 36 * D), dtype=np.uint8)
        kb, _, ks, vb, _, vs = ref.places(D)
        for at in (np.unique(ks), np.unique(vs)):
            bits = rng.choice([0x7E00, 0xFC00, 0x7BFF, 0xF001], self.pool[..., at].shape)
            self.pool[..., at] = bits & 255
            self.pool[..., at + 1] = bits >> 8
        self.k, self.v = [], []
        for b in range(S):
            n = self.n_keys[b]
            kk = rng.standard_normal((n, G, D)).astype(np.float32) if k is None else k[b]
            vv = rng.standard_normal((n, G, D)).astype(np.float32) if v is None else v[b]
            pages = self.table[b][np.arange(n) // page].astype(np.int64)
            slots = np.where(pages < self.P, pages * page + np.arange(n) % page, ref.NONE)
            fast_store(self.pool, slots, kk, vv, page)
            self.k.append(ref.values(*ref.quantise(kk)))
            self.v.append(ref.values(*ref.quantise(vv)))
        self.T = self.q_off[-1]
        self.q = rng.standard_normal((max(1, self.T), H, D)).astype(np.float32)

    def run(self, max_q=None, max_n_keys=None, in_place=False, extra=2, times=1):
        H, G, D, page, window, sinks = self.shape
        max_q = max_q or max(1, max(self.n_new))
        max_n_keys = max_n_keys or max(1, max(self.n_keys))
        rows = self.T + extra
        q = np.concatenate([self.q[:self.T], np.full((extra, H, D), 3, np.float32)])
        dq = B.from_array(q)
        o = dq if in_place else filled(rows * H * D)
        need = ops.kv4_attn_ws_bytes(self.S, max_q, max_n_keys, H, G, D, window, sinks)
        ws = B(max(256, need))
        dev = [B.from_array(self.pool), u32(self.table), u32(self.n_keys), u32(self.q_off)]
        for _ in range(times):
            ops.kv4_attn(dq, *dev, o, self.S, rows, max_q, max_n_keys, self.M, H, G, D, self.P,
                         page, window, sinks, ws)
        ops.sync()
        got = o.download(rows * H * D).reshape(rows, H, D)
        np.testing.assert_array_equal(got[self.T:], 3 if in_place else 7)  # left as they were
        return got[:self.T]

    def want(self):
        H, G, D, page, window, sinks = self.shape
        out = [ref.attention(self.q[a:a + m], self.k[b], self.v[b], n, window, sinks)
               for b, (n, m, a) in enumerate(zip(self.n_keys, self.n_new, self.q_off))]
        return np.concatenate(out) if out else np.zeros((0, H, D))


def fast_store(pool, slots, k, v, page):
    """ref.store by whole arrays (every slot of its own)."""
    D = k.shape[-1]
    kb, ksh, ks, vb, vsh, vs = ref.places(D)
    ok = slots < pool.shape[0] * page
    s = slots[ok].astype(np.int64)
    p, i, t = s // page, s % page // 32, s % 32
    for x, b, sh, at in ((k, kb, ksh, ks), (v, vb, vsh, vs)):
        c, d = ref.quantise(x[ok])
        for g in range(k.shape[1]):
            for nib in (0, 4):
                sel = sh[t] == nib
                rows, e = np.nonzero(sel)
                at_b = b[t[rows], e]
                keep = 0xF0 if nib == 0 else 0x0F
                old = pool[p[rows], g, i[rows], at_b]
                pool[p[rows], g, i[rows], at_b] = (old & keep) | (c[rows, g, e] << nib)
            for blk in range(D // 32):
                two = np.ascontiguousarray(d[:, g, blk]).view(np.uint8).reshape(-1, 2)
                pool[p, g, i, at[t, 32 * blk]] = two[:, 0]
                pool[p, g, i, at[t, 32 * blk] + 1] = two[:, 1]


def close(got, want, batch):
    """f32 sums and two-part operands. With N(0, 1) rows a score is at most about 8:
    its error is 8 * (2^-23 of the parts, 2^-25 sqrt(128) of f32 sums, 2^-24 of the
    exponent), the weights' own 2^-22: together under 5e-6 of a weight. Twice that in
    the 2-norm; per element against the largest value, ten times it (errors of some
    hundred weights that do not cancel)."""
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    got, want = got[fine], want[fine]
    if not want.size or not np.any(want):
        np.testing.assert_array_equal(got, want)
        return
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)
    assert np.max(np.abs(got - want)) <= 1e-4 * np.max(np.abs(want))


SHAPES = [(16, 8, 128), (32, 8, 64), (3, 3, 128), (8, 1, 64), (10, 2, 128), (14, 2, 64),
          (6, 1, 128), (4, 1, 64)]


@pytest.mark.parametrize("H,G,D", SHAPES)
@pytest.mark.parametrize("page", [32, 64, 256])
def test_decode_of_a_ragged_batch(H, G, D, page, rng):
    x = Batch(rng, [1, 31, 32, 33, 0, 257, 700], [1, 1, 1, 1, 0, 1, 1], H, G, D, page)
    close(x.run(), x.want(), x)


@pytest.mark.parametrize("H,G,D", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 4), (100, 40)])
def test_drafts_with_windows(H, G, D, window, sinks, rng):
    x = Batch(rng, [5, 33, 150, 64, 400], [5, 2, 3, 0, 4], H, G, D, 64, window, sinks)
    close(x.run(), x.want(), x)


@pytest.mark.parametrize("H,G,D", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (50, 0), (70, 37)])
def test_prompts(H, G, D, window, sinks, rng):
    x = Batch(rng, [1, 70, 129, 300, 40], [1, 70, 33, 100, 0], H, G, D, 32, window, sinks)
    close(x.run(), x.want(), x)


@pytest.mark.parametrize("window,sinks", [(1, 2**32 - 1), (2**32 - 1, 2**32 - 1), (2**31, 0),
                                          (2**31 - 1, 2**31), (40, 2**31 - 1)])
@pytest.mark.parametrize("new", [(1, 2, 1), (70, 3, 0)])
def test_windows_and_sinks_past_the_sequences(window, sinks, new, rng):
    x = Batch(rng, [90, 33, 200], new, 4, 2, 64, 32, window, sinks)
    close(x.run(), x.want(), x)
    table = np.full((3, 7), ref.NONE, np.uint32)
    check_plan([90, 33, 200], list(new), table, list(range(30)), 80, 30, 32, window, sinks)


@pytest.mark.parametrize("keys,new,page", [(3000, 1, 64), (5001, 1, 128), (4100, 3, 32),
                                           (2500, 130, 64), (2049, 2049, 64)])
def test_long_sequences(keys, new, page, rng):
    x = Batch(rng, [keys], [new], 2, 1, 128, page)
    close(x.run(), x.want(), x)
    y = Batch(rng, [keys, 40], [new, 1], 4, 2, 64, page, window=1000, sinks=5)
    close(y.run(), y.want(), y)


@pytest.mark.parametrize("new", [1, 3, 40])
def test_rows_that_see_nothing_are_zeros(new, rng):
    x = Batch(rng, [new, 100], [new, 1], 4, 2, 128, 32)
    x.n_keys = [new - 1, 100]  # the first row lies before the sequence
    got = x.run()
    want = np.concatenate([np.zeros((1, 4, 128)), ref.attention(
        x.q[1:new], x.k[0][:new - 1], x.v[0][:new - 1], new - 1) if new > 1 else np.zeros((0, 4, 128)),
        ref.attention(x.q[new:new + 1], x.k[1], x.v[1], 100)])
    close(got, want, x)
    assert not got[0].any()


@pytest.mark.parametrize("new", [1, 4, 60])
def test_refused_sequences_are_nan_and_the_others_are_not(new, rng):
    x = Batch(rng, [200, 100, 90], [new, new, new], 16, 8, 128, 32)
    want = x.want()
    x.table[1, 1] = 10 ** 9  # no such page
    got = x.run(max_n_keys=150)  # the first has more keys
    assert np.isnan(got[:new]).all() and np.isnan(got[new:2 * new]).all()
    close(got[2 * new:], want[2 * new:], x)


@pytest.mark.parametrize("news", [(1, 5), (2, 70)])
def test_more_rows_than_max_q_are_refused(news, rng):
    x = Batch(rng, [100, 100], news, 4, 2, 64, 64)
    got = x.run(max_q=news[1] - 1)
    close(got[:news[0]], x.want()[:news[0]], x)
    assert np.isnan(got[news[0]:]).all()


@pytest.mark.parametrize("H,G,D,news", [
    (16, 2, 128, (3, 1, 0, 2, 3)), (16, 2, 128, (6, 4, 1, 5, 6)), (32, 8, 64, (12, 7, 4, 0, 9)),
    (4, 4, 128, (48, 17, 33, 1, 16)), (6, 2, 64, (7, 11, 6, 16, 5))])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5)])
def test_drafts_of_more_rows_than_a_chunk(H, G, D, news, window, sinks, rng):
    keys = [max(n, k) for n, k in zip(news, (2500, 40, 700, 5, 1400))]
    x = Batch(rng, keys, news, H, G, D, 64, window, sinks)
    want = x.want()
    close(x.run(), want, x)
    close(x.run(in_place=True), want, x)
    x.n_keys[1] = 3000  # refused: more than the call's bound
    got = x.run(max_n_keys=2500)
    one = slice(x.q_off[1], x.q_off[2])
    assert np.isnan(got[one]).all()
    got[one] = want[one]
    close(got, want, x)


MIXED = ([2500, 300, 3000, 0, 2100, 60, 2400], [1, 300, 4, 0, 130, 60, 9])


@pytest.mark.parametrize("H,G,D,page,window,sinks", [
    (16, 8, 128, 64, 0, 0), (32, 8, 64, 32, 0, 0), (8, 1, 128, 256, 2300, 4), (3, 3, 64, 128, 0, 0)])
def test_single_tokens_and_prompts_together(H, G, D, page, window, sinks, rng):
    """Bounds past which a call takes both kernels."""
    x = Batch(rng, *MIXED, H, G, D, page, window, sinks)
    want = x.want()
    close(x.run(), want, x)
    close(x.run(in_place=True, times=1), want, x)


def test_refusals_of_single_tokens_and_prompts_together(rng):
    x = Batch(rng, *MIXED, 4, 2, 128, 64)
    want = x.want()
    x.table[2, 7] = ref.NONE  # of a draft
    x.table[4, 9] = x.P + 3   # of a prompt
    x.n_keys[6] = 2700        # both past the bound
    x.n_keys[0] = 2699
    got = x.run(max_q=200, max_n_keys=2600)
    for b in (0, 1, 2, 4, 6):  # (sequence 1 has more rows than max_q; 2 more keys than the bound)
        assert np.isnan(got[x.q_off[b]:x.q_off[b + 1]]).all(), b
    close(got[x.q_off[5]:x.q_off[6]], want[x.q_off[5]:x.q_off[6]], x)


@pytest.mark.parametrize("H,G,D,window,sinks", [(8, 4, 128, 0, 0), (4, 1, 64, 0, 0),
                                                (4, 2, 64, 700, 3)])
def test_more_row_tiles_than_threads_some_of_them_long(H, G, D, window, sinks, rng):
    """The pieces come from a list; the long sequences' row tiles are cut."""
    keys, news = rng.integers(1, 700, 60), rng.choice([0, 1, 5, 40, 100, 600], 60)
    keys[[3, 30, 59]], news[[3, 30, 59]] = (5000, 3100, 2500), (300, 64, 600)
    news = np.minimum(news, keys)
    x = Batch(rng, keys.tolist(), news.tolist(), H, G, D, 64, window, sinks)
    want = x.want()
    close(x.run(times=2), want, x)
    close(x.run(in_place=True), want, x)
    x.n_keys[3] = 6000  # refused
    got = x.run(max_n_keys=5000)
    one = slice(x.q_off[3], x.q_off[4])
    assert np.isnan(got[one]).all()
    got[one] = want[one]
    close(got, want, x)


def test_many_single_tokens_and_prompts_together(rng):
    keys = rng.integers(1, 60, 400)
    news = np.minimum(rng.choice([0, 1, 1, 1, 30], 400), keys)
    keys[[7, 300]], news[[7, 300]] = (2500, 2200), (1, 40)
    x = Batch(rng, keys.tolist(), news.tolist(), 4, 2, 64, 32)
    close(x.run(), x.want(), x)


def test_a_lone_draft_of_more_rows_than_a_chunk(rng):
    x = Batch(rng, [5000], [5], 16, 2, 128, 128)
    close(x.run(times=2), x.want(), x)


@pytest.mark.parametrize("new", [2, 70])
def test_sequences_with_rows_behind_the_last_are_refused(new, rng):
    """As after a plan whose tokens did not all fit: the keys of the others are missing."""
    x = Batch(rng, [100, 100], [new, new], 4, 2, 64, 64)
    want, T, H, D = x.want(), 2 * new, 4, 64
    o, ws = filled(T * H * D), B(1 << 24)
    ops.kv4_attn(B.from_array(x.q), B.from_array(x.pool), u32(x.table), u32(x.n_keys),
                 u32(x.q_off), o, 2, T - 1, new, 100, x.M, H, 2, D, x.P, 64, 0, 0, ws)
    ops.sync()
    got = o.download(T * H * D).reshape(T, H, D)
    close(got[:new], want[:new], x)
    assert np.isnan(got[new:-1]).all() and (got[-1] == 7).all()


@pytest.mark.parametrize("new", [1, 4, 64])
def test_nan_and_infinity_reach_exactly_the_rows_that_see_them(new, rng):
    """A NaN in K makes rows NaN, one in V the 32 dims of its block; rows before it,
    and rows whose window has passed it, keep their values."""
    n, D = 130, 128
    k, v = (rng.standard_normal((n, 2, D)).astype(np.float32) for _ in range(2))
    k[n - 2, 0, 3] = np.nan
    v[n - 1, 1, 40] = np.inf
    v[n - 90, 1, 100] = np.nan
    x = Batch(rng, [n], [new], 4, 2, D, 32, window=80, sinks=3, k=[k], v=[v])
    got, want = x.run(), x.want()
    close(got, want, x)
    assert np.isnan(got[-1, :2]).all() and np.isnan(got[-1, 2:, 32:64]).all()
    assert np.isfinite(got[-1, 2:, :32]).all()


def test_rows_of_q_with_nan_or_infinity_are_nan(rng):
    x = Batch(rng, [50, 60], [1, 40], 16, 8, 128, 64)
    x.q[0, 3, 7], x.q[20, 5, 0] = np.nan, np.inf
    got = x.run()
    bad = np.zeros((41, 16), bool)
    bad[0, 3] = bad[20, 5] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 30.0])
def test_small_and_large_queries(new, scale, rng):
    x = Batch(rng, [300], [new], 4, 2, 128, 64)
    x.q *= np.float32(scale)
    got, want = x.run(), x.want()
    # Scores grow with q: their error too (see close).
    tol = 1e-5 * max(1.0, scale)
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


@pytest.mark.parametrize("new", [1, 5, 90])
def test_in_place_and_again(new, rng):
    x = Batch(rng, [260, 400], [new, new], 16, 8, 128, 64)
    a = x.run(times=2)
    np.testing.assert_array_equal(a, x.run(in_place=True))


def test_weights_far_below_the_largest_count(rng):
    """One key with all the weight and thousands near nothing, whose sum shows."""
    n, D = 4000, 64
    k = np.zeros((n, 1, D), np.float32)
    k[0, 0, 0] = 8.0
    v = rng.standard_normal((n, 1, D)).astype(np.float32)
    x = Batch(rng, [n], [1], 1, 1, D, 64, k=[k], v=[v])
    x.q[:] = 0
    x.q[0, 0, 0] = 11.0  # a score of 11 against zeros
    close(x.run(), x.want(), x)


@pytest.mark.parametrize("new,D", [(1, 64), (3, 64), (40, 64), (2, 128)])
def test_nan_in_a_lone_sequences_cache(new, D, rng):
    n = 70
    k, v = (rng.standard_normal((n, 2, D)).astype(np.float32) for _ in range(2))
    v[n - new, 0, 33] = np.nan  # the first new token's own
    k[n - 1, 1, 0] = np.inf     # the last one's
    x = Batch(rng, [n], [new], 8, 2, D, 32, k=[k], v=[v])
    got, want = x.run(), x.want()
    close(got, want, x)
    assert np.isnan(got[0, 0, 32:64]).all() and np.isfinite(got[0, 0, :32]).all()
    assert np.isnan(got[-1, 4:]).all()


@pytest.mark.parametrize("new", [1, 30])
def test_a_lone_refused_sequence(new, rng):
    x = Batch(rng, [100], [new], 4, 2, 128, 32)
    assert np.isnan(x.run(max_n_keys=99)).all()
    x.n_keys = [0]
    assert not x.run(max_n_keys=99).any()


@pytest.mark.parametrize("S,new", [(700, (0, 1, 1)), (300, (1, 2, 3)), (2500, (0, 1, 9)),
                                   (70, (60, 300))])
def test_many_sequences(S, new, rng):
    """More sequences, or row tiles, than a workgroup has threads."""
    keys = rng.integers(1, 90, S)
    news = np.minimum(rng.choice(new, S), keys)
    keys[5], news[5] = 400, max(new)
    x = Batch(rng, keys.tolist(), news.tolist(), 4, 2, 64, 32)
    close(x.run(), x.want(), x)


def test_pages_behind_four_gibibytes(rng):
    """Slots whose bytes lie past 32 bits: append, read and both attentions."""
    H, G, D, page = 16, 8, 128, 256
    pb = ops.kv4_page_bytes(G, D, page)
    P = (1 << 32) // pb + 40
    pool = B(P * pb)
    n = 600
    k, v = (rng.standard_normal((n, G, D)).astype(np.float32) for _ in range(2))
    table = np.array([P - 1, P - 37, P - 2], np.uint32)
    slots = table[np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
    ops.kv4_append(B.from_array(k), B.from_array(v), u32(slots), pool, n, G, D, P, page)
    gk, gv = read_back(pool, u32(slots), n, G, D, P, page)
    kq, vq = ref.values(*ref.quantise(k)), ref.values(*ref.quantise(v))
    np.testing.assert_array_equal(gk, kq)
    np.testing.assert_array_equal(gv, vq)
    for m in (1, 20, 40):  # one token, chunks of rows, the prompt kernel
        q = rng.standard_normal((m, H, D)).astype(np.float32)
        o = filled(m * H * D)
        ws = B(max(256, ops.kv4_attn_ws_bytes(1, m, n, H, G, D)))
        ops.kv4_attn(B.from_array(q), pool, u32(table), u32([n]), u32([0, m]), o, 1, m, m, n, 3, H,
                     G, D, P, page, 0, 0, ws)
        ops.sync()
        close(o.download(m * H * D).reshape(m, H, D), ref.attention(q, kq, vq, n), None)
    pool.free()


# --------------------------------------------------------------- whole steps --
class Server:
    """A layer of a serving loop: pool, two tables and free lists that take turns, and a
    reference that keeps every sequence's values."""

    def __init__(self, rng, S, H, G, D, page, blocks, pages, tokens, window, sinks, pairing):
        self.__dict__.update(locals())
        inv = oracle.rope_inv_freq(D, 1e6)
        self.gains = [rng.normal(1, 0.1, D).astype(np.float32) for _ in range(2)]
        self.inv = inv
        self.dev = [B.from_array(x) for x in (*self.gains, inv)]
        self.pool = B.from_array(rng.integers(0, 256, pages * ops.kv4_page_bytes(G, D, page),
                                              dtype=np.uint8))
        self.table = [u32(np.full(S * blocks, ref.NONE)) for _ in range(2)]
        free = np.concatenate([[pages], rng.permutation(pages)])
        self.free = [u32(free), u32(np.zeros(pages + 1))]
        self.keys, self.new = u32(np.zeros(S)), u32(np.zeros(S))
        self.q_off, self.lost = u32(np.zeros(S + 1)), u32([0])
        self.pos, self.slots = u32(np.zeros(tokens)), u32(np.zeros(tokens))
        self.plan_ws = B(ops.kv4_plan_ws_bytes(S))
        self.raw = [B(4 * tokens * h * D) for h in (H, G, G)]
        self.qn, self.o = filled(tokens * H * D), filled(tokens * H * D)
        self.attn_ws = {}
        self.k = [np.zeros((0, G, D), np.float32) for _ in range(S)]
        self.v = [np.zeros((0, G, D), np.float32) for _ in range(S)]

    def call(self, turn, max_q):
        """The step's three calls, from table and free list `turn` to the others."""
        S, H, G, D, page = self.S, self.H, self.G, self.D, self.page
        T, W, N = self.tokens, self.window, self.sinks
        ops.kv4_plan(self.keys, self.new, self.table[turn], self.table[1 - turn], self.free[turn],
                     self.free[1 - turn], self.q_off, self.pos, self.slots, self.lost, S,
                     self.blocks, self.pages, T, page, W, N, self.plan_ws)
        ops.kv4_prologue(*self.raw, *self.dev, EPS, self.pairing, self.pos, self.slots, self.qn,
                         self.pool, T, H, G, D, self.pages, page)
        most = self.blocks * page
        if max_q not in self.attn_ws:
            self.attn_ws[max_q] = B(max(256, ops.kv4_attn_ws_bytes(S, max_q, most, H, G, D, W, N)))
        ops.kv4_attn(self.qn, self.pool, self.table[1 - turn], self.keys, self.q_off, self.o, S, T,
                     max_q, most, self.blocks, H, G, D, self.pages, page, W, N,
                     self.attn_ws[max_q])

    def lengths(self, keep, new):
        """keep[b]: keys kept of sequence b; new[b] more follow. Uploads lengths and rows."""
        T, D = self.tokens, self.D
        total = int(np.sum(new))
        raw = [self.rng.standard_normal((T, h, D)).astype(np.float32)
               for h in (self.H, self.G, self.G)]
        pos = np.concatenate([np.arange(a, a + m) for a, m in zip(keep, new)]).astype(np.int64)
        at = np.concatenate([[0], np.cumsum(new)])
        kn = raw[1][:total].copy()
        qn = raw[0][:total].copy()
        for t in range(total):
            for x, g in ((qn, self.gains[0]), (kn, self.gains[1])):
                y = oracle.rmsnorm(x[t].ravel(), g, D, x.shape[1], EPS)
                x[t] = oracle.rope(y, 1, x.shape[1], D, int(pos[t]), self.inv,
                                   self.pairing).reshape(-1, D)
        for b in range(self.S):
            s = slice(at[b], at[b + 1])
            kq, vq = (ref.values(*ref.quantise(x[s])) for x in (kn, raw[2]))
            self.k[b] = np.concatenate([self.k[b][:keep[b]], kq])
            self.v[b] = np.concatenate([self.v[b][:keep[b]], vq])
        self.at, self.q_ref = at, qn
        self.keys.upload(np.array([len(x) for x in self.k], np.uint32))
        self.new.upload(np.array(new, np.uint32))
        for buf, x in zip(self.raw, raw):
            buf.upload(x)

    def check(self):
        ops.sync()
        total, H, D = self.at[-1], self.H, self.D
        assert self.lost.download(1, np.uint32)[0] == 0
        np.testing.assert_array_equal(self.qn.download(total * H * D).reshape(total, H, D),
                                      self.q_ref)
        got = self.o.download(total * H * D).reshape(total, H, D)
        want = np.concatenate([ref.attention(self.q_ref[self.at[b]:self.at[b + 1]], self.k[b],
                                             self.v[b], len(self.k[b]), self.window, self.sinks)
                               for b in range(self.S)])
        close(got, want, None)
        return got


STEPS = [([0, 0, 0, 0], [40, 0, 7, 1]),      # prompts, one sequence waits
         ([40, 0, 7, 1], [1, 33, 1, 1]),     # a prompt beside single tokens
         ([41, 33, 8, 2], [4, 4, 4, 4]),     # drafts
         ([42, 37, 8, 5], [1, 1, 1, 1]),     # some of them taken back
         ([0, 38, 9, 6], [20, 1, 0, 1]),     # one ends and another begins, one idles
         ([20, 39, 9, 7], [1, 1, 1, 1])]


@pytest.mark.parametrize("H,G,D,page,window,sinks,pairing", [
    (4, 2, 128, 32, 0, 0, "neox"), (8, 2, 64, 32, 20, 3, "norm")])
def test_a_serving_loop(H, G, D, page, window, sinks, pairing, rng):
    s = Server(rng, 4, H, G, D, page, 4, 16, 80, window, sinks, pairing)
    for i, (keep, new) in enumerate(STEPS):
        s.lengths(keep, new)
        s.call(i % 2, max(new))
        s.check()


def test_a_serving_loop_from_captured_graphs(rng):
    """Two graphs take turns (from one table and free list to the other and back); each
    is replayed several times, with eager work between, and every replay is checked."""
    s = Server(rng, 4, 4, 2, 128, 32, 4, 16, 80, 24, 2, "neox")
    eager = Server(np.random.default_rng(0), 2, 4, 2, 128, 32, 4, 8, 8, 0, 0, "neox")
    stream = ops.Stream()
    ops.set_stream(stream)
    try:
        graphs = []
        for max_q in (40, 4):  # prompts, and few rows
            for turn in range(2):
                s.attn_ws.setdefault(max_q, B(max(256, ops.kv4_attn_ws_bytes(
                    4, max_q, 128, 4, 2, 128, 24, 2))))
                with ops.Graph() as g:
                    s.call(turn, max_q)
                graphs.append(g)
        for i, (keep, new) in enumerate(STEPS * 2):
            if i == len(STEPS):
                keep = [0, 0, 0, 0]
            s.lengths(keep, new)
            graphs[(0 if max(new) > 4 else 2) + i % 2].launch()
            s.check()
            eager.lengths([0, 0], [1, 4])
            eager.call(0, 4)
            eager.check()
        for g in graphs:
            g.free()
    finally:
        ops.sync()
        ops.set_stream(None)
        stream.free()


def test_a_captured_mixed_batch_follows_its_lengths(rng):
    """One graph (both kernels, pieces from a list) replayed as sequences shrink, grow back
    and go: every replay against the formula."""
    H, G, D, page = 4, 2, 64, 32
    keys = rng.integers(200, 700, 300)
    news = rng.choice([1, 1, 1, 70], 300)
    keys[[9, 200]], news[[9, 200]] = (3000, 2600), (1, 200)
    x = Batch(rng, keys.tolist(), news.tolist(), H, G, D, page)
    o, q = filled(x.T * H * D), B.from_array(x.q)
    ws = B(ops.kv4_attn_ws_bytes(x.S, 200, 3000, H, G, D))
    pool, table, n_keys, q_off = B.from_array(x.pool), u32(x.table), u32(keys), u32(x.q_off)
    stream = ops.Stream()
    ops.set_stream(stream)
    try:
        with ops.Graph() as g:
            ops.kv4_attn(q, pool, table, n_keys, q_off, o, x.S, x.T, 200, 3000, x.M, H, G, D, x.P,
                         page, 0, 0, ws)
        for less in (0, 100, 130, 0):
            now = np.where(np.arange(300) % 2 == 0, keys - less, keys)
            n_keys.upload(now.astype(np.uint32))
            g.launch()
            ops.sync()
            got = o.download(x.T * H * D).reshape(x.T, H, D)
            want = np.concatenate([
                ref.attention(x.q[a:a + m], x.k[b][:n], x.v[b][:n], n)
                for b, (n, m, a) in enumerate(zip(now.tolist(), x.n_new, x.q_off))])
            close(got, want, x)
        g.free()
    finally:
        ops.sync()
        ops.set_stream(None)
        stream.free()


def test_two_streams_at_once(rng):
    """Two batches with workspaces of their own on two streams: each one's bits are those
    of the call alone."""
    xs = [Batch(rng, [900, 33, 500], [m] * 3, 16, 8, 128, 64) for m in (1, 30)]
    alone = [x.run(extra=0) for x in xs]
    H, G, D, page, window, sinks = xs[0].shape
    streams = [ops.Stream(), ops.Stream()]
    held, outs = [], []
    for x, st in zip(xs, streams):
        m = max(x.n_new)
        o = filled(x.T * H * D)
        ws = B(max(256, ops.kv4_attn_ws_bytes(3, m, 900, H, G, D)))
        held.append([B.from_array(x.q), B.from_array(x.pool), u32(x.table), u32(x.n_keys),
                     u32(x.q_off), o, ws])
        outs.append(o)
    ops.sync()
    try:
        for _ in range(4):
            for x, st, h in zip(xs, streams, held):
                ops.set_stream(st)
                ops.kv4_attn(*h[:6], 3, x.T, max(x.n_new), 900, x.M, H, G, D, x.P, page, 0, 0,
                             h[6])
        for st in streams:
            ops.set_stream(st)
            ops.sync()
    finally:
        ops.set_stream(None)
    for o, want, x in zip(outs, alone, xs):
        np.testing.assert_array_equal(o.download(x.T * H * D).reshape(x.T, H, D), want)
    for st in streams:
        st.free()
