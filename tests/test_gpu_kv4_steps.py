"""Steps of the paged 4-bit cache (plan, prologue, attention) that lose keys: rows that would
see one are NaN until it is new again, the others are right."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref as ref
from flock_amd import ops
from test_gpu_kv4 import B, Batch, Server, check_plan, close, u32

pytestmark = pytest.mark.gpu


class Losing(Server):
    """A Server beside the reference's table: what is not in it reads as NaN."""

    def __init__(self, *args):
        super().__init__(*args)
        self.want_table = np.full((self.S, self.blocks), ref.NONE, np.uint32)
        self.want_free = self.free[0].download(1 + self.pages, np.uint32)[1:].tolist()

    def expect(self, new):
        keys = [len(x) for x in self.k]
        self.want_table, self.want_free, _, _, _, self.want_lost = ref.plan(
            keys, new, self.want_table, self.want_free, self.tokens, self.pages, self.page,
            self.window, self.sinks)

    def check(self, turn, new, limit=None):
        """Returns, for each sequence, whether its rows are numbers."""
        limit = limit or self.tokens
        ops.sync()
        H, D = self.H, self.D
        np.testing.assert_array_equal(
            self.table[1 - turn].download(self.S * self.blocks, np.uint32), self.want_table.ravel())
        assert self.lost.download(1, np.uint32)[0] == self.want_lost
        got = self.o.download(self.tokens * H * D).reshape(-1, H, D)
        numbers = []
        for b, m in enumerate(new):
            rows = slice(self.at[b], self.at[b + 1])
            n = len(self.k[b])
            want = ref.attention(self.q_ref[rows], self.k[b], self.v[b], n, self.window, self.sinks)
            there = self.want_table[b][np.arange(n) // self.page] < self.pages
            for i in range(m):
                j, p = np.arange(n), n - m + i
                seen = j <= p
                if self.window:
                    seen &= (j > p - self.window) | (j < self.sinks)
                if not there[seen].all():
                    want[i] = np.nan
            refused = self.at[b + 1] > limit
            if refused:
                want = np.full((max(0, limit - self.at[b]), H, D), np.nan)
                rows = slice(self.at[b], self.at[b] + len(want))
            close(got[rows], want, None)
            numbers.append(bool(np.isfinite(want).all()) and not refused if m else None)
        return numbers

    def step(self, turn, keep, new, max_q, limit=None):
        """limit: rows of the step's arrays."""
        self.lengths(keep, new)
        whole, self.tokens = self.tokens, limit or self.tokens
        self.expect(new)
        self.call(turn, max_q)
        self.tokens = whole
        return self.check(turn, new, limit)


# (kept keys, new ones), and whose rows are numbers.
DRY = [([0, 0], [32, 32], [True, True]),
       ([32, 32], [1, 0], [False, None]),   # no page for it
       ([33, 0], [1, 0], [False, None]),    # the other's comes free
       ([34, 0], [1, 0], [False, None]),
       ([35, 0], [30, 0], [False, None]),   # past the missing block
       ([65, 0], [1, 0], [False, None]),
       ([0, 0], [40, 0], [False, None]),    # its last page is taken from the next step on
       ([0, 0], [40, 0], [True, None]),     # all of it new
       ([40, 0], [1, 0], [True, None])]
BACK = [([0, 0], [70, 40], [True, True]), ([70, 40], [1, 1], [True, True]),
        ([71, 41], [50, 2], [True, True]), ([121, 43], [1, 1], [True, True]),
        ([70, 44], [1, 1], [False, True]),  # behind what the window left
        ([71, 45], [3, 1], [False, True]), ([74, 46], [22, 0], [False, None]),
        ([96, 46], [31, 1], [True, True]),  # keys from 65 on, in the block that it still had
        ([127, 47], [1, 1], [True, True])]


# ... and the rows of the step's arrays.
OVER = [([0, 0, 0], [40, 33, 20], [True, True, True], 93),
        ([40, 33, 20], [1, 1, 1], [True, True, False], 2),
        ([41, 34, 21], [1, 2, 1], [True, True, False], 4),   # past the one that was not stored
        ([42, 36, 0], [30, 30, 22], [True, False, False], 55),
        ([72, 66, 22], [1, 1, 0], [True, False, None], 2),
        ([72, 32, 0], [2, 5, 24], [True, True, True], 31),
        ([74, 37, 24], [1, 30, 1], [True, False, False], 12),
        ([75, 48, 24], [0, 30, 1], [None, True, True], 31),  # from the first not stored on
        ([75, 78, 25], [1, 1, 1], [True, True, True], 3)]


@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (8, 2, 64)])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_tokens_past_the_arrays_are_not_seen(H, G, D, rows, rng):
    s = Losing(rng, 3, H, G, D, 32, 8, 24, 120, 0, 0, "neox")
    for i, (keep, new, want, limit) in enumerate(OVER):
        assert s.step(i % 2, keep, new, max(new) if rows == "few" else 120, limit) == want, i


@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (8, 2, 64)])
@pytest.mark.parametrize("steps,pages,window,sinks", [(DRY, 2, 0, 0), (DRY, 2, 500, 3),
                                                      (BACK, 16, 32, 0)])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_keys_that_were_not_stored_are_not_seen(H, G, D, steps, pages, window, sinks, rows, rng):
    s = Losing(rng, 2, H, G, D, 32, 8, pages, 120, window, sinks, "neox")
    for i, (keep, new, want) in enumerate(steps):
        assert s.step(i % 2, keep, new, max(new) if rows == "few" else 120) == want, i


def test_keys_that_were_not_stored_are_not_seen_by_captured_steps(rng):
    """The two graphs that take turns, replayed through both ways to lose keys."""
    for steps, pages, window in ((DRY, 2, 0), (BACK, 16, 32)):
        s = Losing(rng, 2, 4, 2, 128, 32, 8, pages, 120, window, 0, "norm")
        stream = ops.Stream()
        ops.set_stream(stream)
        try:
            s.attn_ws[120] = B(max(256, ops.kv4_attn_ws_bytes(2, 120, 256, 4, 2, 128, window)))
            graphs = []
            for turn in range(2):
                with ops.Graph() as g:
                    s.call(turn, 120)
                graphs.append(g)
            for i, (keep, new, want) in enumerate(steps):
                s.lengths(keep, new)
                s.expect(new)
                graphs[i % 2].launch()
                assert s.check(i % 2, new) == want, i
            for g in graphs:
                g.free()
        finally:
            ops.sync()
            ops.set_stream(None)
            stream.free()


@pytest.mark.parametrize("S,M", [(5, 7), (16, 130), (17, 65), (700, 9)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3), (1, 0)])
def test_plans_that_run_dry_equal_the_reference(S, M, window, sinks, rng):
    """Few pages, lengths taken back by any number, entries of the caller's own."""
    page, n_pages = 32, max(1, S * M // 5)
    table = np.full((S, M), ref.NONE, np.uint32)
    free = rng.permutation(n_pages).tolist()
    keys, lost = np.zeros(S, np.int64), 0
    for step in range(8):
        new = rng.choice([0, 1, 4, page, M * page // 2], S)
        what = rng.random(S)
        keys = np.where(what < 0.1, 0, np.where(what < 0.3, keys * rng.random(S), keys + new))
        keys = np.minimum(keys.astype(np.int64), M * page + 5)
        new = np.minimum(new, keys)
        tokens = max(1, int(new.sum()) + (step % 3) * 5)
        table, free, *_, count = check_plan(keys, new, table, free, tokens, n_pages, page, window,
                                            sinks, in_place=step % 2 == 1)
        lost += count
    assert lost > 0


@pytest.mark.parametrize("S,M", [(1, 4), (16, 70), (17, 5), (1300, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3), (1, 40)])
def test_plans_of_more_tokens_than_rows_equal_the_reference(S, M, window, sinks, rng):
    page, n_pages = 32, S * M + 1
    table = np.full((S, M), ref.NONE, np.uint32)
    free = rng.permutation(n_pages).tolist()
    keys, marked = np.zeros(S, np.int64), 0
    for step in range(8):
        new = rng.choice([0, 1, 4, page, M * page // 2], S)
        keys = np.minimum(np.where(rng.random(S) < 0.1, 0, keys + new), M * page + 5)
        new = np.minimum(new, keys)
        tokens = max(1, int(new.sum() * (1, 0.4, 0.9)[step % 3]) - step % 2)
        table, free, *_ = check_plan(keys, new, table, free, tokens, n_pages, page, window, sinks,
                                     in_place=step % 2 == 1)
        marked += ((table >= 1 << 31) & (table != ref.NONE)).sum()
    assert S == 1 or marked > 0


def test_marks_of_a_pool_of_more_than_two_to_the_31_slots():
    n_pages, table = 1 << 26, np.full((2, 3), ref.NONE, np.uint32)
    free = [5, n_pages - 2, 0, n_pages - 1, 77]
    for keys, new, tokens, want in (([70, 20], [70, 20], 41, 49),
                                    ([70, 25], [29, 25], 54, 24),  # of 41 its even neighbour
                                    ([71, 26], [31, 1], 32, 0), ([72, 27], [1, 1], 2, 0)):
        table, free, _, _, _, lost = check_plan(keys, new, table, free, tokens, n_pages, 32, 0, 0)
        assert lost == want
    assert free == [5] and table[0].tolist() == [77, n_pages - 1, 0]


def test_a_captured_mixed_batch_as_sequences_end_begin_and_change(rng):
    """One graph (both kernels, pieces from lists) whose lengths and rows all change: sequences
    end and come back, prompts become single tokens and single tokens prompts, row tiles that
    were cut are whole and cut again. Rows of no sequence stay as they were."""
    H, G, D, page, S, T = 4, 2, 64, 32, 300, 6000
    most = rng.integers(80, 500, S)
    most[[9, 200, 250]] = 3000, 2600, 2200
    x = Batch(rng, most.tolist(), [1] * S, H, G, D, page)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    dq, o = B.from_array(q), B(4 * T * H * D)
    ws = B(ops.kv4_attn_ws_bytes(S, 200, 3000, H, G, D))
    pool, table, n_keys, q_off = B.from_array(x.pool), u32(x.table), u32(most), u32([0] * (S + 1))
    stream = ops.Stream()
    ops.set_stream(stream)
    try:
        with ops.Graph() as g:
            ops.kv4_attn(dq, pool, table, n_keys, q_off, o, S, T, 200, 3000, x.M, H, G, D, x.P,
                         page, 0, 0, ws)
        for i in range(5):
            keys = np.where(rng.random(S) < 0.2, 0, most - rng.integers(0, 80, S))
            news = np.minimum(rng.choice([0, 1, 1, 1, 1, 1, 2, 2, 40, 70], S), keys)
            if i % 2 == 0:  # a long prompt, a chunk and a single token, all far on
                keys[[9, 200, 250]] = most[[9, 200, 250]]
                news[[9, 200, 250]] = (1, 200, 64) if i < 4 else (200, 1, 64)
            else:
                keys[[9, 200, 250]], news[[9, 200, 250]] = (90, 2000, 0), (70, 1, 0)
            off = np.concatenate([[0], np.cumsum(news)])
            assert off[-1] < T
            n_keys.upload(keys.astype(np.uint32))
            q_off.upload(off.astype(np.uint32))
            o.upload(np.full(T * H * D, 7, np.float32))
            g.launch()
            ops.sync()
            got = o.download(T * H * D).reshape(T, H, D)
            want = np.concatenate([
                ref.attention(q[a:a + m], x.k[b][:n], x.v[b][:n], n)
                for b, (n, m, a) in enumerate(zip(keys.tolist(), news.tolist(), off.tolist()))])
            assert (got[off[-1]:] == 7).all()
            close(got[:off[-1]], want, x)
        g.free()
    finally:
        ops.sync()
        ops.set_stream(None)
        stream.free()


@pytest.mark.parametrize("below", [17.3, 20.5, 26.3])
@pytest.mark.parametrize("H,m", [(1, 1), (8, 7)])  # the kernel for few rows, and for prompts
def test_a_million_equal_weights_far_below_the_largest(below, H, m):
    """A key of weight 1 and value 0, and 2^20 of weight 2^-below and value 1. Weights are held
    as 2^10 and less in two f16 parts, the second of them to half of 2^-24: 2^-35 of the largest
    for each key. 1e-5 for the rest (see close)."""
    n, D, page = 1 << 20, 64, 256
    k, v = np.zeros((n, 1, D), np.float32), np.ones((n, 1, D), np.float32)
    k[0, 0, 0], v[0] = 8, 0
    q = np.zeros((m, H, D), np.float32)
    q[..., 0] = below * np.log(2)  # over sqrt(64), times 8
    P = n // page
    pool, ids = B(P * ops.kv4_page_bytes(1, D, page)), u32(np.arange(P))
    slots, dk, dv = u32(np.arange(n)), B.from_array(k), B.from_array(v)
    ops.kv4_append(dk, dv, slots, pool, n, 1, D, P, page)
    o, ws = B(4 * q.size), B(ops.kv4_attn_ws_bytes(1, m, n, H, 1, D))
    ops.kv4_attn(B.from_array(q), pool, ids, u32([n]), u32([0, m]), o, 1, m, m, n, P, H, 1, D, P,
                 page, 0, 0, ws)
    ops.sync()
    got = o.download(q.size).reshape(m, H * D).astype(np.float64)
    weight = np.exp(-q[0, 0, 0].astype(np.float64))
    for i in range(m):
        others = n - m + i
        want = others * weight / (1 + others * weight)
        assert np.abs(got[i] - want).max() <= others * 2.0 ** -35 + 1e-5 * want
