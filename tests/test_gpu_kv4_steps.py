"""Steps of the paged 4-bit cache (plan, prologue, attention) that lose keys: rows that would
see one are NaN until it is new again, the others are right."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref as ref
from flock_amd import ops
from test_gpu_kv4 import B, Server, check_plan, close

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

    def check(self, turn, new):
        """Returns, for each sequence, whether its rows are numbers."""
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
            close(got[rows], want, None)
            numbers.append(bool(np.isfinite(want).all()) if m else None)
        return numbers

    def step(self, turn, keep, new, max_q):
        self.lengths(keep, new)
        self.expect(new)
        self.call(turn, max_q)
        return self.check(turn, new)


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
