"""Plans of the paged 4-bit cache over many steps, without a GPU: what the table of the
reference plan (which the GPU's equals entry by entry) lets attention read is what the
sequence itself stored."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref as ref


class Slots:
    """A pool that remembers, for each slot, which row of which step it holds: what each step's
    prologue stored, through plan after plan."""

    def __init__(self, S, M, page, n_pages, window=0, sinks=0):
        self.M, self.page, self.n_pages, self.window, self.sinks = M, page, n_pages, window, sinks
        self.table = np.full((S, M), ref.NONE, np.uint32)
        self.free = list(range(n_pages))
        self.holds = {}
        self.rows = [{} for _ in range(S)]  # by key: the row that it was new in, last
        self.steps = self.lost = 0

    def step(self, keys, new, max_tokens=None):
        """Returns, for each sequence, whether attention gives numbers (no new row sees a key
        without a page), or None where it has no rows or is refused."""
        S, page = len(keys), self.page
        T = max(1, sum(new)) if max_tokens is None else max_tokens
        self.steps += 1
        self.table, self.free, q_off, pos, slots, self.lost = ref.plan(
            keys, new, self.table, self.free, T, self.n_pages, page, self.window, self.sinks)
        ids = [ref.unmark(int(e), self.n_pages, page)[0] for e in self.table.ravel()]
        held = [e for e in ids if e < self.n_pages] + self.free
        assert sorted(held) == list(range(self.n_pages)), "a page lost, or twice"
        for b in range(S):
            for i in range(new[b]):
                t, j = q_off[b] + i, keys[b] - new[b] + i
                self.rows[b][j] = (self.steps, t)
                if t < T and slots[t] != ref.NONE:
                    assert pos[t] == j
                    self.holds[slots[t]] = (self.steps, t)
        return [self.sees_only_its_own(b, keys[b], new[b]) if
                new[b] and q_off[b + 1] <= T and keys[b] <= self.M * page else None
                for b in range(S)]

    def sees_only_its_own(self, b, n, m):
        numbers = True
        for j in range(n):
            if self.window and j >= self.sinks and j <= n - m - self.window:
                continue  # no new row sees it
            entry = int(self.table[b, j // self.page])
            if entry >= self.n_pages:
                numbers = False
                continue
            got = self.holds.get(entry * self.page + j % self.page)
            assert got == self.rows[b][j], (b, n, m, j, got)
        return numbers


def test_pages_that_come_free_after_a_loss_go_to_no_block_with_keys_before():
    s = Slots(2, 4, 32, 2)
    assert s.step([32, 32], [32, 32]) == [True, True]
    assert s.step([33, 32], [1, 0]) == [False, None] and s.lost == 1
    assert s.step([34, 0], [1, 0])[0] is False and s.lost > 0   # the other's page comes free
    assert s.step([35, 0], [1, 0])[0] is False and s.lost > 0
    # The block after it is the sequence's again, and the missing one still counts.
    assert s.step([65, 0], [30, 0])[0] is False and s.lost > 0
    assert s.step([66, 0], [1, 0])[0] is False and s.lost > 0
    s.step([0, 0], [0, 0])
    assert s.step([66, 0], [66, 0])[0] is False  # three blocks of two pages
    assert s.step([60, 0], [60, 0])[0] is True and s.lost == 0


def test_a_sequence_that_lost_everything():
    s = Slots(2, 2, 32, 1)
    assert s.step([20, 11], [20, 11]) == [True, False] and s.lost == 11
    s.step([0, 11], [0, 0])
    assert s.step([0, 12], [0, 1])[1] is False and s.lost > 0
    assert s.step([0, 13], [0, 13])[1] is True and s.lost == 0  # all of it new


def test_keys_after_a_loss_planned_again_as_new():
    s = Slots(2, 4, 32, 3)
    s.step([64, 32], [64, 32])
    assert s.step([70, 32], [6, 0])[0] is False and s.lost == 6
    s.step([70, 0], [0, 0])
    assert s.step([71, 0], [1, 0])[0] is False
    assert s.step([72, 0], [7, 0])[0] is False  # not all of the block's keys
    assert s.step([72, 0], [8, 0])[0] is True and s.lost == 0


def test_lengths_taken_back_behind_the_window():
    s = Slots(1, 8, 32, 8, window=64)
    assert s.step([200], [200]) == [True]
    assert s.step([201], [1]) == [True]           # keys below 137 are given back
    assert s.step([150], [1]) == [False] and s.lost > 0
    for n in range(151, 193):
        assert s.step([n], [1])[0] is (n >= 192)  # from 128 on, which is its own
    assert s.lost == 0
    assert s.step([150], [150]) == [True] and s.lost == 0


def test_a_window_of_one_sees_no_key_that_was_lost():
    s = Slots(2, 4, 32, 2, window=1)
    assert s.step([32, 32], [32, 32]) == [True, True]
    assert s.step([33, 33], [1, 1]) == [False, False] and s.lost == 2
    assert s.step([34, 34], [1, 1]) == [True, True] and s.lost == 0  # their first pages came back
    assert s.step([36, 36], [2, 2], max_tokens=1) == [None, None] and s.lost == 3
    assert s.step([37, 37], [1, 1]) == [True, True] and s.lost == 0
    s = Slots(1, 4, 32, 1, window=1, sinks=33)
    s.step([32], [32])
    assert s.step([33], [1]) == [False] and s.step([34], [1]) == [False]  # a sink was lost


def test_drafts_taken_back_never_reach_behind_the_window():
    """Verified tokens and a draft in turn: what a step keeps is what the next one sees."""
    s = Slots(1, 20, 32, 20, window=40, sinks=3)
    rng = np.random.default_rng(3)
    n = 90
    assert s.step([n], [n]) == [True]
    while n < 600:
        draft = int(rng.integers(1, 9))
        assert s.step([n + draft], [draft]) == [True] and s.lost == 0
        n += int(rng.integers(0, draft + 1))


@pytest.mark.parametrize("seed", range(30))
def test_random_steps_read_only_what_was_stored(seed):
    rng = np.random.default_rng(seed)
    S, M, page = int(rng.integers(1, 6)), int(rng.integers(1, 7)), 32
    window, sinks = (0, 0) if seed % 2 else (int(rng.integers(1, 90)), int(rng.integers(0, 50)))
    s = Slots(S, M, page, int(rng.integers(1, S * M + 2)), window, sinks)
    keys = np.zeros(S, int)
    numbers = 0
    for _ in range(80):
        new = rng.choice([0, 1, 1, 5, 33, M * page // 2], S)
        what = rng.random(S)
        back = keys - rng.integers(0, 70, S)
        keys = np.where(what < 0.08, 0, np.where(what < 0.25, np.maximum(back, 0), keys)) + new
        fit = keys <= M * page + 3
        new, keys = np.where(fit, new, 0), np.where(fit, keys, 0)
        if rng.random() < 0.2:  # planned anew, from its first token
            b = int(rng.integers(0, S))
            new[b] = keys[b]
        got = s.step(keys.tolist(), new.tolist())
        numbers += sum(x is True for x in got)
        if s.lost == 0:
            assert False not in got
    assert numbers > 0


@pytest.mark.parametrize("n_pages,page", [(1, 32), (100, 256), ((1 << 26) - 1, 32), (1 << 26, 32),
                                          ((1 << 27) - 1, 32), ((1 << 24) - 1, 256)])
def test_marks_of_pages_are_no_pages_and_come_back(n_pages, page):
    assert ref.unmark(ref.NONE, n_pages, page)[0] >= n_pages
    for page_id in {0, n_pages // 3, n_pages // 2, n_pages - 1}:
        for key in range(page):
            e = ref.mark(page_id, key, n_pages, page)
            got = ref.unmark(e, n_pages, page)
            assert n_pages <= e < ref.NONE and got[0] == page_id
            assert got[1] == (key & ~1 if n_pages * page >= 1 << 31 else key)


def test_rows_past_the_arrays_leave_nothing_to_be_read():
    s = Slots(2, 4, 32, 8)
    s.step([40, 40], [40, 40])
    assert s.step([41, 41], [1, 1], max_tokens=1) == [True, None] and s.lost == 1
    assert s.step([42, 42], [1, 1]) == [True, False] and s.lost > 0
    assert s.step([43, 43], [1, 2]) == [True, False] and s.lost > 0
    assert s.step([44, 44], [1, 4]) == [True, True] and s.lost == 0  # from the lost one on


def test_rows_past_the_arrays_planned_again():
    s = Slots(2, 4, 32, 8)
    s.step([40, 40], [40, 40])
    assert s.step([75, 75], [35, 35], max_tokens=50) == [True, None] and s.lost == 20
    assert s.step([75, 75], [0, 35]) == [None, True] and s.lost == 0


def test_a_prompt_past_the_arrays_goes_on_from_what_was_stored():
    s = Slots(1, 4, 32, 4)
    assert s.step([100], [100], max_tokens=70) == [None] and s.lost == 30
    assert s.step([100], [30]) == [True] and s.lost == 0
    s = Slots(1, 4, 32, 4)
    assert s.step([100], [100], max_tokens=70) == [None]
    assert s.step([101], [30]) == [False] and s.lost > 0  # one was left out
    s = Slots(1, 4, 32, 4)
    assert s.step([100], [100], max_tokens=70) == [None]
    assert s.step([65], [1]) == [True] and s.step([66], [1]) == [True] and s.lost == 0


@pytest.mark.parametrize("seed", range(30))
def test_random_steps_of_more_tokens_than_rows(seed):
    rng = np.random.default_rng(100 + seed)
    S, M, page = int(rng.integers(1, 6)), int(rng.integers(1, 7)), 32
    window, sinks = (0, 0) if seed % 2 else (int(rng.integers(1, 90)), int(rng.integers(0, 50)))
    s = Slots(S, M, page, int(rng.integers(S * M // 2 + 1, S * M + 2)), window, sinks)
    keys = np.zeros(S, int)
    numbers = 0
    for _ in range(80):
        new = rng.choice([0, 1, 1, 5, 33], S)
        keys = np.where(rng.random(S) < 0.1, 0, keys) + new
        fit = keys <= M * page
        new, keys = np.where(fit, new, 0), np.where(fit, keys, 0)
        short = rng.random() < 0.3
        got = s.step(keys.tolist(), new.tolist(),
                     max(1, int(new.sum()) - int(rng.integers(1, 40))) if short else None)
        numbers += sum(x is True for x in got)
        if s.lost == 0:
            assert False not in got
    assert numbers > 0


@pytest.mark.parametrize("window", [1, 2, 31, 33])
@pytest.mark.parametrize("sinks", [0, 1, 33])
def test_random_steps_with_narrow_windows(window, sinks):
    """Pages run out, rows are short and lengths are taken back, all at once."""
    for seed in range(6):
        rng = np.random.default_rng(seed)
        S, M, page = 4, 6, 32
        s = Slots(S, M, page, 9, window, sinks)
        keys = np.zeros(S, int)
        numbers = 0
        for _ in range(80):
            new = rng.choice([0, 1, 1, 5, 40], S)
            what = rng.random(S)
            back = np.maximum(keys - rng.integers(0, 70, S), 0)
            keys = np.where(what < 0.08, 0, np.where(what < 0.2, back, keys)) + new
            fit = keys <= M * page
            new, keys = np.where(fit, new, 0), np.where(fit, keys, 0)
            short = int(rng.integers(1, 40)) * (rng.random() < 0.2)
            got = s.step(keys.tolist(), new.tolist(), max(1, int(new.sum()) - short))
            numbers += sum(x is True for x in got)
            if s.lost == 0:
                assert False not in got
        assert numbers > 0
