"""Decode attention over shared prefixes on the GPU, through the C ABI, against 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest

import oracle
from flock_amd import ops

pytestmark = pytest.mark.gpu
B = ops.DeviceBuffer
EPS = oracle.QWEN3_EPS
NAN = float("nan")


def dev(a, dtype=np.float32):
    return B.from_array(np.ascontiguousarray(a, dtype).ravel())


class Batch:
    """Sequences in groups: prefix[g] shared keys, own[g] the own keys of each of group g's
    sequences; `before` and `after` sequences belong to no group. Rows that nobody sees hold
    `junk`."""

    def __init__(self, rng, prefix, own, heads=16, kv=8, d=128, before=(), after=(), gap=3,
                 junk=NAN, q_scale=1.0, k_scale=1.0, v_scale=1.0, max_prefix=None,
                 max_n_keys=None):
        self.H, self.G, self.d = heads, kv, d
        self.prefix = list(prefix)
        self.n_keys = list(before) + [n for g in own for n in g] + list(after)
        off = [len(before)]
        for g in own:
            off.append(off[-1] + len(g))
        self.off, self.S = off, len(self.n_keys)
        row, self.prefix_row, self.own_row = gap, [], []
        for n in self.prefix:
            self.prefix_row.append(row)
            row += n + gap
        for n in self.n_keys:
            self.own_row.append(row)
            row += n + gap
        self.k = np.full((row + 64, kv, d), junk, np.float32)
        self.v = np.full((row + 64, kv, d), junk, np.float32)
        for at, n in zip(self.prefix_row + self.own_row, self.prefix + self.n_keys):
            self.k[at:at + n] = rng.standard_normal((n, kv, d), np.float32) * k_scale
            self.v[at:at + n] = rng.standard_normal((n, kv, d), np.float32) * v_scale
        self.q = rng.standard_normal((self.S, heads, d), np.float32) * np.float32(q_scale)
        self.max_prefix = max(self.prefix + [0]) if max_prefix is None else max_prefix
        self.max_n_keys = max(self.n_keys + [0]) if max_n_keys is None else max_n_keys

    def group(self, b):
        for g in range(len(self.prefix)):
            if self.off[g] <= b < self.off[g + 1]:
                return g
        return None

    def rows(self, b):
        g = self.group(b)
        p = [] if g is None else range(self.prefix_row[g], self.prefix_row[g] + self.prefix[g])
        return list(p) + list(range(self.own_row[b], self.own_row[b] + self.n_keys[b]))

    def shape(self):
        return (len(self.prefix), self.S, self.max_prefix, self.max_n_keys, self.H, self.G, self.d)

    def arrays(self):
        return (dev(self.prefix_row, np.uint64), dev(self.prefix, np.uint32),
                dev(self.off, np.uint32), dev(self.own_row, np.uint64),
                dev(self.n_keys, np.uint32))

    def ws(self):
        return B(max(256, ops.decode_shared_ws_bytes(*self.shape())))

    def run(self, in_place=False):
        q = dev(self.q)
        o = q if in_place else dev(np.full(self.q.size, 7))
        ops.attn_decode_shared(q, dev(self.k), dev(self.v), *self.arrays(), o, *self.shape(),
                               self.ws())
        ops.sync()
        return o.download(self.q.size).reshape(self.q.shape)

    def want(self, seqs=None, q=None):
        """(o in 64 bits, how far each row may be off).

        A product's operands are off by 2^-22 each and the product of their second
        parts (2^-22) is left out; sums of d products and of a row's weights pass
        through fewer than d / 4 + 32 rounded f32 additions in turn. So a score is off by
        at most e = (3 * 2^-22 + (d / 4 + 32) 2^-24) sum |q_i k_i| / sqrt(d) and by 2^-24
        of itself, a weight by a factor of 1 + 2 e + 2^-20 (its exponential, its parts, its
        scaling between partial results), and so is the sum; values count with 2^-22
        and the sums above again."""
        d, m = self.d, self.H // self.G
        q = self.q if q is None else q
        o = np.zeros(q.shape)
        tol = np.zeros(q.shape[:2])
        for b in range(self.S) if seqs is None else seqs:
            r = self.rows(b)
            if not r:
                continue
            for h in range(self.H):
                k = self.k[r, h // m].astype(np.float64)
                v = self.v[r, h // m].astype(np.float64)
                x = q[b, h].astype(np.float64)
                s = k @ x / math.sqrt(d)
                size = (np.abs(k) @ np.abs(x)).max() / math.sqrt(d)
                w = np.exp(s - s.max())
                w /= w.sum()
                o[b, h] = w @ v
                chain = (d / 4 + 32) * 2.0 ** -24
                e = (3 * 2.0 ** -22 + chain) * size + 2.0 ** -24 * np.abs(s).max()
                tol[b, h] = (4 * e + 2.0 ** -19 + chain) * np.abs(v).max()
        return o, tol[..., None]

    def check(self, **kw):
        got = self.run(**kw)
        o, tol = self.want()
        err = np.abs(got - o)
        assert np.isfinite(got).all()
        assert (err <= tol).all(), (err.max(), np.argwhere(err > tol)[:5])
        return got


SHAPES = [
    # prefix of each group, own keys of its sequences, heads, kv heads, head_dim
    ([513], [[9, 9, 9, 9]], 16, 8, 128),
    ([1], [[1]], 16, 8, 128),
    ([31], [[32, 33]], 16, 8, 128),
    ([63, 64, 65], [[0, 1], [2], [64, 31, 65]], 16, 8, 128),
    ([127, 0, 129], [[5, 0], [3, 0, 40], [17]], 8, 8, 64),
    ([1000], [[1 + 7 * i for i in range(65)]], 16, 8, 128),     # 130 rows of a kv head
    ([300, 77], [[3] * 40, [50] * 33], 32, 8, 64),
    ([2000], [[1, 2, 3]], 8, 1, 128),                           # eight heads a kv head
    ([700], [[20] * 17], 35, 5, 128),                           # seven
    ([255], [[0] * 5], 3, 3, 64),                               # no own keys at all
    ([4100], [[100, 200]], 6, 2, 64),
    ([64] * 9, [[1 + i] for i in range(9)], 4, 4, 128),         # groups of one
    ([33, 40, 50], [[], [8, 9], []], 16, 8, 128),               # empty groups
    ([96], [[130] * 300], 2, 1, 64),                            # more sequences than CUs
]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_attention(i, rng):
    prefix, own, H, G, d = SHAPES[i]
    print("shape", SHAPES[i], flush=True)
    batch = Batch(rng, prefix, own, H, G, d, q_scale=2.0)
    a = batch.check()
    assert np.array_equal(a, batch.run())          # the same bits again
    assert np.array_equal(a, batch.run(in_place=True))


@pytest.mark.parametrize("n,H,G,d", [(257, 2, 1, 64), (700, 2, 2, 128)])
def test_more_groups_than_the_plan_has_threads(n, H, G, d, rng):
    """Empty groups and groups without a prefix among them, long ones at the ends of the plan's
    rounds; sequences in several rounds too."""
    prefix = [int(x) for x in rng.integers(0, 70, n)]
    own = [[int(x) for x in rng.integers(0, 40, rng.integers(0, 4))] for _ in range(n)]
    for g in (0, 255, 256, n - 1):
        prefix[g], own[g] = 600, [5] * 130
    batch = Batch(rng, prefix, own, H, G, d, gap=1, before=[0, 3], after=[9])
    a = batch.check()
    assert np.array_equal(a, batch.run())


def test_sequences_outside_every_group(rng):
    Batch(rng, [90, 70], [[4], [5, 6]], before=[30, 0], after=[1, 77]).check()


def test_no_keys_at_all_is_zeros(rng):
    batch = Batch(rng, [0, 10], [[0, 2], [0]], after=[0])
    got = batch.check()
    assert not got[0].any() and not got[3].any() and got[1].any()


@pytest.mark.parametrize("bounds", [(1, 1), (40000, 9000)])
def test_loose_bounds(bounds, rng):
    """Bounds far above the lengths change nothing but the launch."""
    batch = Batch(rng, [130], [[40, 3]], max_prefix=130 * bounds[0], max_n_keys=40 + bounds[1])
    batch.check()


@pytest.mark.parametrize("P,S,own,H,G,d", [(20000, 3, 77, 16, 8, 128), (9001, 70, 5, 32, 8, 64),
                                           (131072, 2, 1, 2, 1, 128), (5, 3, 20000, 4, 2, 128)])
def test_every_key_counts_once(P, S, own, H, G, d, rng):
    """q = 0: every weight is the same, so o is the mean of the values. Values are whole
    numbers, and one key more or less would move a mean by 4 / n or more where the key's
    value is 4 off it; the mean's own roundings are 2^-22 and the sums' of it."""
    batch = Batch(rng, [P], [[own] * S], H, G, d, q_scale=0.0)
    seen = ~np.isnan(batch.v)
    batch.v[seen] = rng.integers(4, 12, seen.sum()) * rng.choice([-1, 1], seen.sum())
    got = batch.run()
    for b in range(S):
        v = batch.v[batch.rows(b)].astype(np.float64)
        want = np.repeat(v.mean(0), H // G, axis=0)
        size = np.abs(v).mean()
        assert np.abs(got[b] - want).max() <= min(2.0 ** -18 * size, 2.0 / len(v))


@pytest.mark.parametrize("case", ["q", "k", "v", "tiny", "huge"])
def test_scales(case, rng):
    scale = {"q": dict(q_scale=1e4, k_scale=1e-4), "k": dict(q_scale=1e-6, k_scale=1e6),
             "v": dict(v_scale=1e-9), "tiny": dict(q_scale=1e-12, k_scale=1e-12, v_scale=1e-30),
             "huge": dict(q_scale=1e-18, k_scale=1e18, v_scale=1e30)}[case]
    Batch(rng, [200], [[40, 0, 3]], **scale).check()
    Batch(rng, [100, 30], [[70], [1]], 8, 4, 64, **scale).check()


def test_values_of_growing_size(rng):
    """Later keys' values far above earlier ones', and the other way round. Keys and values
    are off by 2^-22 of themselves or 2^-33 of the largest near them, so that a row's error is
    within the usual bound of its largest value."""
    for order in (1, -1):
        batch = Batch(rng, [1500], [[90, 0]], q_scale=1.5)
        scale = (2.0 ** np.linspace(-30, 30, 1500)).astype(np.float32)[::order]
        batch.v[batch.prefix_row[0]:][:1500] *= scale[:, None, None]
        batch.check()
        batch = Batch(rng, [1500], [[90, 0]], 4, 4, 64, q_scale=1.5)
        scale = (2.0 ** np.linspace(-20, 4, 1500)).astype(np.float32)[::order]
        batch.k[batch.prefix_row[0]:][:1500] *= scale[:, None, None]
        batch.check()


@pytest.mark.parametrize("H,G,d", [(64, 64, 64), (128, 64, 128)])
def test_sizes_that_jump_from_chain_to_chain(H, G, d, rng):
    """Few runs of many chains (a kv head has eight), whose keys and values have sizes of their
    own: 0, and 2^-90 to 2^90 apart from one to the next, and from tile to tile in one."""
    k_scale = [0, 40, -20, 90, -90, 0, 3, -60]
    v_scale = [0, -40, 60, -100, 90, 0, -3, 30]
    batch = Batch(rng, [70, 33, 300, 64, 5, 129, 1, 200],
                  [[3, 70], [1], [40, 0, 5], [33], [], [64, 2], [90], [7, 7, 7]], H, G, d)
    for g in range(8):
        seqs = range(batch.off[g], batch.off[g + 1])
        spans = [(batch.prefix_row[g], batch.prefix[g])]
        spans += [(batch.own_row[b], batch.n_keys[b]) for b in seqs]
        for at, n in spans:
            batch.k[at:at + n] *= np.float32(2.0 ** k_scale[g])
            batch.v[at:at + n] *= np.float32(2.0 ** v_scale[g])
        for b in seqs:
            batch.q[b] *= np.float32(2.0 ** -k_scale[g])
    at = batch.prefix_row[2]
    batch.k[at + 64:at + 128] = 0
    batch.v[at + 64:at + 128] = 0
    batch.v[at + 192:at + 256] *= np.float32(2.0 ** -100)
    batch.k[at + 128:at + 160] *= np.float32(2.0 ** -30)
    batch.check()
    # An infinite value reaches its sequence, none behind it.
    batch.v[batch.own_row[1] + 5, :, 0] = math.inf
    got = batch.run()
    assert not np.isfinite(got[1]).all(-1).any()
    rest = np.arange(batch.S) != 1
    o, tol = batch.want(np.flatnonzero(rest))
    assert (np.abs(got - o) <= tol)[rest].all()


def test_one_key_takes_all(rng):
    """Scores up to hundreds apart: running maxima that move late."""
    batch = Batch(rng, [3000], [[40, 900]], q_scale=4.0, k_scale=4.0)
    batch.k[batch.prefix_row[0] + 2990] = batch.k[batch.prefix_row[0] + 5] * 3
    batch.check()


def test_scores_below_the_range_of_f32_have_no_weight(rng):
    """Own keys (a part of their own) and some of the prefix so far below that their scores
    overflow: the rest is what counts. Beside keys 2^136 times as large, which keys 0 .. 31 of
    the prefix are (one tile), operands are off by 2^-33 of those, here by all of
    themselves: scores of 0 instead of their own, for all but keys 32 .. 39."""
    batch = Batch(rng, [40], [[3, 70]], q_scale=0.0)
    batch.q[:] = 1e20
    batch.k[batch.prefix_row[0]:][:40] *= np.float32(1e-21)
    for at, n in [(batch.own_row[0], 3), (batch.own_row[1], 70), (batch.prefix_row[0] + 7, 5)]:
        batch.k[at:at + n] = -1e20
    got = batch.run()
    rows = [batch.prefix_row[0] + i for i in range(40) if not 7 <= i < 12]
    batch.rows = lambda b: rows
    batch.k[batch.prefix_row[0]:][:32] = 0
    o, tol = batch.want()
    assert (np.abs(got - o) <= tol).all()


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
def test_what_is_not_finite_reaches_who_sees_it(bad, rng):
    batch = Batch(rng, [100, 60], [[5, 40], [33, 70]])
    batch.v[batch.prefix_row[1] + 7, 3, 11] = bad       # group 1's prefix, kv head 3
    batch.k[batch.own_row[0] + 2, 5, 0] = NAN           # sequence 0's own, kv head 5
    batch.v[batch.own_row[1] + 39, 0, :] = bad
    got = batch.run()
    fine = np.isfinite(got)
    hit = np.zeros_like(fine)
    hit[2:, 6:8, 11] = True
    hit[0, 10:12] = True
    hit[1, 0:2] = True
    # (Of a row that the bad value reaches, other dims may be NaN too.)
    rows = hit.any(-1)
    assert fine[~rows].all()
    assert not fine[hit].any()


# ------------------------------------------------------------------ refusals --
def test_counts_beyond_their_bounds_are_nan(rng):
    batch = Batch(rng, [50, 80], [[3, 9], [4, 2]], max_prefix=60, max_n_keys=8)
    got = batch.run()
    o, tol = batch.want(seqs=[0])
    assert np.abs(got[0] - o[0]).max() <= tol[0].max()
    assert np.isnan(got[1:]).all()


@pytest.mark.parametrize("off", [[0, 3, 2], [0, 2, 5], [3, 1, 4], [0, 0xffffffff, 4]])
def test_offsets_that_fall_or_pass_the_end_are_nan(off, rng):
    batch = Batch(rng, [50, 80], [[3, 9], [4, 2]])
    batch.off = off
    assert np.isnan(batch.run()).all()


# ---------------------------------------------------------------------- step --
class Step:
    """One layer's step of a batch, with its caches on the device."""

    def __init__(self, rng, batch, pairing="neox", stacked=False):
        self.b, self.pairing = batch, pairing
        H, G, d, S = batch.H, batch.G, batch.d, batch.S
        qkv = rng.standard_normal((S, (H + 2 * G) * d), np.float32)
        self.parts = np.split(qkv, [H * d, (H + G) * d], axis=1)
        self.gq = rng.normal(1.5, 0.1, d).astype(np.float32)
        self.gk = rng.normal(1, 0.1, d).astype(np.float32)
        self.inv = ops.rope_inv_freq(d, 1e6)
        if stacked:
            self.raw = dev(qkv)
            at = self.raw.ptr
            self.ptrs = (at, at + 4 * H * d, at + 4 * (H + G) * d)
            self.stride = (H + 2 * G) * d
        else:
            self.raw = [dev(p) for p in self.parts]
            self.ptrs, self.stride = [r.ptr for r in self.raw], 0
        self.kc, self.vc = dev(batch.k), dev(batch.v)
        self.dev = [dev(self.gq), dev(self.gk), dev(self.inv)]
        self.qn, self.o = dev(np.full(S * H * d, 7)), dev(np.full(S * H * d, 7))
        self.arrays, self.ws = batch.arrays(), batch.ws()

    def launch(self):
        ops.decode_layer_shared(*self.ptrs, *self.dev, EPS, self.pairing, self.qn, self.kc,
                                self.vc, *self.arrays, self.o, *self.b.shape(), self.ws,
                                in_stride=self.stride)

    def expect(self, live):
        """The rows that the step writes, into the batch's caches; qn."""
        b = self.b
        qn = np.zeros((b.S, b.H, b.d), np.float32)
        for s in live:
            g = b.group(s)
            pos = (0 if g is None else b.prefix[g]) + b.n_keys[s] - 1
            q, k = (oracle.rope(oracle.rmsnorm(x[s], gain, b.d, n, EPS), 1, n, b.d, pos, self.inv,
                                self.pairing)
                    for x, gain, n in ((self.parts[0], self.gq, b.H), (self.parts[1], self.gk, b.G)))
            qn[s] = np.asarray(q).reshape(b.H, b.d)
            row = b.own_row[s] + b.n_keys[s] - 1
            b.k[row] = np.asarray(k).reshape(b.G, b.d)
            b.v[row] = self.parts[2][s].reshape(b.G, b.d)
        return qn

    def check(self, live, refused=()):
        b = self.b
        qn = self.expect(live)
        shape = qn.shape
        got_qn = self.qn.download(qn.size).reshape(shape)
        got = self.o.download(qn.size).reshape(shape)
        for x in (got_qn, got):
            assert np.isnan(x[list(refused)]).all()
        rest = [s for s in range(b.S) if s not in refused]
        assert np.array_equal(got_qn[rest], qn[rest])
        for cache, want in ((self.kc, b.k), (self.vc, b.v)):
            assert np.array_equal(cache.download(want.size).view(np.uint32),
                                  want.ravel().view(np.uint32))
        o, tol = b.want(live, qn)
        assert (np.abs(got[rest] - o[rest]) <= tol[rest]).all()
        return got


@pytest.mark.parametrize("H,G,d,pairing,stacked", [(16, 8, 128, "neox", False),
                                                   (16, 8, 128, "norm", True),
                                                   (12, 3, 64, "neox", True),
                                                   (8, 1, 64, "norm", False)])
def test_step(H, G, d, pairing, stacked, rng):
    batch = Batch(rng, [70, 0, 300], [[1, 2], [5, 1], [33, 40, 1]], H, G, d, after=[9])
    step = Step(rng, batch, pairing, stacked)
    step.launch()
    ops.sync()
    step.check(range(batch.S))


def test_step_with_idle_and_refused_sequences(rng):
    batch = Batch(rng, [70, 200], [[0, 5, 13], [2, 0]], max_prefix=100, max_n_keys=9)
    step = Step(rng, batch)
    step.launch()
    ops.sync()
    # Group 1's prefix is beyond its bound: its sequences are refused, the idle one too.
    got = step.check([1], refused=[2, 3, 4])
    assert not got[0].any()


def test_step_whose_offsets_fall_appends_nothing(rng):
    batch = Batch(rng, [70, 20], [[3], [2, 5]])
    batch.off = [0, 2, 1]
    step = Step(rng, batch)
    step.launch()
    ops.sync()
    step.check([], refused=[0, 1, 2])


def test_step_equals_the_ragged_step_on_copies(rng):
    """Prefixes copied before each sequence's own keys, through flk_decode_layer_ragged: qn and
    the new rows are the same bits, o within twice the usual bound."""
    batch = Batch(rng, [150, 40], [[3, 20], [1, 64, 2]])
    step = Step(rng, batch)
    step.launch()
    ops.sync()
    rows, off, n = [], [], []
    for b in range(batch.S):
        off.append(len(rows))
        rows += batch.rows(b)
        n.append(len(rows) - off[-1])
    k, v = dev(batch.k[rows]), dev(batch.v[rows])
    S, H, G, d = batch.S, batch.H, batch.G, batch.d
    qn, o = B(4 * S * H * d), B(4 * S * H * d)
    ws = ops.Workspace(H, G, d, max(n), 0, S)
    ops.decode_layer_ragged(*step.ptrs, *step.dev, EPS, "neox", qn, k, v, dev(off, np.uint64),
                            dev(n, np.uint32), o, S, max(n), H, G, d, ws)
    ops.sync()
    got = step.check(range(S))
    assert np.array_equal(qn.download(S * H * d), step.qn.download(S * H * d))
    new = [off[b] + n[b] - 1 for b in range(S)]
    assert np.array_equal(k.download(len(rows) * G * d).reshape(-1, G, d)[new],
                          batch.k[[batch.rows(b)[-1] for b in range(S)]])
    _, tol = batch.want(q=step.qn.download(S * H * d).reshape(S, H, d))
    assert (np.abs(o.download(S * H * d).reshape(S, H, d) - got) <= 2 * tol).all()


# --------------------------------------------------------- streams and graphs --
def test_captured_step_replayed_as_lengths_and_groups_change(rng):
    """Two steps captured on one workspace, replayed in turn with eager work between;
    each replay equals the eager call."""
    batch = Batch(rng, [90, 40, 0], [[30, 30], [30, 30, 30], [30]], max_prefix=128, max_n_keys=64)
    a, b = Step(rng, batch), Step(rng, batch)
    b.ws = a.ws
    stream = ops.Stream()
    ops.set_stream(stream)
    graphs = []
    for s in (a, b):
        with ops.Graph() as g:
            s.launch()
        graphs.append(g)
    for n_keys, prefix, off in (([30] * 6, [90, 40, 0], [0, 2, 5, 6]),
                                ([1, 64, 0, 31, 32, 33], [128, 1, 77], [0, 1, 1, 6]),
                                ([65, 2, 3, 4, 5, 6], [90, 129, 3], [1, 2, 3, 6]),
                                ([9, 8, 7, 6, 5, 4], [90, 40, 0], [0, 2, 5, 6])):
        print(n_keys, prefix, off, flush=True)
        for s, g in zip((a, b), graphs):
            s.arrays[4].upload(np.array(n_keys, np.uint32))
            s.arrays[1].upload(np.array(prefix, np.uint32))
            s.arrays[2].upload(np.array(off, np.uint32))
            g.launch()
            ops.sync()
            n = batch.S * batch.H * batch.d
            got = [x.download(n) for x in (s.o, s.qn)]
            s.launch()  # eager, over the same rows
            ops.sync()
            for x, y in zip(got, (s.o, s.qn)):
                assert np.array_equal(x, y.download(n), equal_nan=True)
    ops.set_stream(None)
    for g in graphs:
        g.free()
    stream.free()


def test_replays_follow_a_growing_answer(rng):
    """A captured step whose counts grow by one a replay, against 64 bits."""
    batch = Batch(rng, [66], [[1, 31, 62]], gap=8, junk=0.0, max_n_keys=70)
    step = Step(rng, batch)
    stream = ops.Stream()
    ops.set_stream(stream)
    with ops.Graph() as g:
        step.launch()
    for _ in range(4):
        g.launch()
        ops.sync()
        step.check(range(3))
        batch.n_keys = [n + 1 for n in batch.n_keys]
        step.arrays[4].upload(np.array(batch.n_keys, np.uint32))
    ops.set_stream(None)
    g.free()
    stream.free()


def test_rows_behind_four_gigabytes(rng):
    """A prefix and own keys whose bytes, and floats, lie past 32 bits."""
    batch = Batch(rng, [70], [[3, 40]], 4, 4, 128)
    row_bytes = 4 * batch.G * batch.d
    shift = (17 << 30) // row_bytes  # 2^32 floats and a bit more
    n = len(batch.k)
    k, v = B((shift + n) * row_bytes), B((shift + n) * row_bytes)
    k.upload(batch.k, shift * row_bytes)
    v.upload(batch.v, shift * row_bytes)
    arrays = list(batch.arrays())
    arrays[0] = dev(np.array(batch.prefix_row) + shift, np.uint64)
    arrays[3] = dev(np.array(batch.own_row) + shift, np.uint64)
    o = B(4 * batch.q.size)
    ops.attn_decode_shared(dev(batch.q), k, v, *arrays, o, *batch.shape(), batch.ws())
    ops.sync()
    got = o.download(batch.q.size).reshape(batch.q.shape)
    want, tol = batch.want()
    assert (np.abs(got - want) <= tol).all()
    k.free()
    v.free()
