"""Several answers to one prompt, and the score of given ids (flock_amd/model.py): the steps
over shared prefixes, the draws and the log probabilities together, as a captured step
runs them, against the oracle's layers and 64-bit distributions."""
from __future__ import annotations

import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu

from flock_amd import CacheFullError, ops  # noqa: E402
from flock_amd.model import Model  # noqa: E402
from test_gpu_decoder import ocfg  # noqa: E402
from test_gpu_model import VOCAB, build  # noqa: E402

B = ops.DeviceBuffer


def oracle_logits(cfg, layers, embd, gout, ids):
    """Logits behind every position of ids."""
    row = cfg.nKvHeads * cfg.headDim
    x = oracle.embed(embd, ids, VOCAB, cfg.hidden)
    for w in layers:
        kc, vc = (np.zeros(cfg.maxKeys * row, np.float32) for _ in range(2))
        x = oracle.layer_prefill(x, len(ids), w, ocfg(cfg), kc, vc, 0)
    rows = x.reshape(len(ids), cfg.hidden)
    return np.stack([oracle.lm_head(r, gout, cfg.eps, embd, VOCAB, cfg.hidden)[1] for r in rows])


def log_softmax(x):
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def slack(logits):
    """How far a log probability may be off: attention's order of sums moves a logit by
    1e-4 of the largest at most (as for greedy decoding), a log probability by twice that."""
    return 2e-4 * max(1.0, np.abs(logits).max())


@pytest.mark.parametrize("prompt,n,T,settings", [
    ([3, 14, 15, 92, 65], 3, 4, dict()),
    ([7], 2, 3, dict(temperature=0.7, top_k=20)),                       # no prefix at all
    (list(range(5, 405, 20)), 9, 3, dict(top_p=0.8, min_p=0.01)),       # a prompt in two chunks
])
def test_answers_against_oracle(prompt, n, T, settings, rng):
    cfg, layers, embd, gout = build(rng, maxKeys=64)
    m = Model(cfg, layers, embd, gout, VOCAB)
    got = m.answers(prompt, n, T, seed=11, **settings)
    uniform = np.random.default_rng(11).random((T, n), np.float32).astype(np.float64)
    assert len(got) == n and m.nKeys == len(prompt) - 1
    for b, (ids, lp) in enumerate(got):
        assert len(ids) == len(lp) == T
        logits = oracle_logits(cfg, layers, embd, gout, prompt + ids)[len(prompt) - 1:-1]
        off = slack(logits)
        assert np.abs(lp - log_softmax(logits)[np.arange(T), ids]).max() <= off
        for t in range(T):
            x = logits[t].astype(np.float64)
            order = np.argsort(-x, kind="stable")[:settings.get("top_k", 64)]
            temperature = settings.get("temperature", 1.0)
            w = np.exp((x[order] - x[order[0]]) / temperature)
            if len(w) > 1:
                keep = np.cumsum(w) - w < settings.get("top_p", 1.0) * w.sum()
                keep &= w >= settings.get("min_p", 0.0)
                w *= keep
            # The draw's place in the running sums, each off by as much as a weight's
            # exponent twice; at a border the neighbour will do.
            c, u = np.cumsum(w) / w.sum(), uniform[t, b]
            i = int(np.flatnonzero(order == ids[t])[0])
            e = 4 * off / temperature
            assert c[i] >= u - e and c[i] - w[i] / w.sum() <= u + e, (b, t, c[i], u)
    m.free()


def test_greedy_answers_are_generates(rng):
    cfg, layers, embd, gout = build(rng)
    prompt = [3, 14, 15, 92, 65]
    a, b = (Model(cfg, layers, embd, gout, VOCAB, max_generate=32) for _ in range(2))
    got = a.answers(prompt, 4, 6, temperature=0.0)
    want = b.generate(prompt, 6)
    logits = oracle_logits(cfg, layers, embd, gout, prompt + want)[len(prompt) - 1:]
    top = np.sort(logits, -1)
    for ids, _ in got:
        for t in range(6):
            if ids[t] != want[t]:  # only where the two largest are as near as roundings reach
                assert top[t, -1] - top[t, -2] < 1e-4 * max(1.0, abs(top[t, -1]))
                break
    # The cache holds the prompt but for its last id: decoding goes on from there.
    assert a.generate([prompt[-1]], 6) == want
    a.free()
    b.free()


def test_the_captured_step_serves_other_prompts(rng):
    """The same bits as from a model of its own, and again with the same seed; an answer ends
    before its stop, the others go on."""
    cfg, layers, embd, gout = build(rng)
    a = Model(cfg, layers, embd, gout, VOCAB)
    a.answers([9, 8, 7, 6, 5, 4, 3], 5, 4, seed=1)
    graph = a._answers.graph
    a.reset()
    first = a.answers([3, 14, 15], 5, 4, seed=2)
    assert a._answers.graph is graph
    a.reset()
    assert a.answers([3, 14, 15], 5, 4, seed=2) == first
    b = Model(cfg, layers, embd, gout, VOCAB)
    assert b.answers([3, 14, 15], 5, 4, seed=2) == first
    b.reset()
    stop = first[2][0][1]
    ended = b.answers([3, 14, 15], 5, 4, seed=2, eos=[stop, 511])
    for (ids, lp), (was, was_lp) in zip(ended, first):
        n = next((t for t, i in enumerate(was) if i in (stop, 511)), 4)
        assert ids == was[:n] and np.allclose(lp, was_lp[:n], rtol=0, atol=1e-3)
    assert len(ended[2][0]) <= 1
    a.free()
    b.free()


def test_score_against_oracle(rng):
    cfg, layers, embd, gout = build(rng, maxKeys=64)
    m = Model(cfg, layers, embd, gout, VOCAB)
    ids = [int(i) for i in rng.integers(0, VOCAB, 33)]   # chunks of 16, 16 and 1
    logits = oracle_logits(cfg, layers, embd, gout, ids)
    want = log_softmax(logits)[np.arange(32), ids[1:]]
    assert np.abs(m.score(ids) - want).max() <= slack(logits)
    m.reset()
    first, second = m.score(ids[:10]), m.score(ids[10:])   # the first of a call has no score
    assert np.abs(first - want[:9]).max() <= slack(logits)
    assert np.abs(second - want[10:]).max() <= slack(logits)
    m.free()


def test_refusals(rng):
    cfg, layers, embd, gout = build(rng, n_layers=1, maxKeys=16, maxPrefill=4)
    m = Model(cfg, layers, embd, gout, VOCAB)
    for bad in (dict(n=0), dict(n=5), dict(top_k=0), dict(top_k=65), dict(temperature=-1.0),
                dict(temperature=float("inf")), dict(top_p=0.0), dict(min_p=1.5),
                dict(prompt=[])):
        args = dict(prompt=[1, 2], n=2, maxTokens=2)
        args.update(bad)
        with pytest.raises(ValueError):
            m.answers(**args)
    with pytest.raises(CacheFullError):
        m.answers([1, 2, 3], 4, 4)                      # 2 + 16 rows
    with pytest.raises(ValueError):
        m.score([1])
    with pytest.raises(ValueError):
        m.score([1, VOCAB])
    with pytest.raises(CacheFullError):
        m.score(list(range(17)))
    assert m.nKeys == 0 and m.answers([1, 2], 3, 0) == [([], [])] * 3
    m.free()


@pytest.mark.parametrize("n", [1, 3, 300])
def test_advance_seqs(n, rng):
    T = 3
    n_keys = rng.integers(0, 3, n).astype(np.uint32)
    stops = np.array([7, 9], np.uint32)
    dev = B.from_array(n_keys)
    cursor = B.from_array(np.zeros(1, np.uint32))
    uniforms = rng.random((T, n), np.float32)
    uniform, logs, lps = B(4 * n), B(4 * T * n), B(4 * T * n)
    logs.upload(np.zeros(T * n, np.uint32))
    lps.upload(np.zeros(T * n, np.float32))
    uniform.upload(uniforms[0])
    want_log, want_lp, want_u = np.zeros((T, n), np.uint32), np.zeros((T, n), np.float32), uniforms[0]
    for t in range(T + 2):                              # two steps more than the log holds
        token = rng.integers(0, 12, n).astype(np.uint32)
        token[rng.random(n) < 0.1] = 0xffffffff
        lp = rng.standard_normal(n).astype(np.float32)
        ops.advance_seqs(dev, cursor, B.from_array(token), logs, n, T, logprob=B.from_array(lp),
                         logprob_log=lps, stops=B.from_array(stops), n_stops=2,
                         uniform_log=B.from_array(uniforms), uniform=uniform)
        ops.sync()
        ends = (n_keys == 0) | np.isin(token, [7, 9, 0xffffffff])
        n_keys = np.where(ends, 0, n_keys + 1).astype(np.uint32)
        if t < T:
            want_log[t], want_lp[t] = token, lp
        if t + 1 < T:
            want_u = uniforms[t + 1]
        assert np.array_equal(dev.download(n, np.uint32), n_keys)
        assert np.array_equal(logs.download(T * n, np.uint32), want_log.ravel())
        assert np.array_equal(lps.download(T * n), want_lp.ravel())
        assert np.array_equal(uniform.download(n), want_u)
        assert cursor.download(1, np.uint32)[0] == t + 1
