"""Model.answers at the edges of its arguments: a model without prefill, calls that fail."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from flock_amd import ops  # noqa: E402
from flock_amd.model import Model  # noqa: E402
from test_gpu_model import VOCAB, build  # noqa: E402


def test_a_model_that_takes_one_id_at_a_time(rng):
    """maxPrefill 0: one answer at a time, the ids that one of maxPrefill 1 gives."""
    got = []
    for P in (0, 1):
        cfg, layers, embd, gout = build(np.random.default_rng(3), maxPrefill=P)
        m = Model(cfg, layers, embd, gout, VOCAB)
        got.append(m.answers([3, 14, 15], 1, 5, seed=4))
        assert m.nKeys == 2
        with pytest.raises(ValueError):
            m.answers([3, 14, 15], 2, 5)
        m.free()
    assert got[0] == got[1] and len(got[0][0][0]) == 5


def test_a_call_that_fails_feeds_nothing(rng, monkeypatch):
    cfg, layers, embd, gout = build(rng)
    m = Model(cfg, layers, embd, gout, VOCAB)
    first = m.answers([3, 14, 15], 2, 3, seed=4)
    m.reset()
    with pytest.raises((ValueError, TypeError)):
        m.answers([9, 14, 15, 16], 2, 3, seed=-1)

    def failing(*_, **__):
        raise MemoryError
    with monkeypatch.context() as patch:
        patch.setattr(ops, "sample", failing)
        with pytest.raises(MemoryError):
            m.answers([9, 14, 15, 16], 2, 4, seed=4)
    assert m.nKeys == 0 and all(layer.nKeys == 0 for layer in m.layers)
    assert m.answers([3, 14, 15], 2, 3, seed=4) == first
    m.free()


def test_stops_outside_the_vocabulary_end_nothing(rng):
    cfg, layers, embd, gout = build(rng)
    m = Model(cfg, layers, embd, gout, VOCAB)
    first = m.answers([3, 14, 15], 3, 4, seed=4)
    m.reset()
    assert m.answers([3, 14, 15], 3, 4, seed=4, eos=[-1, VOCAB, 1 << 32]) == first
    m.free()


def test_an_answer_without_a_draw_is_an_error(rng):
    """Logits that hold nothing but NaN: not the same as answers that stop at once."""
    cfg, layers, embd, gout = build(rng)
    m = Model(cfg, layers, embd, gout, VOCAB)
    first = m.answers([3, 14, 15], 2, 3, seed=4)
    m.reset()
    m.g_out.upload(np.full(cfg.hidden, np.nan, np.float32))
    for eos in ([], [7]):
        with pytest.raises(RuntimeError, match="no id"):
            m.answers([3, 14, 15], 2, 3, seed=4, eos=eos)
        m.reset()
    m.g_out.upload(gout)
    assert m.answers([3, 14, 15], 2, 3, seed=4) == first
    m.free()
