"""What the entry points for several answers refuse on the host, before any launch (no GPU
needed: the pointers are never read)."""
from __future__ import annotations

import pytest

from flock_amd import _lib, ops
from flock_amd._lib import FlockError

ARG, UNSUPPORTED, WORKSPACE = (_lib.FLK_ERR_ARG, _lib.FLK_ERR_UNSUPPORTED, _lib.FLK_ERR_WORKSPACE)
P = 0x10000          # never read
BIG = (P, 1 << 50)   # a workspace that is never too small


def attn(q=P, kc=P, vc=P, prow=P, npre=P, off=P, srow=P, nk=P, o=P, groups=1, seqs=4, pre=100,
         keys=10, H=16, G=8, d=128, ws=BIG):
    ops.attn_decode_shared(q, kc, vc, prow, npre, off, srow, nk, o, groups, seqs, pre, keys, H, G,
                           d, ws)


def step(q=P, k=P, v=P, gq=P, gk=P, inv=P, pairing="neox", qn=P, kc=P, vc=P, prow=P, npre=P,
         off=P, srow=P, nk=P, o=2 * P, groups=1, seqs=4, pre=100, keys=10, H=16, G=8, d=128,
         ws=BIG, stride=0):
    ops.decode_layer_shared(q, k, v, gq, gk, inv, 1e-6, pairing, qn, kc, vc, prow, npre, off, srow,
                            nk, o, groups, seqs, pre, keys, H, G, d, ws, in_stride=stride)


def refused(code, call, **kw):
    with pytest.raises(FlockError) as e:
        call(**kw)
    assert e.value.code == code, e.value
    assert str(e.value)


@pytest.mark.parametrize("call", [attn, step])
def test_shared(call):
    for name in ("q", "kc", "vc", "prow", "npre", "off", "srow", "nk", "o"):
        refused(ARG, call, **{name: None})
    for name in ("kc", "vc", "prow", "npre", "off", "srow", "nk"):
        refused(ARG, call, **{name: P + 2})
    refused(ARG, call, o=2 * P + 8)
    refused(ARG, call, prow=P + 4)
    refused(ARG, call, srow=P + 4)
    refused(ARG, call, groups=0)
    refused(ARG, call, seqs=0)
    refused(ARG, call, pre=0, keys=0)
    refused(ARG, call, pre=0xffffffff, keys=1)
    refused(UNSUPPORTED, call, seqs=65536)
    refused(UNSUPPORTED, call, groups=65536)
    refused(UNSUPPORTED, call, d=96)
    refused(ARG, call, H=15)
    refused(UNSUPPORTED, call, H=72)
    refused(UNSUPPORTED, call, H=1 << 17, G=1 << 16, seqs=1)


def test_shared_overlaps_and_workspace():
    refused(ARG, attn, q=P + 8)
    refused(ARG, attn, q=2 * P, o=2 * P + 4 * 128)
    refused(ARG, step, qn=2 * P)
    refused(ARG, step, qn=2 * P + 16 * 128, o=2 * P)
    refused(ARG, step, stride=16 * 128 - 1)
    refused(ARG, step, pairing=2)
    for name in ("k", "v", "gq", "gk", "inv", "qn"):
        refused(ARG, step, **{name: None})
    need = ops.decode_shared_ws_bytes(1, 4, 100, 10, 16, 8, 128)
    if need:
        refused(WORKSPACE, attn, ws=None)
        refused(WORKSPACE, attn, ws=(P, need - 1))
        refused(WORKSPACE, step, ws=(P + 16, need))
    assert ops.decode_shared_ws_bytes(1, 4, 100, 10, 16, 8, 96) == 0
    assert ops.decode_shared_ws_bytes(0, 4, 100, 10, 16, 8, 128) == 0


def test_workspaces_grow_with_their_bounds():
    """A workspace for larger bounds holds every smaller call's."""
    def need(groups, seqs, pre, keys, H=16, G=8, d=128):
        return ops.decode_shared_ws_bytes(groups, seqs, pre, keys, H, G, d)

    for groups, seqs, pre, keys in ((1, 1, 0, 1), (1, 4, 513, 9), (3, 64, 9000, 700),
                                    (12, 3000, 131072, 2000), (65535, 65535, 1 << 30, 1 << 30)):
        n = need(groups, seqs, pre, keys)
        assert n <= need(min(groups + 1, 65535), seqs, pre, keys)
        assert n <= need(groups, min(seqs + 1, 65535), pre, keys)
        assert n <= need(groups, seqs, pre + 1, keys)
        assert n <= need(groups, seqs, pre, keys + 1)


def score(logits=P, ld=0, tokens=P, lp=P, ent=P, ids=P, tops=P, rows=2, vocab=1000, k=5, ws=BIG):
    ops.token_logprobs(logits, tokens, lp, rows, vocab, ws, entropy=ent, n_top=k, top_ids=ids,
                       top_logprobs=tops, ld=ld)


def draw(logits=P, ld=0, t=P, k=P, top_p=P, min_p=P, u=P, token=P, lp=P, rows=2, vocab=1000,
         max_k=20, ws=BIG):
    ops.sample(logits, u, token, rows, vocab, max_k, ws, temperature=t, top_k=k, top_p=top_p,
               min_p=min_p, logprob=lp, ld=ld)


def test_scores():
    refused(ARG, score, logits=None)
    for name in ("logits", "tokens", "lp", "ent", "ids", "tops"):
        refused(ARG, score, **{name: P + 2})
    refused(ARG, score, tokens=None)
    refused(ARG, score, ids=None)
    refused(ARG, score, tops=None)
    refused(ARG, score, k=0)
    refused(ARG, score, k=0, ids=None, tops=None, lp=None, ent=None)
    refused(ARG, score, rows=0)
    refused(ARG, score, vocab=0)
    refused(ARG, score, ld=999)
    refused(UNSUPPORTED, score, k=65)
    refused(UNSUPPORTED, score, vocab=1 << 31)
    refused(UNSUPPORTED, score, rows=1 << 24)


def test_samples():
    for name in ("logits", "u", "token"):
        refused(ARG, draw, **{name: None})
    for name in ("logits", "u", "token", "t", "k", "top_p", "min_p", "lp"):
        refused(ARG, draw, **{name: P + 1})
    refused(ARG, draw, max_k=0)
    refused(UNSUPPORTED, draw, max_k=65)
    refused(ARG, draw, rows=0)
    refused(ARG, draw, vocab=0)
    refused(ARG, draw, ld=10)
    need = ops.tokens_ws_bytes(1, 151936, 20)
    if need:
        refused(WORKSPACE, draw, rows=1, vocab=151936, ws=None)
        refused(WORKSPACE, draw, rows=1, vocab=151936, ws=(P, need - 1))
        refused(WORKSPACE, draw, rows=1, vocab=151936, ws=(P + 4, need))
    for rows in (1, 2, 63, 700, 1024, 1025, 5000):
        assert need <= ops.tokens_ws_bytes(rows, 151936, 20) <= ops.tokens_ws_bytes(
            rows + 1, 151936, 20)
    assert ops.tokens_ws_bytes(0, 100, 5) == 0 and ops.tokens_ws_bytes(1, 100, 65) == 0


def advance(nk=P, cursor=P, token=P, log=P, n=3, T=4, lp=P, lp_log=P, stops=P, n_stops=2, u_log=P,
            u=P):
    ops.advance_seqs(nk, cursor, token, log, n, T, logprob=lp, logprob_log=lp_log, stops=stops,
                     n_stops=n_stops, uniform_log=u_log, uniform=u)


def test_advance_seqs():
    for name in ("nk", "cursor", "token", "log", "lp", "lp_log", "stops", "u_log", "u"):
        refused(ARG, advance, **{name: None})
        refused(ARG, advance, **{name: P + 1})
    refused(ARG, advance, n_stops=0)
    refused(ARG, advance, n=0)
