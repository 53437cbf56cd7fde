"""The paged 4-bit cache without a GPU: the reference's own consistency, and the
refusals, which run on the host before any launch."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref as ref
from flock_amd import _lib, ops

FAKE, FAKE2 = 0x10000, 0x40000000


@pytest.mark.parametrize("D", [64, 128])
def test_places_of_a_tile_are_all_distinct_and_fill_it(D):
    kb, ksh, ks, vb, vsh, vs = ref.places(D)
    nibbles = np.concatenate([(2 * b + s // 4).ravel() for b, s in ((kb, ksh), (vb, vsh))])
    scales = np.concatenate([np.unique(x) for x in (ks, vs)])
    used = np.concatenate([nibbles, 2 * scales, 2 * scales + 1, 2 * scales + 2, 2 * scales + 3])
    assert len(np.unique(used)) == len(used) == 2 * 36 * D


@pytest.mark.parametrize("D", [64, 128])
def test_v_words_of_tokens_share_no_byte(D):
    vb = ref.places(D)[3]
    owner = {}
    for t in range(32):
        for b in set(vb[t].tolist()):
            assert owner.setdefault(b, t) == t


def test_quantised_values_are_within_half_a_step():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((500, 128)).astype(np.float32)
    c, d = ref.quantise(x)
    step = np.abs(np.repeat(d.astype(np.float32), 32, -1))
    err = np.abs(ref.values(c, d) - x)
    # Half a step, or what lies past the last code (7 where the largest of the other
    # sign is up to 8 steps, with the scale's own 2^-9 rounded down).
    assert (err <= step * np.where(c == 15, 1 + 2 ** -5, 0.5 + 2 ** -5)).all()


def test_products_of_codes_and_scales_are_exact_in_f16():
    d = np.arange(65536, dtype=np.uint32)
    d = ref.bf16((d << 16).view(np.float32)[np.isfinite((d << 16).view(np.float32))])
    d = np.clip(d, -8160, 8160).astype(np.float16).astype(np.float32)
    for c in range(-8, 8):
        x = d * np.float32(c)
        assert (x.astype(np.float16).astype(np.float32) == x).all()


def test_page_bytes():
    assert ops.kv4_page_bytes(8, 128, 64) == 64 * 8 * 128 * 2 * 9 // 16
    L = _lib.lib()
    for bad in ((0, 128, 64), (8, 96, 64), (8, 128, 48)):
        assert L.flk_kv4_page_bytes(*bad) == 0


def refuse(rc, code, text):
    assert rc == code and text in _lib.lib().flk_last_error().decode(), (
        rc, _lib.lib().flk_last_error())


def plan_call(**kw):
    a = dict(n_keys=FAKE, n_new=FAKE, table_in=FAKE, table_out=FAKE, free_in=FAKE,
             free_out=FAKE2, q_off=FAKE, positions=FAKE, slots=FAKE, lost=FAKE, n_seqs=4,
             max_blocks=8, n_pages=100, max_tokens=16, page=64, window=0, sinks=0, ws=FAKE,
             ws_bytes=1 << 20)
    a.update(kw)
    return _lib.lib().flk_kv4_plan(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_keys=None), -1, "n_keys is null"), (dict(slots=FAKE + 2), -1, "slots must be 4-byte"),
    (dict(page=48), -3, "48"), (dict(n_pages=0), -1, "n_pages"), (dict(n_seqs=0), -1, "n_seqs=0"),
    (dict(n_pages=1 << 26), -3, "32-bit"), (dict(n_seqs=70000), -3, "70000"),
    (dict(free_out=FAKE + 400), -1, "free_out"), (dict(table_out=FAKE + 64), -1, "table_out"),
    (dict(ws=None), -4, "needed"), (dict(ws_bytes=8), -4, "needed"),
    (dict(ws=FAKE + 16), -4, "aligned"), (dict(max_blocks=0), -1, "max_blocks=0"),
    (dict(max_tokens=0), -1, "max_tokens=0")])
def test_plan_refusals(kw, code, text):
    refuse(plan_call(**kw), code, text)


def prologue_call(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, in_stride=0, gq=FAKE, gk=FAKE, inv=FAKE, eps=1e-6, pairing=0,
             positions=FAKE, slots=FAKE, qn=FAKE, pool=FAKE, n=4, H=16, G=8, D=128, n_pages=10,
             page=64)
    a.update(kw)
    return _lib.lib().flk_kv4_prologue(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(k=None), -1, "k_raw is null"), (dict(positions=FAKE + 1), -1, "positions must be"),
    (dict(pool=FAKE + 8), -1, "pool must be 16-byte"), (dict(D=96), -3, "96"),
    (dict(H=15), -1, "multiple"), (dict(H=128), -3, "group"), (dict(n=0), -1, "n_tokens"),
    (dict(pairing=2), -1, "pairing 2"), (dict(in_stride=100), -1, "in_stride 100"),
    (dict(page=16), -3, "16")])
def test_prologue_refusals(kw, code, text):
    refuse(prologue_call(**kw), code, text)


def test_append_and_read_refusals():
    L = _lib.lib()
    refuse(L.flk_kv4_append(FAKE, FAKE, FAKE + 2, FAKE, 1, 8, 128, 4, 64), -1, "slots must be")
    refuse(L.flk_kv4_append(FAKE, FAKE, FAKE, FAKE, 0, 8, 128, 4, 64), -1, "n_tokens")
    refuse(L.flk_kv4_append(FAKE, FAKE, FAKE, FAKE, 1, 0, 128, 4, 64), -1, "n_kv_heads (0)")
    refuse(L.flk_kv4_read(FAKE, FAKE, FAKE + 4, FAKE, 1, 8, 128, 4, 64), -1, "k must be 16-byte")
    refuse(L.flk_kv4_read(FAKE, FAKE, FAKE, FAKE, 1, 8, 32, 4, 64), -3, "head_dim 32")


def attn_call(**kw):
    a = dict(q=FAKE, pool=FAKE, table=FAKE, n_keys=FAKE, q_off=FAKE, o=FAKE2, n_seqs=2, n_tokens=4,
             max_q=2, max_n_keys=4096, max_blocks=64, H=16, G=8, D=128, n_pages=128, page=64,
             window=0, sinks=0, ws=FAKE, ws_bytes=1 << 30)
    a.update(kw)
    return _lib.lib().flk_kv4_attn(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(q=None), -1, "q is null"), (dict(o=FAKE2 + 8), -1, "o must be 16-byte"),
    (dict(table=FAKE + 2), -1, "table must be"), (dict(o=FAKE + 512), -1, "partly over q"),
    (dict(max_n_keys=4097), -1, "4097 keys do not fit"), (dict(n_seqs=0), -1, "n_seqs=0"),
    (dict(max_q=0), -1, "max_q=0"), (dict(H=72), -3, "group"), (dict(D=256), -3, "256"),
    (dict(n_seqs=65536), -3, "65536"), (dict(page=0), -3, "pages of 0")])
def test_attention_refusals(kw, code, text):
    refuse(attn_call(**kw), code, text)


def test_calls_larger_than_a_launch_are_refused():
    L = _lib.lib()
    refuse(plan_call(n_seqs=65535, max_blocks=32769, table_out=FAKE), -3, "65535 x 32769")
    refuse(plan_call(n_seqs=1, max_blocks=0xFFFFFFC1), -3, "exceeds 2^31")
    refuse(prologue_call(n=1 << 24), -3, "16777216 tokens")
    refuse(L.flk_kv4_append(FAKE, FAKE, FAKE, FAKE, 1 << 24, 8, 128, 4, 64), -3, "exceed")
    refuse(L.flk_kv4_read(FAKE, FAKE, FAKE, FAKE, 1 << 24, 8, 128, 4, 64), -3, "exceed")
    big = dict(q=FAKE, o=FAKE, max_n_keys=1 << 20, max_blocks=1 << 20)
    for kw in (dict(n_seqs=65535, max_q=1 << 20, H=64),             # whole row tiles
               dict(n_seqs=32, max_q=128, H=8192, G=1024),         # the merge of prompts
               dict(n_seqs=65535, max_q=1, H=512, G=256)):          # the merge of single tokens
        refuse(attn_call(**big, **kw), -3, "exceed a launch")


def test_attention_workspace_queries():
    L = _lib.lib()
    for bad in ((0, 1, 1, 16, 8, 128, 0, 0), (1, 0, 1, 16, 8, 128, 0, 0),
                (1, 1, 0, 16, 8, 128, 0, 0), (1, 1, 1, 16, 0, 128, 0, 0),
                (1, 1, 1, 16, 5, 128, 0, 0), (1, 1, 1, 16, 8, 96, 0, 0)):
        assert L.flk_kv4_attn_ws_bytes(*bad) == 0


def test_reference_plan_returns_what_it_took():
    free = list(range(40))
    table = np.full((3, 8), ref.NONE, np.uint32)
    t1, f1, q1, pos, slots, lost = ref.plan([100, 64, 0], [100, 64, 0], table, free, 200, 40, 32, 0,
                                            0)
    assert lost == 0 and q1 == [0, 100, 164, 164] and len(f1) == 40 - 6
    assert sorted(slots[:164]) == sorted(set(slots[:164])) and slots[164:] == [ref.NONE] * 36
    t2, f2, *_ = ref.plan([0, 0, 0], [0, 0, 0], t1, f1, 10, 40, 32, 0, 0)
    assert (t2 == ref.NONE).all() and sorted(f2) == free
