"""The steps of serving from a paged cache held in 4 bits, as measurable cases.

Four operators: the plan (block tables and slot maps from request lengths),
the prologue that norms, rotates and appends new tokens in 4 bits, and
attention over the cache for single tokens and drafts and for prompts, each
with an optional sliding window and a few first tokens that stay visible.

The cache is a pool of pages. A page holds `page` tokens: for each kv head,
page / 32 tiles of 32 tokens and 36 * D bytes:

  K codes   16 D  D = 128: [half][key 16][part 4] of 16 bytes
                  D = 64:  [key 16][part 4][half] of 8 bytes
                  token 16 * half + key, dims part * D/4 ..; in each dword, dim
                  t of its 8 is nibble (t >> 1) + 4 * (t & 1)
  K scales   2 D  [key 16][block D/32][half] f16
  V codes   16 D  [chunk D/64][g 4][n 16][slot 8] 16-bit words: token 4 g + slot
                  (slot < 4) or 12 + 4 g + slot, nibble j is dim D/16 n + 4 chunk + j
  V scales   2 D  [g 4][block D/32][slot 8] f16

A code c and its block's scale d stand for (c - 8) * d. Scales have eight
significant bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

EPS = 9.999999974752427e-7  # the layer configuration's default
ROPE_BASE = 1e6
WIDE = {"heads": 16, "kv_heads": 8, "head_dim": 128}
NARROW = {"heads": 32, "kv_heads": 8, "head_dim": 64}


def listed():
    return [
        # A chat server's next token: 16 requests, one new token each. Latency.
        {"name": "plan-16", "kind": "plan", "seqs": 16, "past": 1500, "new_low": 1, "new_high": 1,
         "page": 64, "blocks": 64, "window": 0, "sinks": 0, "lengths": 1},
        # A full server: 2048 requests, drafts of up to 4 tokens, windows that
        # give pages back.
        {"name": "plan-2048", "kind": "plan", "seqs": 2048, "past": 30000, "new_low": 1,
         "new_high": 4, "page": 64, "blocks": 512, "window": 4096, "sinks": 4, "lengths": 2},
        # One layer's new rows in a decode step of 64 requests.
        {"name": "prologue-64", "kind": "prologue", **WIDE, "pairing": "neox", "tokens": 64,
         "past": 8000, "page": 64, "stacked": False, "run": 1},
        # ... and of prompts of 8192 tokens together, from a stacked projection.
        {"name": "prologue-8192", "kind": "prologue", **WIDE, "pairing": "neox", "tokens": 8192,
         "past": 1000, "page": 64, "stacked": True, "run": 2048},
        # A token early in a chat: bound by latency.
        {"name": "decode-1x513", "kind": "attn", **WIDE, "seqs": 1, "new_low": 1, "new_high": 1,
         "past_low": 512, "past_high": 512, "page": 64, "window": 0, "sinks": 0, "lengths": 1},
        # A serving step: 64 requests of 1025 to 16385 keys.
        {"name": "decode-64x16k", "kind": "attn", **WIDE, "seqs": 64, "new_low": 1, "new_high": 1,
         "past_low": 1024, "past_high": 16384, "page": 64, "window": 0, "sinks": 0, "lengths": 3},
        # A long document, one request.
        {"name": "decode-1x131072", "kind": "attn", **WIDE, "seqs": 1, "new_low": 1, "new_high": 1,
         "past_low": 131071, "past_high": 131071, "page": 128, "window": 0, "sinks": 0,
         "lengths": 4},
        # Endless chats: a window of 4096 keys and 4 sinks, 64-wide heads.
        {"name": "decode-128-window", "kind": "attn", **NARROW, "seqs": 128, "new_low": 1,
         "new_high": 1, "past_low": 1000, "past_high": 20000, "page": 32, "window": 4096,
         "sinks": 4, "lengths": 5},
        # Drafts of five tokens to be verified, 16 requests.
        {"name": "draft-16x5", "kind": "attn", **WIDE, "seqs": 16, "new_low": 5, "new_high": 5,
         "past_low": 500, "past_high": 4000, "page": 64, "window": 0, "sinks": 0, "lengths": 6},
        # Prompts of odd lengths together, window and sinks, 64-wide heads.
        {"name": "prefill-7-ragged", "kind": "attn", **NARROW, "seqs": 7, "new_low": 1,
         "new_high": 1500, "past_low": 0, "past_high": 1000, "page": 128, "window": 1024,
         "sinks": 4, "lengths": 7},
        # A chunk of 64 tokens onto a long context.
        {"name": "prefill-64-at-32768", "kind": "attn", **WIDE, "seqs": 1, "new_low": 64,
         "new_high": 64, "past_low": 32768, "past_high": 32768, "page": 64, "window": 0,
         "sinks": 0, "lengths": 8},
        # A long prompt.
        {"name": "prefill-8192", "kind": "attn", **WIDE, "seqs": 1, "new_low": 8192,
         "new_high": 8192, "past_low": 0, "past_high": 0, "page": 64, "window": 0, "sinks": 0,
         "lengths": 9},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """Half the time the benchmark's heads, else any of the supported ones."""
    if rng.random() < 0.5:
        return dict(WIDE)
    kv = rng.choice((1, 2, 3, 4, 5, 8))
    return {"heads": kv * rng.randint(1, 8), "kv_heads": kv, "head_dim": rng.choice((64, 128))}


def _window(rng, longest):
    if rng.random() < 0.5:
        return {"window": 0, "sinks": 0}
    return {"window": _log_int(rng, 1, max(2, longest)), "sinks": rng.choice((0, 1, 4, 4, 37, 100))}


def draw(rng):
    kind = rng.choice(("plan", "prologue", "decode", "decode", "prefill", "prefill"))
    page = rng.choice((32, 64, 64, 128, 256))
    if kind == "plan":
        seqs, past = _log_int(rng, 1, 2048), _log_int(rng, 30, 30000)
        new = rng.choice((1, 1, 4, 100))
        if seqs * new > 60000:
            new = 4
        return {"kind": "plan", "seqs": seqs, "past": past, "new_low": rng.choice((0, 1)),
                "new_high": new, "page": page, "blocks": (past + new) // page + rng.randint(1, 9),
                **_window(rng, past), "lengths": rng.randint(0, 1 << 30)}
    if kind == "prologue":
        while True:
            c = {"kind": "prologue", **_heads(rng), "pairing": rng.choice(("neox", "norm")),
                 "tokens": _log_int(rng, 1, 8192), "past": _log_int(rng, 1, 100000), "page": page,
                 "stacked": rng.random() < 0.5, "run": rng.choice((1, 5, 777, 8192))}
            if work(c)["bytes"] < 2.5e8:
                return c
    while True:
        few = kind == "decode"
        seqs = _log_int(rng, 1, 128 if few else 8)
        low, high = (1, rng.choice((1, 1, 1, 3, 5))) if few else (rng.choice((0, 1, 9)),
                                                                  _log_int(rng, 9, 8192))
        past = _log_int(rng, 30, 131072 if few else 32768)
        c = {"kind": "attn", **_heads(rng), "seqs": seqs, "new_low": low, "new_high": high,
             "past_low": 0 if not few and rng.random() < 0.4 else past // rng.choice((1, 3, 50)),
             "past_high": past, "page": page, **_window(rng, past),
             "lengths": rng.randint(0, 1 << 30)}
        # What the plain form has to hold, padded, and the products.
        keys = seqs * (past + high) * c["kv_heads"] * c["head_dim"]
        scores = seqs * high * c["heads"] * (past + high)
        if keys < 1.1e9 and scores < 1.1e9 and work(c)["flops"] < 2.7e11:
            return c


# ------------------------------------------------------------------ lengths --
def _lengths(case):
    """(keys after the step, new tokens) of each sequence, from the case."""
    r = random.Random(case["lengths"])
    new = [r.randint(case["new_low"], case["new_high"]) for _ in range(case["seqs"])]
    past = [r.randint(case["past_low"], case["past_high"]) for _ in range(case["seqs"])]
    if not any(new):
        new[0] = case["new_high"]
    return [a + b for a, b in zip(past, new)], new


def _wanted(keys, new, blocks, page, window, sinks):
    """Which blocks a sequence holds, [seqs][blocks] (numpy)."""
    keys, new = np.asarray(keys)[:, None], np.asarray(new)[:, None]
    i = np.arange(blocks)[None]
    first = np.maximum(0, keys - new - window + 1)
    return (i * page < keys) & ((window == 0) | ((i + 1) * page > first) | (i * page < sinks))


def _plan_lengths(case):
    """(keys, new, held): a sixteenth of the sequences ends in this step, a
    sixteenth begins; the others hold what the step before left them."""
    r = random.Random(case["lengths"])
    keys, new, before = [], [], []
    for _ in range(case["seqs"]):
        what, past = r.random(), r.randint(1, case["past"])
        n = r.randint(case["new_low"], case["new_high"])
        if what < 1 / 16:
            keys.append(0), new.append(0), before.append(past)
        elif what < 1 / 8:
            n = max(1, n)
            keys.append(n), new.append(n), before.append(0)
        else:
            keys.append(past + n), new.append(n), before.append(past)
    args = (case["blocks"], case["page"], case["window"], case["sinks"])
    held = _wanted(before, [min(1, b) for b in before], *args)
    need = int((_wanted(keys, new, *args) & ~held).sum())
    return keys, new, held, int(held.sum()) + need + need // 4 + 16


# ------------------------------------------------------------------- inputs --
def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _i32(values):
    return torch.as_tensor(np.asarray(values, np.int64).astype(np.int32), device="cuda")


def _inv_freq(d):
    return torch.tensor([1.0 / math.pow(ROPE_BASE, 2.0 * j / d) for j in range(d // 2)],
                        dtype=torch.float32, device="cuda")


def _pool(gen, pages, kv_heads, page, d):
    """A filled pool: codes with a bell's shape (two 3-bit numbers and a bit),
    scales of rows near unit size with the sign of the largest value."""
    shape = (pages, kv_heads, page // 32, 36 * d)

    def bits(mask):
        return torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda",
                             generator=gen).bitwise_and_(mask)

    pool = bits(0x77).add_(bits(0x77)).add_(bits(0x11))
    for at in (16 * d, 34 * d):
        u = torch.rand(*shape[:3], d, device="cuda", generator=gen) * 2 - 1
        scale = (u * 0.25 + u.sign() * 0.25).bfloat16().half()
        pool[..., at:at + 2 * d] = scale.view(torch.uint8)
    return pool


def _table(gen, held):
    """Pages dealt out at random to the held blocks; -1 elsewhere."""
    held = torch.from_numpy(held).cuda()
    n = int(held.sum())
    table = torch.full(held.shape, -1, dtype=torch.int32, device="cuda")
    table[held] = torch.randperm(n, device="cuda", generator=gen).int()
    return table, n


def _attn_inputs(case, seed):
    keys, new = _lengths(case)
    page = case["page"]
    blocks = -(-max(keys) // page)
    gen = _gen(seed)
    table, pages = _table(gen, _wanted(keys, new, blocks, page, case["window"], case["sinks"]))
    pages = max(1, pages)
    H, d = case["heads"], case["head_dim"]
    q = torch.randn(sum(new), H, d, device="cuda", generator=gen)
    return {"q": q, "table": table, "pages": pages, "blocks": blocks, "keys": _i32(keys),
            "q_off": _i32(np.concatenate([[0], np.cumsum(new)])), "max_q": max(new),
            "max_keys": max(keys), "pool": _pool(gen, pages, case["kv_heads"], page, d)}


def _prologue_inputs(case, seed):
    n, H, G, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    gen = _gen(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    qkv = randn(n, (H + 2 * G) * d)
    q, k, v = (qkv[:, :H * d], qkv[:, H * d:(H + G) * d], qkv[:, (H + G) * d:])
    if not case["stacked"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    # Runs of tokens (prompts; a decode step has runs of one), each at its own
    # position of a sequence whose pages lie anywhere.
    page, run = case["page"], min(case["run"], n)
    runs = -(-n // run)
    past = torch.randint(0, case["past"] + 1, (runs,), device="cuda", generator=gen)
    t = torch.arange(n, device="cuda")
    pos = past[t // run] + t % run
    per = (run + page - 1) // page + 1  # pages that a run can touch
    pages = torch.randperm(runs * per, device="cuda", generator=gen)
    block = pos // page - (past // page)[t // run]
    slots = pages[(t // run) * per + block] * page + pos % page
    return {"q": q, "k": k, "v": v, "gq": 1 + 0.1 * randn(d), "gk": 1 + 0.1 * randn(d),
            "inv": _inv_freq(d), "pos": pos.int(), "slots": slots.int(), "pages": runs * per}


def _plan_inputs(case, seed):
    keys, new, held, pages = _plan_lengths(case)
    gen = _gen(seed)
    table, used = _table(gen, held)
    perm = torch.randperm(pages, device="cuda", generator=gen).int()
    table = torch.where(table >= 0, perm[table.clamp(min=0).long()], -1).int()
    free = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    free[0] = pages - used
    free[1:1 + pages - used] = perm[used:]
    return {"keys": _i32(keys), "new": _i32(new), "table": table, "free": free, "pages": pages,
            "tokens": max(1, sum(new))}


class _State:
    """What a serving program holds between calls."""

    def __init__(self, case, **kw):
        self.case = case
        self.__dict__.update(kw)


def prepare(case, seed):
    if case["kind"] == "plan":
        x = _plan_inputs(case, seed)
        i32 = dict(dtype=torch.int32, device="cuda")
        return _State(case, **x, table_out=torch.zeros_like(x["table"]),
                      free_out=torch.zeros_like(x["free"]),
                      q_off=torch.zeros(case["seqs"] + 1, **i32),
                      pos=torch.zeros(x["tokens"], **i32), slots=torch.zeros(x["tokens"], **i32),
                      lost=torch.zeros(1, **i32),
                      ws=torch.empty(64 * case["seqs"] + 4096, dtype=torch.uint8, device="cuda"))
    if case["kind"] == "prologue":
        x = _prologue_inputs(case, seed)
        n, H, G, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        return _State(case, **x, qn=torch.zeros(n, H, d, device="cuda"),
                      k_out=torch.zeros(n, G, d, device="cuda"),
                      v_out=torch.zeros(n, G, d, device="cuda"),
                      pool=torch.zeros(x["pages"], G, case["page"] // 32, 36 * d,
                                       dtype=torch.uint8, device="cuda"))
    x = _attn_inputs(case, seed)
    return _State(case, **x, o=torch.zeros_like(x["q"]),
                  ws=torch.empty(256 << 20, dtype=torch.uint8, device="cuda"))


# --------------------------------------------------------------- plain forms --
def _plain_plan(s):
    c = s.case
    page, window, sinks = c["page"], c["window"], c["sinks"]
    blocks, pages, total = c["blocks"], s.pages, s.tokens
    keys, new = s.keys.long(), s.new.long()
    i = torch.arange(blocks, device="cuda")
    first = (keys - new - window + 1).clamp(min=0)[:, None]
    want = (i * page < keys[:, None]) & (torch.full_like(i, window == 0, dtype=torch.bool)
                                         | ((i + 1) * page > first) | (i * page < sinks))
    have = (s.table >= 0) & (s.table < pages)
    need, drop = want & ~have, have & ~want
    n_free = s.free[0].long()
    rank = need.flatten().cumsum(0).view_as(need) - 1
    got = need & (rank < n_free)
    taken = s.free[1:][(n_free - 1 - rank).clamp(0, max(pages - 1, 0))]
    table = torch.where(got, taken, torch.where(need | drop, -1, s.table)).int()
    left = n_free - torch.minimum(need.sum(), n_free)
    at = torch.arange(pages, device="cuda")
    rest = torch.where(at < left, s.free[1:], 0)
    places = torch.where(drop, left + drop.flatten().cumsum(0).view_as(drop) - 1, pages)
    rest = torch.cat([rest, rest[:1]]).scatter(0, places.flatten(), torch.where(
        drop, s.table, 0).flatten())[:pages]
    free = torch.cat([(left + drop.sum())[None], rest.long()]).int()
    ends = new.cumsum(0)
    q_off = torch.cat([torch.zeros_like(ends[:1]), ends])
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(ends, t, right=True).clamp(max=len(keys) - 1)
    live = t < ends[-1]
    pos = torch.where(live, keys[b] - new[b] + t - q_off[b], 0)
    entry = table[b, (pos // page).clamp(max=blocks - 1)].long()
    ok = live & (pos < blocks * page) & (entry >= 0)
    slots = torch.where(ok, entry * page + pos % page, -1)
    return {"table": table, "free": free, "q_off": q_off.int(), "positions": pos.int(),
            "slots": slots.int(), "lost": (ends[-1] - ok.sum())[None].int()}


def _plain_norm_rope(x, gain, inv, pos, pairing):
    """RMSNorm and rotation with the roundings the framework's ops define:
    pairwise sums of squares, one rounding of 1 / sqrt, exact products before
    each rounded sum of the rotation. x [n][heads][d]."""
    d = x.shape[-1]
    p = x * x
    while p.shape[-1] > 1:
        h = p.shape[-1] // 2
        p = p[..., :h] + p[..., h:]
    scale = (1.0 / torch.sqrt((p / d + EPS).double())).float()
    x = (x * scale) * gain
    theta = (pos.double()[:, None] * inv.double()).float().double()
    c, s = torch.cos(theta).float()[:, None], torch.sin(theta).float()[:, None]
    a, b = x.chunk(2, -1) if pairing == "neox" else (x[..., 0::2], x[..., 1::2])
    first = (-b.double() * s.double() + (a * c).double()).float()
    second = (b.double() * c.double() + (a * s).double()).float()
    if pairing == "neox":
        return torch.cat([first, second], -1)
    return torch.stack([first, second], -1).flatten(-2)


def _plain_quant(x):
    """The values that rows x [..., d] have in 4 bits."""
    y = x.unflatten(-1, (-1, 32))
    high, low = y.amax(-1, keepdim=True), y.amin(-1, keepdim=True)
    m = torch.where(high >= -low, high, low)
    d = (m / -8).clamp(-8160, 8160).bfloat16().half().float()
    inv = torch.where(d == 0, 0.0, 1.0 / d)
    values = (y * inv).round().clamp(-8, 7) * d
    return torch.where(torch.isfinite(y).all(-1, keepdim=True), values, math.nan).flatten(-2)


def _plain_prologue(s):
    c = s.case
    n, d = c["tokens"], c["head_dim"]
    q, k, v = (x.reshape(n, -1, d) for x in (s.q, s.k, s.v))
    k = _plain_norm_rope(k, s.gk, s.inv, s.pos, c["pairing"])
    return {"qn": _plain_norm_rope(q, s.gq, s.inv, s.pos, c["pairing"]), "k": _plain_quant(k),
            "v": _plain_quant(v)}


def _plain_unpack(pool, table, d):
    """K and V of every block of every sequence, f32 [seqs][kv heads][keys][d]."""
    x = pool[table.clamp(min=0).long()].transpose(1, 2)  # [seqs][kv heads][blocks][tiles][36 d]
    x = x.flatten(2, 3)
    lead = x.shape[:3]
    kc, ks, vc, vs = x.split((16 * d, 2 * d, 16 * d, 2 * d), -1)

    def nibbles(t):
        return torch.stack([t & 15, t >> 4], -1)

    dims = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device=x.device)
    kc = nibbles(kc).view(*lead, -1, 8)[..., dims]
    if d == 128:
        kc = kc.view(*lead, 2, 16, 4, 32)
    else:
        kc = kc.view(*lead, 16, 4, 2, 16).permute(0, 1, 2, 5, 3, 4, 6)
    ks = ks.contiguous().view(torch.float16).view(*lead, 16, d // 32, 2)
    ks = ks.permute(0, 1, 2, 5, 3, 4).float()
    k = (kc.reshape(*lead, 2, 16, d // 32, 32).float() - 8) * ks[..., None]
    # chunk, g, n, half, token of four, nibble -> half, g, token, n, chunk, nibble
    vc = nibbles(vc).view(*lead, d // 64, 4, 16, 2, 4, 4).permute(0, 1, 2, 6, 4, 7, 5, 3, 8)
    vs = vs.contiguous().view(torch.float16).view(*lead, 4, d // 32, 2, 4)
    vs = vs.permute(0, 1, 2, 5, 3, 6, 4).float()
    v = (vc.reshape(*lead, 2, 4, 4, d // 32, 32).float() - 8) * vs[..., None]
    return (y.reshape(*lead[:2], -1, d) for y in (k, v))


def _plain_attn(s):
    c = s.case
    H, G, d, B = c["heads"], c["kv_heads"], c["head_dim"], c["seqs"]
    k, v = _plain_unpack(s.pool, s.table, d)
    k, v = k[:, :, :s.max_keys], v[:, :, :s.max_keys]
    new = s.q_off[1:] - s.q_off[:-1]
    i = torch.arange(s.max_q, device="cuda")
    rows = (s.q_off[:-1, None] + i).clamp(max=max(s.q.shape[0] - 1, 0)).long()
    q = s.q[rows].view(B, s.max_q, G, H // G, d).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.reshape(B, G, -1, d) * (1 / math.sqrt(d)), k.transpose(2, 3))
    scores = scores.view(B, G, H // G, s.max_q, s.max_keys)
    p = ((s.keys - new)[:, None] + i)[..., None]
    j = torch.arange(s.max_keys, device="cuda")
    seen = j <= p
    if c["window"]:
        seen &= (j > p - c["window"]) | (j < c["sinks"])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    weights = torch.exp_(scores.sub_(top))
    total = weights.sum(-1, keepdim=True)
    o = torch.matmul(weights.view(B, G, -1, s.max_keys), v).view(B, G, H // G, s.max_q, d)
    o = torch.where(total > 0, o / total, 0).permute(0, 3, 1, 2, 4).reshape(B, s.max_q, H, d)
    return {"o": o[i < new[:, None]]}


# ---------------------------------------------------------------------- runs --
def run(s):
    c = s.case
    kind = c["kind"]
    if not own:
        if kind == "plan":
            return _plain_plan(s)
        return _plain_prologue(s) if kind == "prologue" else _plain_attn(s)
    from flock_amd import ops
    if kind == "plan":
        ops.kv4_plan(s.keys, s.new, s.table, s.table_out, s.free, s.free_out, s.q_off, s.pos,
                     s.slots, s.lost, c["seqs"], c["blocks"], s.pages, s.tokens, c["page"],
                     c["window"], c["sinks"], (s.ws, s.ws.numel()))
        return {"table": s.table_out, "free": s.free_out, "q_off": s.q_off, "positions": s.pos,
                "slots": s.slots, "lost": s.lost}
    H, G, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    if kind == "prologue":
        n = c["tokens"]
        ops.kv4_prologue(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.gq, s.gk, s.inv, EPS,
                         c["pairing"], s.pos, s.slots, s.qn, s.pool, n, H, G, d, s.pages, page,
                         in_stride=(H + 2 * G) * d if c["stacked"] else 0)
        ops.kv4_read(s.pool, s.slots, s.k_out, s.v_out, n, G, d, s.pages, page)
        return {"qn": s.qn, "k": s.k_out, "v": s.v_out}
    ops.kv4_attn(s.q, s.pool, s.table, s.keys, s.q_off, s.o, c["seqs"], s.q.shape[0], s.max_q,
                 s.max_keys, s.blocks, H, G, d, s.pages, page, c["window"], c["sinks"],
                 (s.ws, s.ws.numel()))
    return {"o": s.o}


# ---------------------------------------------------------------------- work --
def _seen(first, last, window, sinks):
    """Keys that queries at positions first .. last see: (together, summed)."""
    if not window:
        return last + 1, (last + 1) * (last + 2) // 2 - first * (first + 1) // 2
    begin = max(0, first - window + 1)
    together = last + 1 - begin + min(sinks, begin)
    p = np.arange(first, last + 1, dtype=np.int64)
    begins = np.maximum(0, p - window + 1)
    return together, int((p + 1 - begins + np.minimum(sinks, begins)).sum())


def work(case):
    if case["kind"] == "plan":
        _, new, held, pages = _plan_lengths(case)
        seqs = case["seqs"]
        return {"bytes": 8 * seqs * case["blocks"] + 8 * (pages - int(held.sum())) + 12 * seqs
                + 8 * sum(new), "flops": 0}
    H, G, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "prologue":
        # Raw rows in, q out, the cache's bytes out and in again, rows out.
        n = case["tokens"]
        return {"bytes": n * (4 * d * (2 * H + 4 * G) + 2 * G * d * 9 // 8 + 8), "flops": 0}
    keys, new = _lengths(case)
    together = pairs = 0
    for k, n in zip(keys, new):
        if n:
            a, b = _seen(k - n, k - 1, case["window"], case["sinks"])
            together, pairs = together + a, pairs + b
    return {"bytes": together * G * d * 9 // 8 + 8 * sum(new) * H * d, "flops": 4.0 * H * d * pairs}


# --------------------------------------------------------- 64-bit references --
def _places(d):
    """Where token t of a tile and dim e lie: (byte, shift) of K's and V's codes
    and the byte of their scales, each [32][d]."""
    t, e = np.meshgrid(np.arange(32), np.arange(d), indexing="ij")
    half, key = t // 16, t % 16
    part, inside = e // (d // 4), e % (d // 4)
    piece = d // 8  # bytes of a part
    at = (half * 64 + key * 4 + part) if d == 128 else (key * 8 + part * 2 + half)
    octet, u = inside // 8, inside % 8
    nib = u // 2 + 4 * (u % 2)
    k_byte, k_shift = at * piece + octet * 4 + nib // 2, 4 * (nib % 2)
    ks = 16 * d + 2 * ((key * (d // 32) + e // 32) * 2 + half)
    g, slot = key // 4, key % 4 + 4 * half
    n, rest = e // (d // 16), e % (d // 16)
    word = ((rest // 4 * 4 + g) * 16 + n) * 8 + slot
    v_byte, v_shift = 18 * d + 2 * word + rest % 4 // 2, 4 * (rest % 2)
    vs = 34 * d + 2 * ((g * (d // 32) + e // 32) * 8 + slot)
    return [torch.from_numpy(a).cuda() for a in (k_byte, k_shift, ks, v_byte, v_shift, vs)]


def _tile64(tiles, byte, shift, scale):
    """tiles [n][36 d] bytes -> [n * 32][d] values in 64 bits."""
    code = (tiles[:, byte].long() >> shift) & 15
    bits = tiles[:, scale].int() | (tiles[:, scale + 1].int() << 8)
    d = torch.where(bits > 32767, bits - 65536, bits).short().view(torch.float16).double()
    return ((code - 8) * d).flatten(0, 1)


def _attn64(case, seed):
    x = _attn_inputs(case, seed)
    keys, new = _lengths(case)
    H, G, d = case["heads"], case["kv_heads"], case["head_dim"]
    group, places = H // G, _places(d)
    o = torch.zeros(sum(new), H, d, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, m) in enumerate(zip(keys, new)):
        if not m:
            continue
        pos = torch.arange(n - m, n, device="cuda")
        j = torch.arange(n, device="cuda")
        hidden = j > pos[:, None]
        if case["window"]:
            hidden |= (j <= pos[:, None] - case["window"]) & (j >= case["sinks"])
        pages = x["table"][b, :-(-n // case["page"])].clamp(min=0).long()
        for g in range(G):
            tiles = x["pool"][pages, g].flatten(0, 1)
            k, v = _tile64(tiles, *places[:3])[:n], _tile64(tiles, *places[3:])[:n]
            for h in range(g * group, (g + 1) * group):
                p = (x["q"][row:row + m, h].double() @ k.t()) / math.sqrt(d)
                p = torch.softmax(p.masked_fill_(hidden, -math.inf), -1)
                o[row:row + m, h] = p @ v
        row += m
    return o


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    if case["kind"] == "attn":
        return {"o": _attn64(case, seed)}
    x = _prologue_inputs(case, seed)
    n, H, d = case["tokens"], case["heads"], case["head_dim"]
    q = x["q"].reshape(n, H, d).double()
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * x["gq"].double()
    # The angle is position * inv_freq rounded to 32 bits, as the op defines it.
    angle = (x["pos"].double()[:, None] * x["inv"].double()).float().double()[:, None]
    z = torch.view_as_complex(torch.stack(
        [q[..., :d // 2], q[..., d // 2:]] if case["pairing"] == "neox" else
        [q[..., 0::2], q[..., 1::2]], -1)) * torch.polar(torch.ones_like(angle), angle)
    q = torch.cat([z.real, z.imag], -1) if case["pairing"] == "neox" else torch.view_as_real(
        z).flatten(-2)
    return {"qn": q, "k": None, "v": None}  # codes at a border have no value in 64 bits
