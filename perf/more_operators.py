"""Several answers to one prompt, as measurable cases.

Three operators: attention of a decode step whose sequences share long
prefixes (alone, and as a layer's whole step with norm, rotation and append),
the log probabilities of given tokens with entropy and top alternatives, and
sampling from the top alternatives by given uniform numbers.

Caches are [rows][kv_heads][head_dim] in f32. Group g's prefix lies at rows
prefix_row[g] .. + n_prefix[g], its sequences are seq_off[g] .. seq_off[g + 1],
and sequence b's own keys lie at rows seq_row_off[b] .. + n_keys[b].
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
VOCAB = 151936


def listed():
    return [
        # A few answers to a short question, early on: bound by latency.
        {"name": "step-4x513", "kind": "step", **WIDE, "groups": 1, "seqs": 4, "prefix_low": 513,
         "prefix_high": 513, "own_low": 9, "own_high": 9, "pairing": "neox", "stacked": False,
         "lengths": 1},
        # One layer's step of 64 answers to a prompt of 8192 tokens.
        {"name": "step-64x8k", "kind": "step", **WIDE, "groups": 1, "seqs": 64,
         "prefix_low": 8192, "prefix_high": 8192, "own_low": 257, "own_high": 257,
         "pairing": "neox", "stacked": True, "lengths": 2},
        # 16 questions about one long document, answers of any length so far.
        {"name": "attn-16x32k", "kind": "attn", **WIDE, "groups": 1, "seqs": 16,
         "prefix_low": 32768, "prefix_high": 32768, "own_low": 1, "own_high": 900, "lengths": 3},
        # A server's batch: five prompts of odd lengths, 200 answers, 64-wide heads.
        {"name": "attn-5-groups", "kind": "attn", **NARROW, "groups": 5, "seqs": 200,
         "prefix_low": 300, "prefix_high": 9000, "own_low": 0, "own_high": 700, "lengths": 4},
        # 128 answers to a document of 131072 tokens: products count.
        {"name": "attn-128x128k", "kind": "attn", **WIDE, "groups": 1, "seqs": 128,
         "prefix_low": 131072, "prefix_high": 131072, "own_low": 1, "own_high": 300,
         "lengths": 5},
        # The log probability of each generated token, with five alternatives.
        {"name": "score-1", "kind": "score", "rows": 1, "vocab": VOCAB, "pad": 0, "top": 5,
         "masked": False},
        # A step of 64 answers, 20 alternatives each.
        {"name": "score-64", "kind": "score", "rows": 64, "vocab": VOCAB, "pad": 0, "top": 20,
         "masked": False},
        # Rows of an odd vocabulary inside wider rows, most ids masked by a grammar.
        {"name": "score-333-odd", "kind": "score", "rows": 333, "vocab": 32003, "pad": 62,
         "top": 64, "masked": True},
        # A prompt's own log probabilities (perplexity): no alternatives.
        {"name": "score-2048", "kind": "score", "rows": 2048, "vocab": VOCAB, "pad": 0, "top": 0,
         "masked": False},
        # The next token of one answer, and of the answers of a full batch.
        {"name": "sample-1", "kind": "sample", "rows": 1, "vocab": VOCAB, "pad": 0, "top": 20,
         "masked": False},
        {"name": "sample-256", "kind": "sample", "rows": 256, "vocab": VOCAB, "pad": 0, "top": 50,
         "masked": False},
        # A smaller odd vocabulary with a grammar's mask.
        {"name": "sample-100-odd", "kind": "sample", "rows": 100, "vocab": 50021, "pad": 11,
         "top": 64, "masked": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """Half the time the benchmark's heads, else any of the supported ones."""
    if rng.random() < 0.5:
        return dict(WIDE)
    kv = rng.choice((1, 2, 3, 4, 5, 8))
    return {"heads": kv * rng.randint(1, 8), "kv_heads": kv, "head_dim": rng.choice((64, 128))}


def draw(rng):
    kind = rng.choice(("step", "attn", "attn", "score", "sample"))
    if kind in ("score", "sample"):
        while True:
            top = rng.choice((0, 1, 5, 20, 64) if kind == "score" else (1, 5, 20, 50, 64))
            c = {"kind": kind, "rows": _log_int(rng, 1, 2048), "vocab": _log_int(rng, 200, 200000),
                 "pad": rng.choice((0, 0, 1, 3, 64)), "top": top}
            c["masked"] = c["vocab"] > 1000 and rng.random() < 0.4
            # (The plain form sorts whole rows.)
            if c["rows"] * c["vocab"] < (1 << 28 if top == 0 else 40e6):
                return c
    while True:
        groups = rng.choice((1, 1, 1, 2, 5, 12))
        seqs = groups * _log_int(rng, 1, 256)
        prefix = _log_int(rng, 1, 131072)
        longest = _log_int(rng, 1, 2000)
        c = {"kind": kind, **_heads(rng), "groups": groups, "seqs": seqs,
             "prefix_low": max(1, prefix // rng.choice((1, 1, 5))), "prefix_high": prefix,
             "lengths": rng.randint(0, 1 << 30)}
        if kind == "step":  # answers go in step
            c.update(own_low=longest, own_high=longest, pairing=rng.choice(("neox", "norm")),
                     stacked=rng.random() < 0.5)
        else:
            c.update(own_low=rng.choice((0, 1, longest)), own_high=longest)
        # What the plain form has to hold: scores, and own keys padded to the longest.
        scores = seqs * c["heads"] * (prefix + longest)
        rows = (groups * prefix + 2 * seqs * longest) * c["kv_heads"] * c["head_dim"]
        if scores < 2.8e8 and rows < 5e8 and work(c)["flops"] < 1.3e11:
            return c


# ------------------------------------------------------------------ lengths --
def _lengths(case):
    """(prefix of each group, first sequence of each group and the end, own
    keys of each sequence), from the case."""
    r = random.Random(case["lengths"])
    groups, seqs = case["groups"], case["seqs"]
    prefix = [r.randint(case["prefix_low"], case["prefix_high"]) for _ in range(groups)]
    cuts = sorted(r.randint(0, seqs) for _ in range(groups - 1))
    own_keys = [r.randint(case["own_low"], case["own_high"]) for _ in range(seqs)]
    return prefix, [0] + cuts + [seqs], own_keys


# ------------------------------------------------------------------- inputs --
def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _inv_freq(d):
    return torch.tensor([1.0 / math.pow(ROPE_BASE, 2.0 * j / d) for j in range(d // 2)],
                        dtype=torch.float32, device="cuda")


def _attn_inputs(case, seed):
    prefix, off, own_keys = _lengths(case)
    H, G, d, B = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    gen = _gen(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def i64(x):
        return torch.tensor(x, dtype=torch.int64, device="cuda")

    cap = max(own_keys) + 8  # rows kept for each answer
    starts = np.concatenate([[0], np.cumsum(prefix)])
    own_row = int(starts[-1]) + cap * np.arange(B)
    rows = int(starts[-1]) + cap * B
    x = {"prefix_row": i64(starts[:-1].tolist()), "n_prefix": i32(prefix), "seq_off": i32(off),
         "seq_row_off": i64(own_row.tolist()), "n_keys": i32(own_keys), "cap": cap,
         "own_at": int(starts[-1]), "max_prefix": max(prefix), "max_keys": max(1, max(own_keys)),
         "kcache": randn(rows, G, d), "vcache": randn(rows, G, d)}
    if case["kind"] == "attn":
        # Normed heads with gains near 2: some keys stand out.
        return {**x, "q": 2 * randn(B, H, d)}
    qkv = randn(B, (H + 2 * G) * d)
    q, k, v = (qkv[:, :H * d], qkv[:, H * d:(H + G) * d], qkv[:, (H + G) * d:])
    if not case["stacked"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return {**x, "q": q, "k": k, "v": v, "gq": 2 + 0.1 * randn(d), "gk": 1 + 0.1 * randn(d),
            "inv": _inv_freq(d)}


def _logits(case, seed):
    """Logits as a language model's: a bell with a few ids far above it, in some
    rows one id above all; a grammar's mask leaves an eighth of the ids."""
    n, V = case["rows"], case["vocab"]
    gen = _gen(seed)
    wide = torch.randn(n, V + case["pad"], device="cuda", generator=gen).mul_(2.5)
    x = wide[:, :V]
    few = torch.randint(0, V, (n, 12), device="cuda", generator=gen)
    x.scatter_add_(1, few, 6 + 4 * torch.randn(n, 12, device="cuda", generator=gen))
    sure = torch.rand(n, device="cuda", generator=gen) < 0.3
    x[torch.arange(n, device="cuda"), few[:, 0]] += 15.0 * sure
    if case["masked"]:
        step = torch.randint(0, 8, (n, 1), device="cuda", generator=gen)
        x.masked_fill_((torch.arange(V, device="cuda") + step) % 8 != 0, -math.inf)
        few = few - (few + step) % 8
        few += 8 * (few < 0)
    # Given tokens: likely ones, and some that are not.
    tokens = few[torch.arange(n, device="cuda"), torch.randint(0, 12, (n,), device="cuda",
                                                               generator=gen)]
    return x, tokens, gen


def _choices(case, gen):
    """Settings of each row, and a uniform number."""
    n = case["rows"]

    def rand():
        return torch.rand(n, device="cuda", generator=gen)

    temperature = torch.where(rand() < 0.1, 0.0, 0.3 + 1.2 * rand())
    top_k = torch.randint(1, case["top"] + 1, (n,), device="cuda", generator=gen).int()
    top_k = torch.where(rand() < 0.5, case["top"], top_k).int()
    top_p = torch.where(rand() < 0.3, 1.0, 0.5 + 0.5 * rand())
    min_p = torch.where(rand() < 0.5, 0.0, 0.1 * rand())
    return {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "uniform": rand()}


class _State:
    """What a serving program holds between calls."""

    def __init__(self, case, **kw):
        self.case = case
        self.__dict__.update(kw)


def prepare(case, seed):
    if case["kind"] in ("step", "attn"):
        x = _attn_inputs(case, seed)
        B, H, d = case["seqs"], case["heads"], case["head_dim"]
        return _State(case, **x, o=torch.zeros(B, H, d, device="cuda"),
                      qn=torch.zeros(B, H, d, device="cuda"),
                      ws=torch.empty(1 << 30, dtype=torch.uint8, device="cuda"))
    x, tokens, gen = _logits(case, seed)
    n, k = case["rows"], max(1, case["top"])
    i32 = dict(dtype=torch.int32, device="cuda")
    more = {"uniform": None} if case["kind"] == "score" else _choices(case, gen)
    return _State(case, **more, logits=x, tokens=tokens.int(),
                  logprob=torch.zeros(n, device="cuda"), entropy=torch.zeros(n, device="cuda"),
                  top_ids=torch.zeros(n, k, **i32), top_logprobs=torch.zeros(n, k, device="cuda"),
                  token=torch.zeros(n, **i32),
                  ws=torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))


# --------------------------------------------------------------- plain forms --
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


def _plain_attn(s, q):
    """Scores over the shared keys as one product for all of a group's rows,
    scores over own keys as one for each sequence, one softmax over both."""
    c = s.case
    H, G, d, B = c["heads"], c["kv_heads"], c["head_dim"], c["seqs"]
    prefix, off, _ = _lengths(c)
    m = H // G
    q = q.view(B, G, m, d) * (1 / math.sqrt(d))
    o = torch.empty(B, G, m, d, device="cuda")
    row = 0
    for g in range(c["groups"]):
        a, b, n = off[g], off[g + 1], prefix[g]
        if a < b:
            k = s.kcache[row:row + n].transpose(0, 1).contiguous()
            v = s.vcache[row:row + n].transpose(0, 1).contiguous()
            x = q[a:b].transpose(0, 1).reshape(G, -1, d)
            shared = torch.matmul(x, k.transpose(1, 2)).view(G, b - a, m, n).transpose(0, 1)
            i = torch.arange(s.max_keys, device="cuda")
            rows = s.seq_row_off[a:b, None] + i
            ko = s.kcache[rows].transpose(1, 2).contiguous()  # [seqs][kv heads][keys][d]
            vo = s.vcache[rows].transpose(1, 2).contiguous()
            mine = torch.matmul(q[a:b], ko.transpose(2, 3))
            hidden = i >= s.n_keys[a:b, None]
            mine.masked_fill_(hidden[:, None, None], -math.inf)
            top = torch.maximum(shared.amax(-1), mine.amax(-1)).clamp(min=-3e38)[..., None]
            shared = torch.exp(shared - top)
            mine = torch.exp(mine - top)
            total = shared.sum(-1, keepdim=True) + mine.sum(-1, keepdim=True)
            x = torch.matmul(shared.transpose(0, 1).reshape(G, -1, n), v)
            x = x.view(G, b - a, m, d).transpose(0, 1) + torch.matmul(mine, vo)
            o[a:b] = x / total
        row += n
    return o.view(B, H, d)


def _new_rows(s):
    """Views of the rows that a step appends: answers go in step."""
    c = s.case
    at, n = s.own_at, c["own_low"]
    return tuple(x[at:].view(c["seqs"], s.cap, c["kv_heads"], c["head_dim"])[:, n - 1]
                 for x in (s.kcache, s.vcache))


def _positions(case):
    prefix, off, own_keys = _lengths(case)
    group = np.repeat(np.arange(case["groups"]), np.diff(off))
    return torch.tensor(np.asarray(prefix)[group] + np.asarray(own_keys) - 1, device="cuda")


def _plain_step(s):
    c = s.case
    B, d = c["seqs"], c["head_dim"]
    q, k, v = (x.reshape(B, -1, d) for x in (s.q, s.k, s.v))
    pos = _positions(c)
    qn = _plain_norm_rope(q, s.gq, s.inv, pos, c["pairing"])
    new_k, new_v = _new_rows(s)
    new_k.copy_(_plain_norm_rope(k, s.gk, s.inv, pos, c["pairing"]))
    new_v.copy_(v)
    return {"o": _plain_attn(s, qn), "qn": qn, "k": new_k, "v": new_v}


def _plain_top(x, k):
    """The k largest with their places, ties to the lowest."""
    top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return top[:, :k], ids[:, :k]


def _plain_logprob(x, tokens):
    top = x.amax(-1, keepdim=True)
    total = torch.exp(x - top).sum(-1, keepdim=True)
    return x.gather(1, tokens[:, None].long()) - top - torch.log(total), top, total


def _plain_score(s):
    x, k = s.logits, s.case["top"]
    lp, top, total = _plain_logprob(x, s.tokens)
    e = torch.exp(x - top)
    spread = torch.where(e > 0, e * (top - x), 0.0).sum(-1)
    out = {"logprob": lp[:, 0], "entropy": torch.log(total[:, 0]) + spread / total[:, 0]}
    if k:
        best, ids = _plain_top(x, k)
        out.update(top_ids=ids.int(), top_logprobs=best - top - torch.log(total))
    return out


def _plain_sample(s):
    """Weights in 64 bits: a uniform number next to a border decides the token."""
    x, k = s.logits, s.case["top"]
    best, ids = _plain_top(x, k)
    best = best.double()
    place = torch.arange(k, device="cuda")
    t = s.temperature.double()[:, None]
    w = torch.where(t > 0, torch.exp((best - best[:, :1]) / t), (place == 0).double())
    w = torch.where(place < s.top_k[:, None], w, 0.0)
    before = w.cumsum(-1) - w
    w = torch.where(before < s.top_p.double()[:, None] * w.sum(-1, keepdim=True), w, 0.0)
    w = torch.where(w >= s.min_p.double()[:, None], w, 0.0)
    sums = w.cumsum(-1)
    at = (sums <= s.uniform.double()[:, None] * sums[:, -1:]).sum(-1)
    at = torch.minimum(at, (w > 0).sum(-1) - 1)
    token = ids.gather(1, at[:, None])[:, 0]
    return {"token": token.int(), "logprob": _plain_logprob(x, token)[0][:, 0]}


# ---------------------------------------------------------------------- runs --
def run(s):
    c = s.case
    kind = c["kind"]
    if not own:
        if kind == "attn":
            return {"o": _plain_attn(s, s.q)}
        return {"step": _plain_step, "score": _plain_score, "sample": _plain_sample}[kind](s)
    from flock_amd import ops
    ws = (s.ws, s.ws.numel())
    if kind in ("score", "sample"):
        n, V, k = c["rows"], c["vocab"], c["top"]
        logits, ld = s.logits.data_ptr(), V + c["pad"]
        if kind == "sample":
            ops.sample(logits, s.uniform, s.token, n, V, k, ws, temperature=s.temperature,
                       top_k=s.top_k, top_p=s.top_p, min_p=s.min_p, logprob=s.logprob, ld=ld)
            return {"token": s.token, "logprob": s.logprob}
        out = {"logprob": s.logprob, "entropy": s.entropy}
        if k:
            out.update(top_ids=s.top_ids, top_logprobs=s.top_logprobs)
        ops.token_logprobs(logits, s.tokens, s.logprob, n, V, ws, entropy=s.entropy, n_top=k,
                           top_ids=s.top_ids if k else None,
                           top_logprobs=s.top_logprobs if k else None, ld=ld)
        return out
    H, G, d = c["heads"], c["kv_heads"], c["head_dim"]
    shared = (s.prefix_row, s.n_prefix, s.seq_off, s.seq_row_off, s.n_keys, s.o, c["groups"],
              c["seqs"], s.max_prefix, s.max_keys, H, G, d, ws)
    if kind == "attn":
        ops.attn_decode_shared(s.q, s.kcache, s.vcache, *shared)
        return {"o": s.o}
    ops.decode_layer_shared(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.gq, s.gk, s.inv, EPS,
                            c["pairing"], s.qn, s.kcache, s.vcache, *shared,
                            in_stride=(H + 2 * G) * d if c["stacked"] else 0)
    k, v = _new_rows(s)
    return {"o": s.o, "qn": s.qn, "k": k, "v": v}


# ---------------------------------------------------------------------- work --
def work(case):
    if case["kind"] in ("score", "sample"):
        n = case["rows"]
        return {"bytes": n * (4 * case["vocab"] + 12 + (8 * case["top"] if case["kind"] == "score"
                                                        else 20)), "flops": 0}
    prefix, off, own_keys = _lengths(case)
    H, G, d, B = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    seqs = np.diff(off)
    rows = sum(p for p, n in zip(prefix, seqs) if n) + sum(own_keys)
    pairs = sum(p * int(n) for p, n in zip(prefix, seqs)) + sum(own_keys)
    extra = 2 * B * (H + 2 * G) * d if case["kind"] == "step" else B * H * d
    return {"bytes": 8 * rows * G * d + 4 * (extra + B * H * d) + 12 * B,
            "flops": 4.0 * H * d * pairs}


# --------------------------------------------------------- 64-bit references --
def _exact_attn(x, case, q):
    prefix, off, own_keys = _lengths(case)
    H, G, d = case["heads"], case["kv_heads"], case["head_dim"]
    o = torch.zeros(case["seqs"], H, d, dtype=torch.float64, device="cuda")
    for h in range(G):
        heads = slice(h * (H // G), (h + 1) * (H // G))
        row = 0
        for g, n in enumerate(prefix):
            kp = x["kcache"][row:row + n, h].double()
            vp = x["vcache"][row:row + n, h].double()
            row += n
            for b0 in range(off[g], off[g + 1], 32):  # a few sequences at a time
                b1 = min(b0 + 32, off[g + 1])
                sp = (q[b0:b1, heads] @ kp.t()) / math.sqrt(d)
                for b in range(b0, b1):
                    r = x["own_at"] + b * x["cap"]
                    ko = x["kcache"][r:r + own_keys[b], h].double()
                    vo = x["vcache"][r:r + own_keys[b], h].double()
                    so = (q[b, heads] @ ko.t()) / math.sqrt(d)
                    p = torch.softmax(torch.cat([sp[b - b0], so], -1), -1)
                    o[b, heads] = p[:, :n] @ vp + p[:, n:] @ vo
    return o


def _exact_step(case, seed):
    x = _attn_inputs(case, seed)
    B, d = case["seqs"], case["head_dim"]
    # The angle is position * inv_freq rounded to 32 bits, as the op defines it.
    angle = (_positions(case).double()[:, None] * x["inv"].double()).float().double()[:, None]

    def turned(rows, gain):
        y = rows.reshape(B, -1, d).double()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * gain.double()
        neox = case["pairing"] == "neox"
        z = torch.complex(y[..., :d // 2], y[..., d // 2:]) if neox else torch.complex(
            y[..., 0::2].contiguous(), y[..., 1::2].contiguous())
        z = z * torch.polar(torch.ones_like(angle), angle)
        return torch.cat([z.real, z.imag], -1) if neox else torch.view_as_real(z).flatten(-2)

    q, k = turned(x["q"], x["gq"]), turned(x["k"], x["gk"])
    v = x["v"].reshape(B, -1, d)
    last = x["own_at"] + x["cap"] * torch.arange(B, device="cuda") + case["own_low"] - 1
    # Attention's own error, not the norm's: it starts from rows rounded to 32 bits.
    x["kcache"][last], x["vcache"][last] = k.float(), v
    return {"o": _exact_attn(x, case, q), "qn": q, "k": k, "v": v.double()}


def _exact_tokens(x, choices):
    """The token of each row: the first alternative at which the distribution
    function of those that stay exceeds the row's number."""
    temperature, top_k, top_p, min_p, uniform = (choices[n].cpu().numpy() for n in (
        "temperature", "top_k", "top_p", "min_p", "uniform"))
    tokens = []
    for b, row in enumerate(x):
        row = row.cpu().numpy()
        least = np.partition(row, -top_k[b])[-top_k[b]]
        ids = np.flatnonzero(row >= least)
        ids = ids[np.argsort(-row[ids], kind="stable")][:top_k[b]]
        if temperature[b] == 0:
            tokens.append(int(ids[0]))
            continue
        values = row[ids].astype(np.float64)
        p = np.exp((values - values[0]) / np.float64(temperature[b]))
        p = p[:1 + np.searchsorted(p.cumsum() / p.sum(), np.float64(top_p[b]))]
        p = p[p >= np.float64(min_p[b])]
        at = np.searchsorted(p.cumsum() / p.sum(), np.float64(uniform[b]), side="right")
        tokens.append(int(ids[min(at, len(p) - 1)]))
    return torch.tensor(tokens)


def exact(case, seed):
    if case["kind"] == "attn":
        x = _attn_inputs(case, seed)
        return {"o": _exact_attn(x, case, x["q"].double())}
    if case["kind"] == "step":
        return _exact_step(case, seed)
    x, tokens, gen = _logits(case, seed)
    if case["kind"] == "sample":
        tokens = _exact_tokens(x, _choices(case, gen)).cuda()
    lp, entropy, tops = [], [], []
    for i in range(0, case["rows"], 64):
        y = x[i:i + 64].double()
        p = torch.log_softmax(y, -1)
        lp.append(p.gather(1, tokens[i:i + 64, None].long())[:, 0])
        entropy.append(-torch.where(p > -math.inf, p.exp() * p, 0.0).sum(-1))
        if case["top"]:
            tops.append(p.topk(case["top"], -1).values)
    if case["kind"] == "sample":
        return {"token": tokens.int(), "logprob": torch.cat(lp)}
    out = {"logprob": torch.cat(lp), "entropy": torch.cat(entropy)}
    if case["top"]:
        out.update(top_ids=None, top_logprobs=torch.cat(tops))
    return out
