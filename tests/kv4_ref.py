"""The paged 4-bit cache in numpy: scales and codes, places of a tile, plans, and
attention in 64 bits."""
from __future__ import annotations

import math

import numpy as np

NONE = 0xFFFFFFFF


def bf16(x):
    """f32 rounded to bf16 (half to even), as f32; x finite."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32)


def quantise(x):
    """x [..., D] f32 -> (codes uint8 [..., D], scales f16 [..., D / 32])."""
    y = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    ok = np.isfinite(y).all(-1)
    z = np.where(ok[..., None], y, np.float32(0))
    hi, lo = z.max(-1), z.min(-1)
    m = np.where(hi >= -lo, hi, lo)
    d = bf16(np.clip(m / np.float32(-8), -8160, 8160)).astype(np.float16)
    f = d.astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(f == 0, np.float32(0), np.float32(1) / f)
    with np.errstate(over="ignore"):
        c = np.clip(np.rint(z * inv[..., None]), -8, 7).astype(np.int32) + 8
    c = np.where(ok[..., None], c, 8).astype(np.uint8)
    d = np.where(ok, d, np.float16(np.nan)).astype(np.float16)
    return c.reshape(x.shape), d


def values(codes, scales):
    d = np.repeat(scales.astype(np.float32), 32, -1)
    return (codes.astype(np.float32) - 8) * d


def places(D):
    """(K byte, K shift, K scale byte, V byte, V shift, V scale byte), each [32][D]."""
    t, e = np.meshgrid(np.arange(32), np.arange(D), indexing="ij")
    half, key, part, octet, u = t // 16, t % 16, e // (D // 4), e % (D // 4) // 8, e % 8
    lane = half * 64 + key * 4 + part if D == 128 else key * 8 + part * 2 + half
    nib = u // 2 + 4 * (u % 2)
    kb = lane * (D // 8) + octet * 4 + nib // 2
    ks = 16 * D + 2 * ((key * (D // 32) + e // 32) * 2 + half)
    g, slot, n, rest = key // 4, key % 4 + 4 * half, e // (D // 16), e % (D // 16)
    vb = 18 * D + 2 * (((rest // 4 * 4 + g) * 16 + n) * 8 + slot) + rest % 4 // 2
    vs = 34 * D + 2 * ((g * (D // 32) + e // 32) * 8 + slot)
    return kb, 4 * (nib % 2), ks, vb, 4 * (rest % 2), vs


def store(pool, slots, k, v, page):
    """k, v [n][G][D] f32 into pool uint8 [pages][G][page / 32][36 D]."""
    D = k.shape[-1]
    kb, ksh, ks, vb, vsh, vs = places(D)
    (kc, kd), (vc, vd) = quantise(k), quantise(v)
    n_slots = pool.shape[0] * page
    for i, s in enumerate(slots):
        if s >= n_slots:
            continue
        tiles = pool[s // page, :, s % page // 32]
        t = s % 32
        for codes, scales, b, sh, at in ((kc, kd, kb, ksh, ks), (vc, vd, vb, vsh, vs)):
            for e in range(D):
                byte = tiles[:, b[t, e]]
                keep = 0xF0 if sh[t, e] == 0 else 0x0F
                tiles[:, b[t, e]] = (byte & keep) | (codes[i, :, e] << sh[t, e])
            for e in range(0, D, 32):
                two = np.ascontiguousarray(scales[i, :, e // 32]).view(np.uint8).reshape(-1, 2)
                tiles[:, at[t, e]] = two[:, 0]
                tiles[:, at[t, e] + 1] = two[:, 1]


def load(pool, page):
    """(k, v) f32 [pages * page][G][D] of a whole pool."""
    P, G, T, nb = pool.shape
    D = nb // 36
    kb, ksh, ks, vb, vsh, vs = places(D)

    def one(b, sh, at):
        c = (pool[..., b] >> sh.astype(np.uint8)) & 15
        d = (pool[..., at].astype(np.uint16) | (pool[..., at + 1].astype(np.uint16) << 8))
        x = (c.astype(np.float32) - 8) * d.view(np.float16).astype(np.float32)
        return x.transpose(0, 2, 3, 1, 4).reshape(P * page, G, D)

    with np.errstate(invalid="ignore"):
        return one(kb, ksh, ks), one(vb, vsh, vs)


def mark(page_id, key, n_pages, page):
    """The entry of a page whose block's keys from its `key`-th on were not stored."""
    half = n_pages * page >= 1 << 31
    return 1 << 31 | page_id * (page >> half) | key >> half


def unmark(entry, n_pages, page):
    """(page id, or n_pages or more for none; the first of its keys that was not stored)"""
    if entry < 1 << 31:
        return entry, page
    half = n_pages * page >= 1 << 31
    page_id, key = divmod(entry - (1 << 31), page >> half)
    return page_id, key << half


def plan(n_keys, n_new, table, free, max_tokens, n_pages, page, window, sinks):
    """The plan, entry by entry. free: list of page ids, the last taken first."""
    table = np.array(table, np.uint32)
    out, left, back = np.full_like(table, NONE), list(free), []
    q_off, pos, slots, missing = [0], [], [], 0
    for b in range(len(n_keys)):
        n, m = int(n_keys[b]), min(int(n_new[b]), int(n_keys[b]))
        first = max(0, n - m - window + 1)
        stored = n - m + min(m, max(0, max_tokens - q_off[-1]))
        ids = [NONE] * table.shape[1]
        for i in range(table.shape[1]):
            want = i * page < n and (not window or (i + 1) * page > first or i * page < sinks)
            page_id, key = unmark(int(table[b, i]), n_pages, page)
            have = page_id < n_pages
            if have and not want:
                back.append(page_id)
            elif (want and i * page + (key if have else 0) < n - m and (not have or key < page)
                  and (window != 1 or i * page < sinks)):
                # Keys before the new ones that rows see were stored nowhere: no page holds them.
                missing += 1
                if have:
                    out[b, i] = table[b, i]
            elif want:
                ids[i] = page_id if have else left.pop() if left else NONE
                out[b, i] = ids[i]
                if stored < n and (i + 1) * page > stored and ids[i] < n_pages:
                    out[b, i] = mark(ids[i], max(0, stored - i * page), n_pages, page)
        q_off.append(q_off[-1] + m)
        for p in range(n - m, n):
            i = p // page
            s = NONE
            if i < len(ids) and ids[i] < n_pages:
                s = ids[i] * page + p % page
            pos.append(p), slots.append(s)
    lost = missing + sum(1 for t, s in enumerate(slots) if s == NONE or t >= max_tokens)
    pad = max(0, max_tokens - len(pos))
    pos, slots = (pos + [0] * pad)[:max_tokens], (slots + [NONE] * pad)[:max_tokens]
    return out, left + back, q_off, pos, slots, lost


def dealt(n_keys, n_new, blocks, page, window, sinks):
    """(table, q_off) of sequences that hold the blocks of a step, pages in order: as after
    the steps before it, each key new in one of them."""
    table = np.full((len(n_keys), blocks), NONE, np.uint32)
    ids = iter(range(table.size))
    for b, (n, m) in enumerate(zip(n_keys, n_new)):
        for i in range(blocks):
            first = max(0, n - m - window + 1)
            if i * page < n and (not window or (i + 1) * page > first or i * page < sinks):
                table[b, i] = next(ids)
    return table, np.concatenate([[0], np.cumsum(n_new)]).astype(int).tolist()


def attention(q, k, v, n_keys, window=0, sinks=0):
    """64-bit attention of q [m][H][D], the last m of n_keys positions, over k, v
    [n_keys][G][D]. Rows that see nothing are zeros."""
    m, H, D = q.shape
    G = k.shape[1]
    o = np.zeros((m, H, D))
    k, v, q = k.astype(np.float64), v.astype(np.float64), q.astype(np.float64)
    j = np.arange(n_keys)
    for i in range(m):
        p = n_keys - m + i
        seen = j <= p
        if window:
            seen &= (j > p - window) | (j < sinks)
        if not seen.any():
            continue
        for h in range(H):
            g = h // (H // G)
            with np.errstate(invalid="ignore", over="ignore"):
                s = k[seen, g] @ q[i, h] / math.sqrt(D)
                w = np.exp(s - s.max())
                o[i, h] = w @ v[seen, g] / w.sum()
    return o
