"""Plain 64-bit statements of the 4-bit cache, its attention, its page
operations and sampling, for the tests: numpy, written from the definitions."""
from __future__ import annotations

import numpy as np

BLOCK = 16


def block_bytes(D):
    return BLOCK * (D + 8)


def decode(pages, page_size, kv_heads, D):
    """K, V float64 [pages, heads, tokens, D] of a pool's bytes (numpy uint8)."""
    n = pages.shape[0]
    blocks = pages.reshape(n, kv_heads, page_size // BLOCK, block_bytes(D))
    d = np.arange(D)
    r = np.arange(BLOCK)[:, None]
    k_byte, k_nib = r * (D // 2) + d // 2, np.broadcast_to(d % 2, (BLOCK, D))
    e = d % (D // 8)
    v_byte = 8 * D + (r // 8) * 4 * D + d // (D // 8) * (D // 2) + r % 8 // 2 * (D // 8) + \
        e // 4 * 4 + 2 * (r % 2) + e % 4 // 2
    out = []
    for byte, nib, par in ((k_byte, k_nib, 16 * D), (v_byte, np.broadcast_to(e % 2, (BLOCK, D)),
                                                     16 * D + 64)):
        code = (blocks[..., byte] >> (4 * nib).astype(np.uint8)) & 15
        sb = np.ascontiguousarray(blocks[..., par:par + 64]).view(np.float16).astype(np.float64)
        sb = sb.reshape(n, kv_heads, -1, BLOCK, 2)
        x = sb[..., 1:] + sb[..., :1] * (code.astype(np.float64) - 8)
        out.append(x.reshape(n, kv_heads, page_size, D))
    return out


def quantised(x):
    """What the cache holds of fp16/bf16 vectors (float64 in, float64 out)."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        bad = ~np.isfinite(x).all(-1, keepdims=True)
        x = np.clip(np.where(np.isnan(x), 0, x), -65504, 65504).astype(np.float32)
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        scale = ((hi - lo) / np.float32(15)).astype(np.float16)
        s = scale.astype(np.float32)
        base = (lo + np.float32(8) * s).astype(np.float16)
        code = np.clip(np.rint((x - base.astype(np.float32)) / s) + 8, 0, 15)
        code = np.where(s > 0, code, 8)
    got = base.astype(np.float64) + s.astype(np.float64) * (code - 8)
    return np.where(bad, np.nan, got)


def attention(q, K, V, table, lens, page_size, rows_of, scale):
    """O, LSE, and the largest |V| that each row sees. q [S,H,R,D] float64; K, V
    decoded pools; rows_of: new tokens of each slot."""
    S, H, R, D = q.shape
    kvh, pages = K.shape[1], K.shape[0]
    O, L, M = np.zeros((S, H, R, D)), np.full((S, H, R), -np.inf), np.zeros((S, H, R))
    for s in range(S):
        n = min(int(lens[s]), table.shape[1] * page_size)
        at = np.arange(n)
        page = table[s][at // page_size] if n else at
        ok = (page >= 0) & (page < pages)
        page = np.where(ok, page, 0)
        for i in range(min(int(rows_of[s]), R)):
            end = int(lens[s]) - int(rows_of[s]) + i + 1
            see = ok & (at < end)
            if not see.any():
                continue
            for h in range(H):
                kh = h // (H // kvh)
                k, v = K[page[see], kh, at[see] % page_size], V[page[see], kh, at[see] % page_size]
                x = k @ q[s, h, i] * scale
                top = x.max()
                p = np.exp(x - top)
                O[s, h, i] = p @ v / p.sum()
                L[s, h, i] = top + np.log(p.sum())
                M[s, h, i] = np.abs(v).max()
    return O, L, M


# ------------------------------------------------------------ page operations
def pages_for(n, page):
    return (max(int(n), 0) + page - 1) // page


def reserve(table, lens, refs, counts, page):
    free = [p for p in range(len(refs)) if refs[p] <= 0]
    need, past = [], 0
    for n, c in zip(lens, counts):
        now, then = pages_for(n, page), pages_for(max(n, 0) + max(c, 0), page)
        over = max(then - max(now, table.shape[1]), 0)
        past += over
        need.append(then - now - over)
    missing = max(sum(need) - len(free), 0) + past
    table, lens, refs = table.copy(), lens.copy(), refs.copy()
    if missing:
        return table, lens, refs, [missing, 0]
    for s, k in enumerate(need):
        now = pages_for(lens[s], page)
        for j in range(k):
            p = free.pop(0)
            table[s, now + j], refs[p] = p, 1
        lens[s] = max(lens[s], 0) + max(counts[s], 0)
    return table, lens, refs, [0, 0]


def fork(pool, table, lens, refs, parents, children, page):
    S = len(lens)
    old = lens.copy()
    named, pairs, skipped = set(), [], 0
    for p, c in zip(parents, children):
        first = c not in named
        if 0 <= c < S:
            named.add(c)
        if 0 <= p < S and 0 <= c < S and p != c and old[c] <= 0 and first:
            pairs.append((p, c))
        else:
            skipped += 1
    free = [p for p in range(len(refs)) if refs[p] <= 0]
    need = sum(1 for p, _ in pairs if old[p] % page)
    t, n, r, pool = table.copy(), lens.copy(), refs.copy(), pool.copy()
    if need > len(free):
        return pool, t, n, r, [need - len(free), skipped]
    for p, c in pairs:
        whole = max(old[p], 0) // page
        t[c] = -1
        t[c, :whole] = table[p, :whole]
        for x in table[p, :whole]:
            r[x] += 1
        if max(old[p], 0) % page:
            x = free.pop(0)
            t[c, whole], r[x] = x, 1
            pool[x] = pool[table[p, whole]]
        n[c] = max(old[p], 0)
    return pool, t, n, r, [0, skipped]


def free(table, lens, refs, slots, page):
    table, lens, refs = table.copy(), lens.copy(), refs.copy()
    for s in sorted({int(s) for s in slots if 0 <= s < len(lens)}):
        for x in table[s, :pages_for(lens[s], page)]:
            refs[x] -= 1
        table[s], lens[s] = -1, 0
    return table, lens, refs


def compact(pool, table, refs):
    live = int((refs > 0).sum())
    src = [p for p in range(live, len(refs)) if refs[p] > 0]
    dst = [p for p in range(live) if refs[p] <= 0]
    to = np.arange(len(refs))
    pool, r = pool.copy(), np.where(refs > 0, refs, 0)
    for a, b in zip(src, dst):
        to[a], pool[b], r[b], r[a] = b, pool[a], refs[a], 0
    t = np.where((table >= 0) & (table < len(refs)), to[np.clip(table, 0, len(refs) - 1)], -1)
    return pool, t.astype(table.dtype), r.astype(refs.dtype)


# --------------------------------------------------------------------- sampling
def kept(x, temp, top_k, top_p, min_p):
    """(order, how many of it are kept, weights) of a row in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / temp))
    order = np.argsort(-x, kind="stable")
    n = len(x) if top_k is None or top_k <= 0 else min(top_k, len(x))
    if top_p is not None and top_p < 1:
        upto = np.cumsum(w[order[:n]])
        n = max(1, int(np.sum(np.concatenate([[0.0], upto[:-1]]) < top_p * upto[-1])))
    if min_p is not None:
        n = max(1, min(n, int(np.sum(w[order] >= min_p))))
    return order, n, w
