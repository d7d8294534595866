"""Plain 64-bit forms of the paged-cache operators on the CPU, loop by loop, for the
GPU tests (no code of the library)."""
import numpy as np


def dequant(plane, page, dim):
    """A Q8_0 plane's bytes [page * (dim + dim / 16)] as its values [page, dim] in f64."""
    levels = plane[:page * dim].view(np.int8).reshape(page, dim // 32, 32).astype(np.float64)
    scales = plane[page * dim:].view(np.float16).reshape(page, dim // 32, 1).astype(np.float64)
    return (levels * scales).reshape(page, dim)


def values(cache, q8, page, dim):
    """A cache tensor (numpy; bf16 given as f32) as f64 [pages, kv_heads, page, dim]."""
    if not q8:
        return cache.astype(np.float64)
    return np.stack([np.stack([dequant(h, page, dim) for h in p]) for p in cache])


def attention(k, v, q, tables, positions, requests, scale, window, out):
    """k, v [pages, kv_heads, page, dim] f64; returns out and, for each value, the largest
    sum of |scale q k| over the tokens seen and the largest |v|."""
    out = out.astype(np.float64).copy()
    heads, dim = q.shape[1:]
    kv, page = k.shape[1], k.shape[2]
    spread, most = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for t in range(q.shape[0]):
        r = t if requests is None else requests[t]
        if r < 0:
            continue
        last = int(positions[t])
        first = max(0, last + 1 - window) if window else 0
        tok = np.arange(first, last + 1)
        for h in range(heads):
            g = h // (heads // kv)
            if not len(tok):
                out[t, h] = 0.0
                continue
            kk, vv = (c[tables[r, tok // page], g, tok % page] for c in (k, v))
            qh = q[t, h].astype(np.float64)
            s = kk @ qh * scale
            p = np.exp(s - s.max())
            out[t, h] = p @ vv / p.sum()
            spread[t, h] = (np.abs(kk) @ np.abs(qh)).max() * abs(scale)
            most[t, h] = np.abs(vv).max()
    return out, spread, most


def pages(before, more, tables, owned, free, count, page, tokens):
    """rlq_kv_pages; tables, owned (None: tables) and free are changed."""
    own = tables if owned is None else owned
    n = int(count[0])
    stack = [int(p) for p in free[:n]]
    for r in np.flatnonzero(more < 0):
        for c in range(-(-int(before[r]) // page)):
            if own[r, c] >= 0:
                stack.append(int(own[r, c]))
                own[r, c] = -1
    free[n:len(stack)] = stack[n:]
    after, starts = [], [0]
    slots, positions, requests = (np.full(tokens, -1, t) for t in (np.int64, np.int32, np.int32))
    for r in range(len(before)):
        b, m = int(before[r]), max(int(more[r]), 0)
        end = 0 if more[r] < 0 else b + m
        for c in range(-(-b // page), -(-end // page)):
            p = stack.pop()
            tables[r, c] = own[r, c] = p
        for i in range(m):
            t, pos = starts[-1] + i, b + i
            p = int(tables[r, pos // page])
            slots[t], positions[t], requests[t] = -2 if p < 0 else p * page + pos % page, pos, r
        after.append(end)
        starts.append(starts[-1] + m)
    return (np.array(after, np.int32), np.array([len(stack)], np.int32), np.array(starts, np.int32), slots, positions,
            requests)


def rotate(x, positions, freqs, pairs):
    """[tokens, heads, dim] f32, rotated in f64 and rounded once to f32."""
    y = x.astype(np.float64)
    half = len(freqs)
    a = positions.astype(np.float64)[:, None] * freqs.astype(np.float64)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    u, w = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = u * c - w * s, u * s + w * c
    return y.astype(np.float32)


def q8_0(x):
    """Levels int8 [.., dim] and scales f16 [.., dim / 32] of f32 rows."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = (np.abs(b).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
    inv = np.where(d != 0, np.float32(1) / np.where(d != 0, d, 1), 0).astype(np.float32)
    r = (b * inv).astype(np.float32).astype(np.float64)
    q = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -128, 127)
    return q.astype(np.int8).reshape(x.shape), d[..., 0].astype(np.float16)


def select(z, scores, best):
    """Scores (f64), parents, tokens [groups, best]."""
    groups, beams, vocabulary = z.shape
    out = np.full((groups, best), -np.inf), np.full((groups, best), -1), np.full((groups, best), -1)
    for g in range(groups):
        rank = np.full((beams, vocabulary), -np.inf)
        for b in range(beams):
            if scores[g, b] > -np.inf and z[g, b].max() > -np.inf:
                r = z[g, b].astype(np.float64)
                rank[b] = np.float64(scores[g, b]) + r - (r.max() + np.log(np.exp(r - r.max()).sum()))
        order = np.argsort(-rank.reshape(-1), kind="stable")[:best]
        for i, at in enumerate(order):
            if rank.reshape(-1)[at] > -np.inf:
                out[0][g, i], out[1][g, i], out[2][g, i] = rank.reshape(-1)[at], at // vocabulary, at % vocabulary
    return out
