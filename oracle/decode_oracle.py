"""float64 restatement of the operators around the delta, from their definitions (numpy; the checker only)."""
from __future__ import annotations

import numpy as np


def rotate(x, cos, sin, rotary_dim, interleaved):
    """``x [..., D]`` turned by the angles whose cosine and sine are given, ``[..., R/2]``."""
    y = np.array(x, np.float64)
    i = np.arange(rotary_dim // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
    a, b = y[..., first], y[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y


def append(q_out, q, k, v, k_cache, v_cache, positions, slots, cos, sin, dq=None, dk=None, dv=None, interleaved=False):
    """New ``(q_out, k_cache, v_cache)``; rows with a slot or position that does not exist change nothing."""
    q_out, k_cache, v_cache = (np.array(t, np.float64) for t in (q_out, k_cache, v_cache))
    pages, page = k_cache.shape[:2]
    rot = 2 * cos.shape[1]

    def plus(x, d, t):
        return x[t] + (0.0 if d is None else d[t])

    for t in range(q.shape[0]):
        s, pos = int(slots[t]), int(positions[t])
        if s < 0 or s >= pages * page or pos < 0 or pos >= cos.shape[0]:
            continue
        q_out[t] = rotate(plus(q, dq, t), cos[pos], sin[pos], rot, interleaved)
        k_cache[s // page, s % page] = rotate(plus(k, dk, t), cos[pos], sin[pos], rot, interleaved)
        v_cache[s // page, s % page] = plus(v, dv, t)
    return q_out, k_cache, v_cache


def keys_of(cache, table, n):
    """``[n, heads, D]``: the first n keys of the pages of a table row (pages that do not exist are left out)."""
    page = cache.shape[1]
    at = np.arange(n)
    pages = np.asarray(table)[at // page] if n else np.zeros(0, np.int64)
    fine = (pages >= 0) & (pages < cache.shape[0])
    return cache[pages[fine], (at % page)[fine]]


def attention(q, k_cache, v_cache, table, lens, prefix_table=None, prefix_lens=None, starts=None, scale=None):
    """``(out, lse, weighted)``: weighted is the softmax average of |v|, which bounds what errors of the weights do."""
    n_req, heads, d = q.shape
    kv = k_cache.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, weighted, lse = np.zeros(q.shape), np.zeros(q.shape), np.full((n_req, heads), -np.inf)
    group = np.full(n_req, -1)
    for g in range(0 if starts is None else len(starts) - 1):
        group[starts[g]:starts[g + 1]] = g
    for b in range(n_req):
        ks, vs = [keys_of(k_cache, table[b], int(lens[b]))], [keys_of(v_cache, table[b], int(lens[b]))]
        if group[b] >= 0:
            ks.insert(0, keys_of(k_cache, prefix_table[group[b]], int(prefix_lens[group[b]])))
            vs.insert(0, keys_of(v_cache, prefix_table[group[b]], int(prefix_lens[group[b]])))
        k, v = np.concatenate(ks), np.concatenate(vs)
        if not len(k):
            continue
        for h in range(heads):
            z = scale * (k[:, h // (heads // kv)] @ q[b, h])
            top = z.max()
            e = np.exp(z - top)
            lse[b, h] = top + np.log(e.sum())
            out[b, h] = e @ v[:, h // (heads // kv)] / e.sum()
            weighted[b, h] = e @ np.abs(v[:, h // (heads // kv)]) / e.sum()
    return out, lse, weighted


def int4_weights(codes, scales, zeros=None):
    """``W [N, K]`` of codes ``[N, K/2]``, scales and zeros ``[N, groups]``."""
    n, half = codes.shape
    w = np.empty((n, 2 * half))
    w[:, 0::2], w[:, 1::2] = codes & 15, codes >> 4
    group = 2 * half // scales.shape[1]
    zero = 8.0 if zeros is None else np.repeat(zeros & 15, group, axis=1).astype(np.float64)
    return (w - zero) * np.repeat(np.asarray(scales, np.float64), group, axis=1)
