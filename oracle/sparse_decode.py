"""Page-selected decode: key bounds, integer scores, selection, attention in 64 bits."""

from __future__ import annotations

import math

import numpy as np

INV127 = np.float32(1.0) / np.float32(127.0)


def page_bounds(k: np.ndarray) -> tuple[np.ndarray, np.float32]:
    """k [tokens, D] (bf16 values) of one page and kv head: (int8 [2, D], scale)."""

    d = k.shape[1]
    k = k.astype(np.float32)
    if not np.isfinite(k).all():
        return np.zeros((2, d), np.int8), np.float32(np.inf)
    a = np.float32(np.abs(k).max()) if len(k) else np.float32(0)
    s = np.float32(a * INV127)
    if not s > 0:
        return np.zeros((2, d), np.int8), s
    lo = np.clip(np.floor(k.min(0) / s), -127, 127)
    hi = np.clip(np.ceil(k.max(0) / s), -127, 127)
    return np.stack([lo, hi]).astype(np.int8), s


def select(q: np.ndarray, bounds: np.ndarray, scale: np.ndarray, num_select: int, sink: int, recent: int) -> np.ndarray:
    """q [group, D]; bounds int8 [pages, 2, D], scale [pages] of one row and kv head."""

    n = len(scale)
    if n <= num_select:
        return np.arange(n)
    q = q.astype(np.float32)
    sq = np.float32(np.abs(q).max()) * INV127
    qi = np.clip(np.rint(q / (sq if sq > 0 else np.float32(1))), -127, 127).astype(np.int64)
    b = bounds.astype(np.int64)
    best = []
    for p in range(sink, n - recent):
        if np.isinf(scale[p]):
            score = np.inf
        else:
            dot = max(int(np.maximum(h * b[p, 0], h * b[p, 1]).sum()) for h in qi)
            score = float(np.float32(dot) * np.float32(scale[p]))
        best.append((-score, p))
    top = [p for _, p in sorted(best)[: num_select - sink - recent]]
    return np.array(sorted(list(range(sink)) + top + list(range(n - recent, n))))


def sparse_decode(q, cache, indptr, indices, last, bounds, scale, *, num_select, sink, recent, sm_scale=None):
    """(out, lse, spread, selected): q [B, Hq, D], cache [P, 2, PS, Hkv, D], bounds
    int8 [P, Hkv, 2, D], scale [P, Hkv]; selected int32 [B, Hkv, num_select]."""

    batch, hq, d = q.shape
    ps, hkv = cache.shape[2], cache.shape[3]
    g = hq // hkv
    f = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    out, spread = np.zeros((batch, hq, d)), np.zeros((batch, hq, d))
    lse = np.full((batch, hq), -np.inf)
    chosen = np.full((batch, hkv, num_select), -1, np.int32)
    for b in range(batch):
        pages = np.asarray(indices[indptr[b]:indptr[b + 1]], dtype=np.int64)
        for h in range(hkv):
            sel = select(q[b, h * g:(h + 1) * g], bounds[pages, h], scale[pages, h], num_select, sink, recent)
            chosen[b, h, : len(sel)] = sel
            pos = [(p, t) for p in sel for t in range(last[b] if p == len(pages) - 1 else ps)]
            if not pos:
                continue
            pg, off = pages[[p for p, _ in pos]], np.array([t for _, t in pos])
            k, v = cache[pg, 0, off, h].astype(np.float64), cache[pg, 1, off, h].astype(np.float64)
            for m in range(g):
                s = (k @ q[b, h * g + m].astype(np.float64)) * f
                mx = s.max()
                p = np.exp(s - mx)
                lse[b, h * g + m] = mx + np.log(p.sum())
                p /= p.sum()
                out[b, h * g + m], spread[b, h * g + m] = p @ v, p @ np.abs(v)
    return out, lse, spread, chosen
