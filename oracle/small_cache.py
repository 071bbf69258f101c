"""Oracles of the operators that keep a paged cache small, in float64: attention
with a window and sinks, the 4-bit records, accumulated attention weight and
the choice of what to keep.  Written from the formulas, one query at a time."""

from __future__ import annotations

import numpy as np


def row_tokens(cache, indices, lo, hi, last):
    """K, V [tokens, Hkv, D] of a row's pages cache[P, 2, ps, Hkv, D]."""

    if hi <= lo:
        return cache[:0, 0].reshape(0, *cache.shape[3:]), cache[:0, 1].reshape(0, *cache.shape[3:])
    pages = cache[indices[lo:hi]]
    n = (hi - lo - 1) * cache.shape[2] + last
    return (pages[:, i].reshape(-1, *cache.shape[3:])[:n] for i in (0, 1))


def visible(p, n, window, sinks):
    """Which of the n positions a query at position p sees; window None: all up to p."""

    j = np.arange(n)
    see = j <= p
    return see if window is None else see & ((j > p - window) | (j < sinks))


def attend(q, k, v, see, scale):
    """One query token q [Hq, D]: (o [Hq, D], lse [Hq], p [Hq, n], spread [Hq, D] = sum p |v|)."""

    hq, d = q.shape
    group = hq // k.shape[1]
    o, spread = np.zeros((hq, d)), np.zeros((hq, d))
    lse, p = np.full(hq, -np.inf), np.zeros((hq, len(k)))
    at = np.flatnonzero(see)
    if len(at) == 0:
        return o, lse, p, spread
    for h in range(hq):
        s = k[at, h // group].astype(np.float64) @ q[h].astype(np.float64) * scale
        m = s.max()
        e = np.exp(s - m)
        lse[h] = m + np.log(e.sum())
        w = e / e.sum()
        p[h, at] = w
        o[h] = w @ v[at, h // group].astype(np.float64)
        spread[h] = w @ np.abs(v[at, h // group].astype(np.float64))
    return o, lse, p, spread


def paged(q, cache, qo_indptr, indptr, indices, last, scale, window=None, sinks=0):
    """Ragged causal attention: (o, lse, weight list per row, spread)."""

    o, spread = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    weight = []
    for b in range(len(last)):
        k, v = row_tokens(cache, indices, indptr[b], indptr[b + 1], last[b])
        n, q0, q1 = len(k), qo_indptr[b], qo_indptr[b + 1]
        w = np.zeros(n)
        for i in range(q0, q1):
            pos = n - (q1 - i)
            o[i], lse[i], p, spread[i] = attend(q[i], k, v, visible(pos, n, window, sinks), scale)
            w += p.sum(0)
        weight.append(w)
    return o, lse, weight, spread


def to_bf16(x):
    """fp32 rounded to the nearest bf16, as fp32 (finite values)."""

    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def pack4(x):
    """4-bit records of x [..., d] (bf16 values): (codes [..., d] int, scale, minimum [..., 4])."""

    half = np.asarray(x, np.float32) * np.float32(0.5)
    grp = half.reshape(*half.shape[:-1], half.shape[-1] // 4, 4)
    lo, hi = grp.min(-2), grp.max(-2)
    scale = to_bf16((hi - lo) / np.float32(7.5))
    scale = np.where(scale >= 2.0 ** -120, scale, 0).astype(np.float32)
    step = np.where(scale > 0, np.float32(0.5) * scale, np.float32(np.inf))
    code = np.clip(np.rint((grp - lo[..., None, :]) / step[..., None, :]), 0, 15)
    return code.reshape(half.shape).astype(np.int64), scale, lo * np.float32(2)


def record_bytes(code, scale, low):
    """The records' bytes [..., d / 2 + 16]."""

    b = (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)
    tail = np.concatenate([scale, low], -1).astype(np.float32)
    half = (np.ascontiguousarray(tail).view(np.uint32) >> 16).astype(np.uint16)
    return np.concatenate([b, np.ascontiguousarray(half).view(np.uint8).reshape(*half.shape[:-1], 16)], -1)


def unpack4(rec):
    """(values [..., d] float64, scale and code - 8 of every channel) of records."""

    half = rec.shape[-1] - 16
    code = np.stack([rec[..., :half] & 15, rec[..., :half] >> 4], -1).reshape(*rec.shape[:-1], 2 * half).astype(np.int64)
    tail = np.ascontiguousarray(rec[..., half:]).view(np.uint16).astype(np.uint32) << 16
    tail = tail.view(np.float32).astype(np.float64)
    grp = np.arange(2 * half) % 4
    scale, low = tail[..., grp], tail[..., 4 + grp]
    return low + scale * code, scale, code - 8


def select(weight, length, budget, sinks, recent):
    """Positions that a row keeps, ascending."""

    if length <= budget:
        return np.arange(length)
    mid = np.arange(sinks, length - recent)
    w = np.asarray(weight, np.float64)[mid]
    order = np.lexsort((mid, -np.where(np.isnan(w), 0, w), ~np.isnan(w)))  # NaN first, then falling, then position
    kept = mid[order[: budget - sinks - recent]]
    return np.sort(np.concatenate([np.arange(sinks), kept, np.arange(length - recent, length)]))
