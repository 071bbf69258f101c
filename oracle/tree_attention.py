"""Drafted-token trees in 64 bits: ancestor mask, greedy acceptance, attention.

One token at a time from the definitions; no shortcut is shared with the
kernels.  ``parents`` holds indices in the request, -1 for the context.
"""

from __future__ import annotations

import math

import numpy as np


def ancestors(parents) -> np.ndarray:
    """Ancestor-or-self matrix [n, n] of one request."""

    n = len(parents)
    m = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            m[i, j] = True
            j = int(parents[j])
    return m


def pack_bits(m: np.ndarray, words: int) -> np.ndarray:
    """Rows of a 0/1 matrix as int32 words, bit j % 32 of word j / 32."""

    out = np.zeros((m.shape[0], words), np.uint32)
    for i, j in zip(*np.nonzero(m)):
        out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out.view(np.int32)


def accept(parents, tokens, targets) -> tuple[list[int], int]:
    """(indices of the kept path, the model's choice after it) of one request."""

    best, depth = -1, 0
    for i in range(len(parents)):
        path, j = [], i
        while j >= 0:
            path.append(j)
            j = int(parents[j])
        taken = all(parents[k] < 0 or tokens[k] == targets[parents[k]] for k in path)
        if taken and len(path) > depth:
            best, depth = i, len(path)
    if best < 0:
        return [], -1
    path, j = [], best
    while j >= 0:
        path.append(j)
        j = int(parents[j])
    return path[::-1], int(targets[best])


def tree_attention(q, cache, qo_indptr, kv_indptr, kv_indices, last, see, sm_scale=None):
    """q [total, Hq, D], cache [P, 2, PS, Hkv, D] (float64 values of the bf16
    inputs); see[b] bool [n_b, n_b].  Returns (out, lse, spread) in float64;
    spread = sum p |v|, the scale of the output's rounding."""

    total, hq, d = q.shape
    ps, hkv = cache.shape[2], cache.shape[3]
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    out = np.zeros((total, hq, d))
    spread = np.zeros((total, hq, d))
    lse = np.full((total, hq), -np.inf)
    for b in range(len(last)):
        q0, q1 = qo_indptr[b], qo_indptr[b + 1]
        pages = kv_indices[kv_indptr[b]:kv_indptr[b + 1]]
        n_kv = (len(pages) - 1) * ps + last[b] if len(pages) else 0
        ctx = n_kv - (q1 - q0)
        for i in range(q1 - q0):
            pos = list(range(max(ctx, 0))) + [ctx + j for j in range(q1 - q0) if see[b][i, j] and ctx + j >= 0]
            if not pos:
                continue
            pg = np.array([pages[t // ps] for t in pos])
            off = np.array([t % ps for t in pos])
            for h in range(hq):
                k, v = cache[pg, 0, off, h // g], cache[pg, 1, off, h // g]
                s = (k @ q[q0 + i, h]) * scale
                m = s.max()
                p = np.exp(s - m)
                lse[q0 + i, h] = m + np.log(p.sum())
                p /= p.sum()
                with np.errstate(invalid="ignore"):
                    out[q0 + i, h] = p @ v
                    spread[q0 + i, h] = p @ np.abs(v)
    return out, lse, spread
