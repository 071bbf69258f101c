"""Attention with a sliding window and sinks against the oracle
(oracle/small_cache.py).

Tolerance: P and the result are rounded to bf16 (half a step is 2^-8
relative), scores and sums are fp32: |err| <= 2^-8 (|o| + sum p |v|) + 2^-12
sum p |v|; LSE within 2^-12 (1 + |lse|).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import small_cache as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
F = 2.0 ** -12


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64).reshape(-1), dtype=torch.int32, device="cuda")


def _case(lens, n, hq, hkv, d, ps, seed, edit=None):
    """Rows of lens positions, the last n[b] of them with queries; unused slots hold NaN."""

    rng = np.random.default_rng(seed)
    pages = [-(-x // ps) for x in lens]
    pool = sum(pages) + 4
    perm = rng.permutation(pool)
    cache = rng.normal(size=(pool, 2, ps, hkv, d)).astype(np.float32) * rng.choice([0.5, 1, 3], size=(hkv, d))
    indptr = np.cumsum([0] + pages)
    last = [x - (k - 1) * ps if k else 0 for x, k in zip(lens, pages)]
    indices = perm[: sum(pages)].copy()
    for b, k in enumerate(pages):
        if k:
            cache[indices[indptr[b + 1] - 1], :, last[b]:] = np.nan
    qo = np.cumsum([0] + list(n))
    q = rng.normal(size=(qo[-1], hq, d)).astype(np.float32)
    if edit is not None:
        edit(q, cache, indptr, indices, lens)
    ct = torch.as_tensor(cache).to(torch.bfloat16)
    qt = torch.as_tensor(q).to(torch.bfloat16)
    host = dict(q=qt.float().numpy(), cache=ct.float().numpy(), qo=qo, indptr=indptr, indices=indices, last=last)
    dev = dict(q=qt.cuda(), cache=ct.cuda(), qo=_i32(qo), indptr=_i32(indptr), indices=_i32(indices), last=_i32(last))
    return host, dev


def _check(out, lse, host, window, sinks, scale, finite=True):
    want, wlse, _, spread = o.paged(host["q"], host["cache"], host["qo"], host["indptr"], host["indices"], host["last"],
                                    scale, window, sinks)
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    ok = np.isfinite(want)
    if finite:
        assert ok.all()
    assert (np.isnan(out) == np.isnan(want)).all() and (np.isinf(out) == np.isinf(want)).all()
    err = np.abs(np.where(ok, out, 0) - np.where(ok, want, 0))
    sp = np.where(ok, spread, 0)
    assert (err <= U * (np.abs(np.where(ok, want, 0)) + sp) + F * sp + 1e-30).all(), err.max()
    empty = np.isneginf(wlse)
    assert (np.isneginf(lse) == empty).all()
    a, b = np.where(empty, 0, lse), np.where(empty, 0, wlse)
    assert (np.abs(a - b) <= F * (1 + np.abs(b))).all()


def _decode(K, dev, window, sinks, want=0, **kw):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full(dev["q"].shape[:2], 7.0, device="cuda")
    out = K.paged_window_decode(dev["q"], dev["cache"], dev["indptr"], dev["indices"], dev["last"], window=window,
                                sinks=sinks, out_lse=lse, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == want
    return out, lse


def _prefill(K, dev, window, sinks, want=0, **kw):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full(dev["q"].shape[:2], 7.0, device="cuda")
    out = K.paged_window_prefill(dev["q"], dev["cache"], dev["qo"], dev["indptr"], dev["indices"], dev["last"],
                                 window=window, sinks=sinks, out_lse=lse, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == want
    return out, lse


LENS = [1, 16, 17, 0, 300, 2000, 161, 700]
HEADS = [(32, 8, 128, 16), (8, 8, 64, 32), (28, 4, 128, 64), (16, 1, 64, 128), (10, 5, 128, 16), (9, 1, 128, 32)]


@pytest.mark.parametrize("hq,hkv,d,ps", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (129, 0), (250, 17), (5000, 3), (40, 9999)])
def test_decode(K, hq, hkv, d, ps, window, sinks):
    host, dev = _case(LENS, [1] * len(LENS), hq, hkv, d, ps, hq + window)
    _check(*_decode(K, dev, window, sinks), host, window, sinks, d ** -0.5)


def test_decode_rows_beyond_a_block_and_long_rows(K):
    rng = np.random.default_rng(3)
    lens = list(rng.integers(0, 60, 400))
    lens[7], lens[399] = 9000, 4097
    host, dev = _case(lens, [1] * 400, 4, 2, 64, 16, 5)
    _check(*_decode(K, dev, 4000, 2), host, 4000, 2, 64 ** -0.5)


def test_decode_does_not_look_at_hidden_pages(K):
    """Pages in front of the window may have been given away: any id, any content."""

    def edit(q, cache, indptr, indices, lens):
        for b, n in enumerate(lens):
            first = max(0, n - 100) // 16
            indices[indptr[b] + 1: indptr[b] + first] = -7

    host, dev = _case([500, 1999, 160, 90], [1] * 4, 8, 2, 128, 16, 9, edit)
    out, lse = _decode(K, dev, 100, 5)
    host["indices"] = np.where(host["indices"] < 0, 0, host["indices"])
    _check(out, lse, host, 100, 5, 128 ** -0.5)


def test_hidden_nan_and_inf_stay_out(K):
    """inf and NaN at positions that a query does not see, in pages that it reads."""

    def edit(q, cache, indptr, indices, lens):
        for b, n in enumerate(lens):
            for pos in range(3, n - 37):
                cache[indices[indptr[b] + pos // 16], :, pos % 16] = np.nan if pos % 2 else np.inf

    host, dev = _case([200, 45, 333], [1] * 3, 8, 2, 128, 16, 11, edit)
    _check(*_decode(K, dev, 37, 3), host, 37, 3, 128 ** -0.5)
    host, dev = _case([200, 45, 333], [1, 1, 1], 8, 2, 128, 16, 11, edit)
    _check(*_prefill(K, dev, 37, 3), host, 37, 3, 128 ** -0.5)


def test_seen_nan_reaches_the_row(K):
    def edit(q, cache, indptr, indices, lens):
        cache[indices[indptr[1] + 2], 1, 5, 0, 7] = np.nan
        q[2, 3] = np.nan

    host, dev = _case([100, 100, 100], [1] * 3, 8, 2, 64, 16, 12, edit)
    out, lse = _decode(K, dev, 99, 0)
    nan = torch.isnan(out).cpu()
    want = torch.zeros_like(nan)
    want[1, :4, 7] = True
    want[2, 3] = True
    assert torch.equal(nan, want)


def test_scores_of_any_size(K):
    """Scores of thousands, rising and falling along the row: the reference moves often."""

    def edit(q, cache, indptr, indices, lens):
        q *= 40
        for b, n in enumerate(lens):
            for pos in range(n):
                cache[indices[indptr[b] + pos // 16], 0, pos % 16] *= 1 + (pos if b else n - pos) / 20

    host, dev = _case([400, 700], [1, 1], 8, 8, 128, 16, 13, edit)
    _check(*_decode(K, dev, 650, 20), host, 650, 20, 128 ** -0.5)


def test_decode_strides_streams_and_graphs(K):
    host, dev = _case([900, 33, 0, 2048], [1] * 4, 8, 2, 128, 16, 14)
    want, wlse = _decode(K, dev, 300, 4)
    wide = torch.empty(4, 3, 8, 192, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 1, :, 32:160]
    q.copy_(dev["q"])
    out = torch.full((4, 8, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((K._window_decode_workspace_bytes(8, 2, 128),), 255, dtype=torch.uint8, device="cuda")
    args = (q, dev["cache"], dev["indptr"], dev["indices"], dev["last"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.paged_window_decode(*args, window=300, sinks=4, out=out[:, :, 64:192], workspace=ws)
    side.synchronize()
    assert torch.equal(out[:, :, 64:192], want) and (out[:, :, :64] == 5).all() and (out[:, :, 192:] == 5).all()
    # two captured graphs with one workspace, replayed in turn
    got, lse = torch.empty_like(want), torch.empty_like(wlse)
    other = torch.empty_like(want)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        K.paged_window_decode(*args, window=300, sinks=4, out=got, out_lse=lse, workspace=ws)
    with torch.cuda.graph(g2):
        K.paged_window_decode(*args, window=77, sinks=0, out=other, workspace=ws)
    for _ in range(3):
        got.zero_()
        g2.replay()
        g1.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, wlse)
    assert torch.equal(other, _decode(K, dev, 77, 0)[0])


def test_decode_status(K):
    host, dev = _case([100, 100], [1, 1], 4, 2, 64, 16, 15)
    bad = dict(dev, indices=dev["indices"].clone())
    bad["indices"][3] = 10 ** 6
    out, _ = _decode(K, bad, 1000, 0, want=3)
    assert torch.equal(out[1], _decode(K, dev, 1000, 0)[0][1])
    bad = dict(dev, indptr=_i32([0, 7, 99]))
    out, lse = _decode(K, bad, 1000, 0, want=1)
    assert torch.equal(out[0], _decode(K, dev, 1000, 0)[0][0])
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()


@pytest.mark.parametrize("hq,hkv,d,ps", HEADS[:5])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 4), (128, 128), (300, 150), (5000, 3)])
def test_prefill(K, hq, hkv, d, ps, window, sinks):
    n = [1, 16, 5, 0, 300, 130, 161, 64]
    lens = [1, 16, 17, 40, 300, 900, 161, 700]
    host, dev = _case(lens, n, hq, hkv, d, ps, hq + window)
    _check(*_prefill(K, dev, window, sinks), host, window, sinks, d ** -0.5)


def test_prefill_of_a_wide_window_is_the_causal_prefill(K):
    host, dev = _case([700, 129, 64], [500, 129, 1], 8, 2, 128, 16, 21)
    out, lse = _prefill(K, dev, 2 ** 31 - 1, 0)
    want = K.paged_prefill(dev["q"], dev["cache"], dev["qo"], dev["indptr"], dev["indices"], dev["last"])
    assert torch.equal(out, want)


def test_prefill_does_not_look_at_hidden_pages(K):
    def edit(q, cache, indptr, indices, lens):
        for b, n in enumerate(lens):
            first = max(0, n - 60 - 100 + 1) // 16  # window of the first of 60 queries
            indices[indptr[b] + 1: indptr[b] + first] = -7

    host, dev = _case([500, 1999, 160], [60, 60, 60], 8, 2, 128, 16, 22, edit)
    out, lse = _prefill(K, dev, 100, 5)
    host["indices"] = np.where(host["indices"] < 0, 0, host["indices"])
    _check(out, lse, host, 100, 5, 128 ** -0.5)


def test_prefill_rows_meet_only_what_they_see(K):
    """inf and NaN values of single tokens: exactly the rows that see them have them."""

    def edit(q, cache, indptr, indices, lens):
        for pos, kv, val in ((150, 1, np.nan), (171, 1, np.inf), (199, 1, np.nan), (20, 1, np.nan), (240, 0, np.nan)):
            cache[indices[pos // 16], kv, pos % 16, :, 3::7] = val

    host, dev = _case([260], [130], 8, 2, 128, 16, 23, edit)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = K.paged_window_prefill(dev["q"], dev["cache"], dev["qo"], dev["indptr"], dev["indices"], dev["last"],
                                 window=40, sinks=2, status=status)
    want, _, _, spread = o.paged(host["q"], host["cache"], host["qo"], host["indptr"], host["indices"], host["last"],
                                 128 ** -0.5, 40, 2)
    got = out.double().cpu().numpy()
    # a key of NaN makes all of a row that sees it NaN
    assert (np.isfinite(got) == np.isfinite(want)).all()
    ok = np.isfinite(want)
    err = np.abs(np.where(ok, got - np.where(ok, want, 0), 0))
    sp = np.where(np.isfinite(spread), spread, 0)
    assert (err <= U * (np.abs(np.where(ok, want, 0)) + sp) + F * sp).all()


def test_calls_without_entries(K):
    kv = torch.zeros(3, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    K.paged_window_decode(none, kv, _i32([0]), e, e, window=3)
    K.paged_window_prefill(none, kv, _i32([0]), _i32([0]), e, e, window=3)
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(2, 4, device="cuda")
    assert (K.paged_window_decode(q, kv, _i32([0, 0, 0]), e, _i32([0, 0]), window=3, out_lse=lse) == 0).all()
    assert torch.isneginf(lse).all()
    lse.zero_()
    assert (K.paged_window_prefill(q, kv, _i32([0, 1, 2]), _i32([0, 0, 0]), e, _i32([0, 0]), window=3,
                                   out_lse=lse) == 0).all()
    assert torch.isneginf(lse).all()
