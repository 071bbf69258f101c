"""Key bounds, page selection and sparse decode against the oracle
(oracle/sparse_decode.py).

Bounds, scales and selected pages are equal (integers and single fp32
operations).  Attention tolerance as for the tree attention: |err| <=
2^-8 (|o| + sum p |v|) + 2^-12 sum p |v| for P and the result in bf16 and
fp32 scores; LSE within 2^-12 (1 + |lse|).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sparse_decode as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
F = 2.0 ** -12


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64).reshape(-1), dtype=torch.int32, device="cuda")


def _case(K, lens, hq, hkv, d, ps, seed, edit=None):
    rng = np.random.default_rng(seed)
    n = [-(-x // ps) for x in lens]
    pool = sum(n) + 4
    perm = rng.permutation(pool)
    cache = rng.normal(size=(pool, 2, ps, hkv, d)).astype(np.float32) * rng.choice([0.5, 1, 3], size=(hkv, d))
    indptr = np.cumsum([0] + n)
    last = [x - (k - 1) * ps if k else 0 for x, k in zip(lens, n)]
    indices = perm[: sum(n)]
    if edit is not None:
        edit(cache, indptr, indices)
    for b, k in enumerate(n):  # slots past the last token are never read
        if k:
            cache[indices[indptr[b + 1] - 1], :, last[b]:] = np.nan
    ct = torch.as_tensor(cache).to(torch.bfloat16)
    qt = torch.as_tensor(rng.normal(size=(len(lens), hq, d)).astype(np.float32)).to(torch.bfloat16)
    bounds = torch.full((pool, hkv, 2, d), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((pool, hkv), float("nan"), device="cuda")
    full = np.concatenate([indices[indptr[b]: indptr[b + 1] - 1] for b in range(len(lens))] or [[]]).astype(np.int64)
    dev = dict(q=qt.cuda(), cache=ct.cuda(), indptr=_i32(indptr), indices=_i32(indices if len(indices) else [0]),
               last=_i32(last), bounds=bounds, scale=scale)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.page_bounds(dev["cache"], _i32(full), bounds, scale, status=status)
    assert int(status.item()) == 0
    host = dict(q=qt.float().numpy(), cache=ct.float().numpy(), indptr=indptr, indices=indices, last=last,
                bounds=bounds.cpu().numpy(), scale=scale.cpu().numpy())
    return host, dev


def _run(K, dev, select, sink, recent, want=0, **kw):
    b, hq, _ = dev["q"].shape
    hkv = dev["cache"].shape[3]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full((b, hq), 7.0, device="cuda")
    sel = torch.full((b, hkv, select), -9, dtype=torch.int32, device="cuda")
    out = K.paged_sparse_decode(dev["q"], dev["cache"], dev["indptr"], dev["indices"], dev["last"], dev["bounds"],
                                dev["scale"], num_select=select, sink_pages=sink, recent_pages=recent, out_lse=lse,
                                selected=sel, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == want
    return out.double().cpu().numpy(), lse.double().cpu().numpy(), sel.cpu().numpy()


def _check(K, host, dev, select, sink, recent, **kw):
    out, lse, sel = _run(K, dev, select, sink, recent, **kw)
    want, wlse, spread, wsel = o.sparse_decode(host["q"], host["cache"], host["indptr"], host["indices"], host["last"],
                                               host["bounds"], host["scale"], num_select=select, sink=sink, recent=recent)
    assert (sel == wsel).all()
    err = np.abs(out - want)
    assert (err <= U * (np.abs(want) + spread) + F * spread + 1e-30).all(), err.max()
    empty = np.isinf(wlse)
    assert (np.isneginf(lse) == empty).all()
    d = np.where(empty, 0, lse) - np.where(empty, 0, wlse)
    assert (np.abs(d) <= F * (1 + np.abs(np.where(empty, 0, wlse)))).all(), np.abs(d).max()


@pytest.mark.parametrize("d,ps,hkv", [(128, 16, 8), (64, 32, 3), (128, 16, 1), (64, 16, 5), (128, 128, 2)])
def test_bounds(K, d, ps, hkv):
    rng = np.random.default_rng(d + ps + hkv)
    cache = rng.normal(size=(23, 2, ps, hkv, d)).astype(np.float32) * np.exp2(rng.integers(-30, 30, size=(23, 1, 1, 1, 1)))
    cache[3] = 0.0
    cache[4, 0, 1, 0, 5] = np.nan
    cache[5, 0, 2, hkv - 1, 7] = -np.inf
    cache[6, 1] = np.nan  # values are not looked at
    cache[7, 0] = -np.abs(cache[7, 0])
    ct = torch.as_tensor(cache).to(torch.bfloat16)
    ids = rng.permutation(23)[:20]
    lens = rng.integers(0, ps + 1, 20)
    lens[:8] = ps
    bounds = torch.full((23, hkv, 2, d), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((23, hkv), -5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.page_bounds(ct.cuda(), _i32(ids), bounds, scale, page_len=_i32(lens), status=status)
    assert int(status.item()) == 0
    got, gs = bounds.cpu().numpy(), scale.cpu().numpy()
    for p in range(23):
        for h in range(hkv):
            if p not in ids:
                assert (got[p, h] == 99).all() and gs[p, h] == -5.0
                continue
            n = lens[list(ids).index(p)]
            b, s = o.page_bounds(ct[p, 0, :n, h].float().numpy())
            assert (got[p, h] == b).all() and gs[p, h] == s, (p, h)


LENS = [1, 16, 17, 0, 300, 2000, 161, 700]


@pytest.mark.parametrize("d,ps", [(128, 16), (64, 32)])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (4, 4), (28, 4), (16, 1)])
@pytest.mark.parametrize("select,sink,recent", [(10, 1, 2), (1, 0, 1), (33, 4, 8)])
def test_matches_oracle(K, d, ps, hq, hkv, select, sink, recent):
    host, dev = _case(K, LENS, hq, hkv, d, ps, seed=hq + d + select)
    _check(K, host, dev, select, sink, recent)


@pytest.mark.parametrize("lens,select", [([40000], 64), ([16 * 3000 + 5, 20, 9000], 200), ([4096] * 40, 12)])
def test_sizes(K, lens, select):
    host, dev = _case(K, lens, 4, 2, 64, 16, seed=len(lens))
    _check(K, host, dev, select, 2, 3, max_pages=max(-(-x // 16) for x in lens))


def test_ties_go_to_the_lowest_page(K):
    """Pages with the same keys score the same; many at the threshold."""

    def edit(cache, indptr, indices):
        for i, p in enumerate(indices):
            cache[p, 0] = cache[indices[i % 3], 0]

    host, dev = _case(K, [3000, 90], 8, 2, 128, 16, seed=3, edit=edit)
    for select in (5, 64, 65, 127):
        _check(K, host, dev, select, 1, 1)


def test_zero_queries_and_keys(K):
    """All scores equal (0): the selection is the first pages."""

    def edit(cache, indptr, indices):
        cache[:, 0] = 0.0

    host, dev = _case(K, [2000], 8, 2, 128, 16, seed=3, edit=edit)
    _check(K, host, dev, 20, 2, 2)
    host, dev = _case(K, [2000], 8, 2, 128, 16, seed=4)
    dev["q"].zero_()
    _check(K, dict(host, q=host["q"] * 0), dev, 20, 2, 2)


def test_non_finite_keys_are_selected(K):
    def edit(cache, indptr, indices):
        cache[indices[50], 0, 3, 1, 9] = np.nan

    host, dev = _case(K, [2000], 8, 2, 128, 16, seed=3, edit=edit)
    out, _, sel = _run(K, dev, 10, 1, 1)
    assert 50 in sel[0, 1] and np.isnan(out[0, 4:]).all() and np.isfinite(out[0, :4]).all()


def test_strides_stream_and_long_offsets(K):
    host, dev = _case(K, [900, 400], 16, 8, 128, 16, seed=12)
    wide = torch.full((2, 20, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:19] = dev["q"]
    dev["q"] = wide[:, 3:19]
    pages = (1 << 31) // (2 * 16 * 8 * 128) + 200
    used = dev["indices"].long()
    to = pages - 1 - torch.arange(len(used), device="cuda")
    big = torch.empty(pages, 2, 16, 8, 128, dtype=torch.bfloat16, device="cuda")
    bounds = torch.empty(pages, 8, 2, 128, dtype=torch.int8, device="cuda")
    scale = torch.empty(pages, 8, device="cuda")
    big[to], bounds[to], scale[to] = dev["cache"][used], dev["bounds"][used], dev["scale"][used]
    dev.update(cache=big, bounds=bounds, scale=scale, indices=to.to(torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty(16, 2, 128, dtype=torch.bfloat16, device="cuda").permute(1, 0, 2)
    with torch.cuda.stream(side):
        got = _run(K, dev, 9, 1, 2, out=out)
    want, _, spread, wsel = o.sparse_decode(host["q"], host["cache"], host["indptr"], host["indices"], host["last"],
                                            host["bounds"], host["scale"], num_select=9, sink=1, recent=2)
    assert (got[2] == wsel).all()
    assert (np.abs(got[0] - want) <= U * (np.abs(want) + spread) + F * spread).all()


def test_all_pages_equal_decode(K):
    """A budget that covers every page is dense decode."""

    host, dev = _case(K, [700, 30, 1], 8, 2, 128, 16, seed=8)
    out, _, _ = _run(K, dev, 64, 1, 1)
    ref = K.paged_decode(dev["q"], dev["cache"], dev["indptr"], dev["indices"], dev["last"], num_splits=1,
                         workspace=torch.zeros(4096, dtype=torch.uint8, device="cuda"))
    spread = np.abs(host["cache"][np.isfinite(host["cache"])]).max()
    assert (np.abs(out - ref.double().cpu().numpy()) <= 2 * (2 * U + F) * spread).all()


def test_graph_replay_repeats(K):
    host, dev = _case(K, [5000, 900], 8, 2, 128, 16, seed=21)
    args = [dev[k] for k in ("q", "cache", "indptr", "indices", "last", "bounds", "scale")]
    out = torch.empty_like(dev["q"])
    sel = torch.empty(2, 2, 24, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    kw = dict(num_select=24, sink_pages=1, recent_pages=2, max_pages=313, out=out, selected=sel, workspace=ws)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        K.paged_sparse_decode(*args, **kw)
    torch.cuda.synchronize()
    first = out.clone(), sel.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        K.paged_sparse_decode(*args, **kw)
    for _ in range(3):
        out.zero_()
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first[0]) and torch.equal(sel, first[1])


def test_refusals(K):
    from pagelora_b200 import _capi

    host, dev = _case(K, [400, 30], 8, 2, 128, 16, seed=5)
    _run(K, dev, 4, 1, 1, want=_capi.PL_ERR_INVALID_ARGUMENT, max_pages=10)  # a row of 25 pages
    bad = dict(dev, indices=dev["indices"].clone())
    bad["indices"][3] = 10 ** 6
    _run(K, bad, 40, 1, 1, want=_capi.PL_ERR_PAGE_OUT_OF_RANGE)
    for select, sink, recent in ((4, 3, 2), (4, 0, 0), (4, -1, 1)):
        with pytest.raises(RuntimeError, match="invalid"):
            _run(K, dev, select, sink, recent)
    with pytest.raises(RuntimeError, match="workspace"):
        _run(K, dev, 4, 1, 1, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(TypeError):
        _run(K, dict(dev, bounds=dev["bounds"].int()), 4, 1, 1)
    with pytest.raises(ValueError):
        _run(K, dict(dev, scale=dev["scale"][:3]), 4, 1, 1)
    with pytest.raises(RuntimeError, match="unsupported"):
        _run(K, dict(dev, cache=torch.zeros(9, 2, 64, 2, 128, dtype=torch.bfloat16, device="cuda")), 4, 1, 1)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.page_bounds(dev["cache"], _i32([10 ** 6]), dev["bounds"], dev["scale"], status=status)
    assert int(status.item()) == _capi.PL_ERR_PAGE_OUT_OF_RANGE


def test_rows_without_pages(K):
    """Every row is empty and the page list has no entries."""

    _, dev = _case(K, [0, 0], 4, 2, 64, 16, seed=3)
    dev["indices"] = dev["indices"][:0]
    out, lse, sel = _run(K, dev, 4, 1, 1, max_pages=8)
    assert (out == 0).all() and np.isneginf(lse).all() and (sel == -1).all()


@pytest.mark.parametrize("select", [2900, 3044, 30000])
def test_many_selected_pages(K, select):
    """A list of thousands of pages, and budgets that hold all pages of every row (3000 + 44 in the table)."""

    host, dev = _case(K, [48000, 700], 4, 1, 64, 16, seed=31)
    out, lse, sel = _run(K, dev, select, 1, 1)
    want, wlse, spread, chosen = o.sparse_decode(host["q"], host["cache"], host["indptr"], host["indices"], host["last"],
                                                 host["bounds"], host["scale"], num_select=select, sink=1, recent=1)
    assert (sel == chosen).all()
    assert (np.abs(out - want) <= U * (np.abs(want) + spread) + F * spread).all()
    assert (np.abs(lse - wlse) <= F * (1 + np.abs(wlse))).all()
