"""Sparse decode at sizes that change its way through the kernels: rows of
more than 8192 pages, more than eight kv heads, and budgets that cover all pages."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, F = 2.0 ** -8, 2.0 ** -12


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64).reshape(-1), dtype=torch.int32, device="cuda")


def _check(lens, hq, hkv, d, select, sink, recent, seed, ties=False):
    """Selection in integers and attention in 64 bits, with torch operations on the whole row."""

    from pagelora_b200 import kernels as K

    g = torch.Generator(device="cuda").manual_seed(seed)
    n = [-(-x // 16) for x in lens]
    pool = sum(n) + 5
    perm = torch.randperm(pool, generator=g, device="cuda")[: sum(n)].to(torch.int32)
    cache = torch.randn(pool, 2, 16, hkv, d, generator=g, device="cuda").bfloat16()
    if ties:  # few different pages
        cache[:, 0] = cache[torch.arange(pool, device="cuda") % 7, 0]
    q = torch.randn(len(lens), hq, d, generator=g, device="cuda").bfloat16()
    bounds = torch.empty(pool, hkv, 2, d, dtype=torch.int8, device="cuda")
    scale = torch.empty(pool, hkv, device="cuda")
    K.page_bounds(cache, torch.arange(pool, dtype=torch.int32, device="cuda"), bounds, scale)
    indptr = np.cumsum([0] + n)
    last = [x - 16 * (k - 1) for x, k in zip(lens, n)]
    sel = torch.full((len(lens), hkv, select), -9, dtype=torch.int32, device="cuda")
    lse = torch.empty(len(lens), hq, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = K.paged_sparse_decode(q, cache, _i32(indptr), perm, _i32(last), bounds, scale, num_select=select,
                                sink_pages=sink, recent_pages=recent, max_pages=max(n), selected=sel, out_lse=lse,
                                status=status)
    assert int(status.item()) == 0
    group = hq // hkv
    inv = np.float32(1.0) / np.float32(127.0)
    for b in range(len(lens)):
        ids = perm[int(indptr[b]): int(indptr[b + 1])].long()
        for h in range(hkv):
            qg = q[b, h * group:(h + 1) * group].float()
            if n[b] <= select:
                want = list(range(n[b]))
            else:
                sq = qg.abs().max() * float(inv)
                qi = (qg / sq).round().clamp(-127, 127).double()
                bd = bounds[ids, h].double()
                dot = torch.stack([torch.maximum(v * bd[:, 0], v * bd[:, 1]).sum(-1) for v in qi]).amax(0)
                score = (dot.float() * scale[ids, h]).cpu().numpy()
                mid = np.arange(sink, n[b] - recent)
                top = mid[np.lexsort((mid, -score[mid]))][: select - sink - recent]
                want = sorted([*range(sink), *top.tolist(), *range(n[b] - recent, n[b])])
            got = sel[b, h].tolist()
            assert got[: len(want)] == want and all(x == -1 for x in got[len(want):]), (b, h)
            keys = torch.ones(len(want), 16, dtype=torch.bool, device="cuda")
            if want[-1] == n[b] - 1:
                keys[-1, last[b]:] = False
            pages = ids[torch.tensor(want, device="cuda")]
            k, v = (cache[pages, j, :, h][keys].double() for j in (0, 1))
            s = qg.double() @ k.T / d ** 0.5
            p = torch.softmax(s, -1)
            spread, o = p @ v.abs(), p @ v
            err = (out[b, h * group:(h + 1) * group].double() - o).abs()
            assert (err <= U * (o.abs() + spread) + F * spread).all(), (b, h, float(err.max()))
            ref = torch.logsumexp(s, -1)
            assert ((lse[b, h * group:(h + 1) * group].double() - ref).abs() <= F * (1 + ref.abs())).all()


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("lens", [[16 * 8193 - 3], [16 * 8192, 16 * 8195, 70], [16 * 8198 + 1, 16 * 30001, 300]])
@pytest.mark.parametrize("select", [12, 700, 9000])
def test_rows_of_more_than_8192_pages(cuda_device, lens, select, ties):
    _check(lens, 4, 1, 64, select, 2, 3, seed=len(lens) + select, ties=ties)


@pytest.mark.parametrize("hq,hkv", [(9, 9), (24, 12), (64, 16), (80, 20), (256, 16)])
def test_more_than_eight_kv_heads(cuda_device, hq, hkv):
    _check([1000, 15, 3333, 640], hq, hkv, 128, 30, 1, 2, seed=hq)


@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (64, 4, 4)])
def test_budgets_that_cover_all_pages(cuda_device, d, hq, hkv):
    _check([700, 30, 1, 16], hq, hkv, d, 64, 1, 1, seed=d)
