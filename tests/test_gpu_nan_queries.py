"""A query head of NaN gives NaN, in the output and the LSE, however the work
was cut; the heads and rows beside it are as without it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64), dtype=torch.int32, device="cuda")


# contexts that one CTA reads, and that several share; rows that fill one tile per CTA and two
@pytest.mark.parametrize("ctx", [100, 3000, 9000])
@pytest.mark.parametrize("n", [1, 7, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_tree_attention(K, ctx, n, d):
    g = torch.Generator(device="cuda").manual_seed(ctx + n)
    pages = -(-(ctx + n) // 16)
    cache = torch.randn(pages, 2, 16, 2, d, generator=g, device="cuda").bfloat16()
    q = torch.randn(n, 8, d, generator=g, device="cuda").bfloat16()
    mask, _ = K.tree_mask(_i32(range(-1, n - 1)), _i32([0, n]), -(-n // 32))
    table = (_i32([0, n]), _i32([0, pages]), _i32(range(pages)), _i32([ctx + n - 16 * (pages - 1)]))

    def run(q, mask):
        lse = torch.empty(n, 8, device="cuda")
        return K.paged_tree_attention(q, cache, *table, mask, out_lse=lse), lse

    clean, clean_lse = run(q, mask)
    bad = torch.zeros(n, 8, dtype=torch.bool, device="cuda")
    bad[n // 2, 3] = bad[0, 6] = True
    hurt = q.clone()
    hurt[bad] = float("nan")
    out, lse = run(hurt, mask)
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad])


def test_tree_attention_of_a_row_that_sees_nothing(K):
    """Nothing is seen, so the query does not count: 0 and -inf."""

    q = torch.full((2, 4, 128), float("nan"), device="cuda").bfloat16()
    cache = torch.randn(1, 2, 16, 2, 128, device="cuda").bfloat16()
    lse = torch.empty(2, 4, device="cuda")
    out = K.paged_tree_attention(q, cache, _i32([0, 2]), _i32([0, 1]), _i32([0]), _i32([2]), _i32([[0], [3]]), out_lse=lse)
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and out[1].isnan().all() and lse[1].isnan().all()


@pytest.mark.parametrize("rows,lens", [(1, 900), (2, 5000), (40, 1500)])  # several CTAs per (row, kv head), and one
@pytest.mark.parametrize("d,select", [(128, 20), (64, 40), (128, 400)])
def test_sparse_decode(K, rows, lens, d, select):
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    hkv, n = 4, -(-lens // 16)
    pages = rows * n
    cache = torch.randn(pages, 2, 16, hkv, d, generator=g, device="cuda").bfloat16()
    q = torch.randn(rows, 16, d, generator=g, device="cuda").bfloat16()
    bounds = torch.zeros(pages, hkv, 2, d, dtype=torch.int8, device="cuda")
    scale = torch.zeros(pages, hkv, device="cuda")
    K.page_bounds(cache, _i32(range(pages)), bounds, scale)

    def run(q):
        lse = torch.empty(rows, 16, device="cuda")
        out = K.paged_sparse_decode(q, cache, _i32(np.arange(rows + 1) * n), _i32(range(pages)),
                                    _i32([lens - 16 * (n - 1)] * rows), bounds, scale, num_select=select, max_pages=n,
                                    out_lse=lse)
        return out, lse

    clean, clean_lse = run(q)
    bad = torch.zeros(rows, 16, dtype=torch.bool, device="cuda")
    bad[rows // 2, 5] = bad[0, 12:] = True
    hurt = q.clone()
    hurt[bad] = float("nan")
    out, lse = run(hurt)
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert out[~bad].isfinite().all() and lse[~bad].isfinite().all()
    alone = torch.ones(rows, hkv, dtype=torch.bool, device="cuda")  # kv heads without a NaN: the same pages
    alone[rows // 2, 1] = alone[0, 3] = False
    alone = alone.repeat_interleave(4, 1)
    assert torch.equal(out[alone], clean[alone]) and torch.equal(lse[alone], clean_lse[alone])
