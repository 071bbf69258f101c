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
