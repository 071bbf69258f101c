"""Tree attention with long tables: many branches over one prefix, and tables
that name more work than a call can have."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, F = 2.0 ** -8, 2.0 ** -12


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64), dtype=torch.int32, device="cuda")


def test_thousands_of_branches_over_a_long_prefix(cuda_device):
    """4096 requests of a token each, whose page lists (4000 shared pages and one of their own) have 16 million entries."""

    from pagelora_b200 import kernels as K

    batch, shared, hq, d = 4096, 4000, 4, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = torch.randn(shared + batch, 2, 16, 1, d, generator=g, device="cuda").bfloat16()
    q = torch.randn(batch, hq, d, generator=g, device="cuda").bfloat16()
    own = torch.arange(shared, shared + batch, device="cuda", dtype=torch.int32)
    indices = torch.cat([torch.arange(shared, device="cuda", dtype=torch.int32).expand(batch, -1), own[:, None]], 1).flatten()
    last = torch.randint(1, 17, (batch,), generator=g, device="cuda").to(torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = K.paged_tree_attention(q, cache, _i32(np.arange(batch + 1)), _i32(np.arange(batch + 1) * (shared + 1)), indices,
                                 last, torch.ones(batch, 1, dtype=torch.int32, device="cuda"), status=status)
    assert int(status.item()) == 0
    prefix = cache[:shared, :, :, 0].double()
    for b in (0, 1, 777, 2048, batch - 1):
        n = int(last[b])
        k, v = (torch.cat([prefix[:, j].reshape(-1, d), cache[shared + b, j, :n, 0].double()]) for j in (0, 1))
        p = torch.softmax(q[b].double() @ k.T / d ** 0.5, -1)
        o, spread = p @ v, p @ v.abs()
        assert ((out[b].double() - o).abs() <= U * (o.abs() + spread) + F * spread).all(), b


@pytest.mark.parametrize("requests", [2100, 4200, 60000])
def test_a_table_that_goes_back(cuda_device, requests):
    """A qo_indptr and kv_indptr of 0, n, 0, n, ... name the same tokens again and again, up to more than 2^31 places
    of work: the call is refused and writes nothing."""

    from pagelora_b200 import _capi
    from pagelora_b200 import kernels as K

    n, pages, heads, d = 64, 1 << 16, 128, 64
    q = torch.zeros(n, heads, d, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(1, 2, 16, heads, d, dtype=torch.bfloat16, device="cuda")
    back = np.arange(requests + 1) % 2
    out = torch.full_like(q, 3.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.paged_tree_attention(q, cache, _i32(back * n), _i32(back * pages), torch.zeros(pages, dtype=torch.int32, device="cuda"),
                           _i32([16] * requests), torch.ones(n, 2, dtype=torch.int32, device="cuda"), out=out, status=status)
    assert int(status.item()) in (_capi.PL_ERR_UNSUPPORTED, _capi.PL_ERR_INVALID_ARGUMENT)
    assert (out == 3.0).all()
