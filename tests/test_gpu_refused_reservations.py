"""A reservation that is refused names no slot: every entry of slot_page and
slot_offset is -1 (which the append kernels reject) and of positions 0,
whatever the buffers held."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages", [64, 20000])  # one CTA, a cluster
@pytest.mark.parametrize("counts,reason", [
    ([40, 2000, 0], "PL_ERR_ROW_CAPACITY"), ([1, 500, 700], "PL_ERR_POOL_EXHAUSTED"), ([3, 5, 0], "PL_ERR_PAGE_SHARED"),
    ([5, -2, 4], "PL_ERR_INVALID_ARGUMENT"),
])
def test_no_slots(cuda_device, pages, counts, reason):
    from pagelora_b200 import _capi
    from pagelora_b200 import kernels as K

    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda_device)  # noqa: E731
    cap = 100
    refcount = torch.ones(pages, dtype=torch.int32, device=cuda_device)
    refcount[pages - 20:] = 0  # 20 free pages
    if reason == "PL_ERR_PAGE_SHARED":
        refcount[7] = 2
    table = torch.zeros(3, cap, dtype=torch.int32, device=cuda_device)
    table[0, 0], table[1, 0] = 4, 7
    num, last = i32(1, 1, 0), i32(9, 3, 0)
    total = sum(counts)
    # buffers of an earlier step: slots of live tokens
    page, off, pos = (torch.full((total,), v, dtype=torch.int32, device=cuda_device) for v in (4, 2, 77))
    status = i32(0)
    before = [t.clone() for t in (refcount, table, num, last)]
    K.page_reserve(refcount, table, num, last, i32(0, *torch.tensor(counts).cumsum(0).tolist()), 16, slot_page=page,
                   slot_offset=off, positions=pos, status=status)
    assert int(status.item()) == getattr(_capi, reason)
    assert all(torch.equal(a, b) for a, b in zip(before, (refcount, table, num, last)))
    assert (page == -1).all() and (off == -1).all() and (pos == 0).all()
