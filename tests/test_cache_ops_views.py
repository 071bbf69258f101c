"""The wrappers of the cache operators refuse views whose rows overlap: the
kernels would read or write behind the memory that such a view has."""

from __future__ import annotations

import pytest
import torch


class OnDevice:
    """A CPU tensor that says it is on the device (for checks that come before any launch)."""

    def __init__(self, t):
        self.t, self.is_cuda, self.dtype, self.shape = t, True, t.dtype, t.shape
        self.dim, self.stride = t.dim, t.stride


@pytest.mark.parametrize("view", [
    lambda t: t[:1].expand(6, -1), lambda t: t[:1, :1].expand(6, 1), lambda t: t.view(-1).as_strided((6, 4), (3, 1)),
    lambda t: t.view(-1).unfold(0, 4, 1)[:6],
])
def test_overlapping_rows(view):
    from pagelora_b200.kernels import _need_rows

    with pytest.raises(ValueError, match="rows of its own"):
        _need_rows(OnDevice(view(torch.zeros(8, 4, dtype=torch.int32))), "mask", 6)


@pytest.mark.parametrize("view,want", [
    (lambda t: t, (4, 4)), (lambda t: t[:, :2], (4, 2)), (lambda t: t[::2], (8, 4)), (lambda t: t[:, 1:2], (4, 1)),
    (lambda t: t[:1].expand(1, -1), (4, 4)), (lambda t: t.view(-1).as_strided((1, 4), (0, 1)), (4, 4)),
    (lambda t: t[:, :0], (4, 0)),
])
def test_rows_of_their_own(view, want):
    from pagelora_b200.kernels import _need_rows

    assert _need_rows(OnDevice(view(torch.zeros(8, 4, dtype=torch.int32))), "keep", 1) == want


@pytest.mark.gpu
def test_calls_with_overlapping_rows(cuda_device):
    from pagelora_b200 import kernels as K

    i32 = dict(dtype=torch.int32, device=cuda_device)
    one = torch.ones(1, 1, **i32)
    qo, kv = torch.tensor([0, 3], **i32), torch.tensor([0, 1], **i32)
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    cache = torch.zeros(1, 2, 16, 1, 64, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError):
        K.paged_tree_attention(q, cache, qo, kv, kv[:1], kv[1:] + 9, one.expand(3, 1))
    parents = torch.tensor([-1, 0, 1], **i32)
    with pytest.raises(ValueError):
        K.tree_mask(parents, qo, 1, mask=one.expand(3, 1))
    ids = torch.zeros(3, dtype=torch.int64, device=cuda_device)
    two, row = torch.tensor([0, 1, 3], **i32), torch.zeros(1, 3, **i32)
    with pytest.raises(ValueError):
        K.tree_accept(parents, ids, ids, two, kv, keep=row.expand(2, 3), keep_count=kv.clone(), next_token=ids[:2].clone())
    pool = torch.zeros(1, 4, 2, 16, 1, 64, dtype=torch.bfloat16, device=cuda_device)
    tables = torch.zeros(4, **i32), torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(2, **i32)
    with pytest.raises(ValueError):
        K.cache_compact(pool, *tables, torch.zeros(2, **i32), row.expand(2, 3), torch.zeros(2, **i32))


def test_workspaces_that_are_not_contiguous():
    """A workspace's size is that of its entries, which a view may share."""

    from pagelora_b200.kernels import _workspace

    ws = torch.empty(64, dtype=torch.uint8)
    assert _workspace(ws, 16, ws) is ws and _workspace(None, 99, ws).numel() == 99
    for view in (ws[:1].expand(1 << 20), ws[::2], ws.view(8, 8).t()):
        with pytest.raises(ValueError, match="contiguous"):
            _workspace(view, 16, ws)
