"""Attention weight of decode steps where pages or tables are not in order: what
is not seen receives nothing, and the rows beside it keep their weights.

Tolerances of test_gpu_evict.py.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import small_cache as o
from tests.test_gpu_evict import _weights_ok
from tests.test_gpu_window_attention import _case, _i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (9, 1, 128)])
def test_decode_of_rows_whose_pages_are_not_in_the_pool(K, hq, hkv, d):
    """Such positions are not seen: they receive nothing."""

    host, dev = _case([100, 40, 48], [1, 1, 1], hq, hkv, d, 16, 9)
    tables = [dev["indptr"], dev["indices"], dev["last"]]
    before = torch.rand(3, 100, device="cuda")
    good, status = before.clone(), _status()
    want = K.paged_decode_weights(dev["q"], dev["cache"], *tables, good, status=status)
    assert int(status.item()) == 0
    bad = host["indices"].copy()
    bad[7:10] = -1                    # all pages of row 1
    bad[11] = len(host["cache"])      # the middle page of row 2
    weight = before.clone()
    lse = torch.empty(3, hq, device="cuda")
    out = K.paged_decode_weights(dev["q"], dev["cache"], tables[0], _i32(bad), tables[2], weight, out_lse=lse,
                                 status=status)
    assert int(status.item()) == 3
    assert torch.equal(weight[0], good[0]) and torch.equal(out[0], want[0])
    assert torch.equal(weight[1], before[1]) and (out[1] == 0).all() and torch.isneginf(lse[1]).all()
    k, v = o.row_tokens(host["cache"], host["indices"], 10, 13, host["last"][2])
    see = (np.arange(48) < 16) | (np.arange(48) >= 32)
    p = o.attend(host["q"][2], k, v, see, d ** -0.5)[2]
    _weights_ok(weight[2:], before[2:].cpu(), [p.sum(0)], [48])
    assert torch.equal(weight[2, 16:32], before[2, 16:32])


@pytest.mark.parametrize("ends", [[0, 4, 1000, 8, 12], [0, 1000, 8, 12, 16], [0, 4, -3, 8, 12]])
def test_decode_of_rows_behind_a_table_outside_the_entries(K, ends):
    lens = [60, 61, 62, 63]
    host, dev = _case(lens, [1] * 4, 8, 2, 64, 16, 12)
    weight, status = torch.zeros(4, 64, device="cuda"), _status()
    indices = dev["indices"]  # 16 entries
    last = _i32([12] * 4)
    K.paged_decode_weights(dev["q"], dev["cache"], _i32(ends), indices, last, weight, status=status)
    assert int(status.item()) == 1
    for r in range(4):
        a, b = ends[r], ends[r + 1]
        if not 0 <= a <= b <= 16:
            assert (weight[r] == 0).all()
            continue
        alone = torch.zeros(1, 64, device="cuda")
        K.paged_decode_weights(dev["q"][r:r + 1], dev["cache"], _i32([0, b - a]), indices[a:b].contiguous(), last[:1], alone)
        assert torch.allclose(weight[r], alone[0], rtol=2.0 ** -11, atol=1e-9) and (weight[r, :60] > 0).all(), r
