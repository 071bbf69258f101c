"""Log sums of prompt queries of NaN, and rows behind the last request."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_window_attention import _case, _i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


@pytest.mark.parametrize("window", [None, 20])
@pytest.mark.parametrize("d", [64, 128])
def test_log_sums_of_prompt_queries_of_nan(K, window, d):
    """NaN, as those of a decode step, in the output too; queries beside it and queries that see nothing are as ever."""

    host, dev = _case([100, 3], [60, 5], 8, 2, d, 16, 2)
    tables = [dev["qo"], dev["indptr"], dev["indices"], dev["last"]]

    def run(q):
        lse = torch.empty(q.shape[:2], device="cuda")
        if window is None:
            return K.paged_prefill(q, dev["cache"], *tables, out_lse=lse), lse
        return K.paged_window_prefill(q, dev["cache"], *tables, window=window, sinks=2, out_lse=lse), lse

    clean, clean_lse = run(dev["q"])
    bad = torch.zeros(65, 8, dtype=torch.bool, device="cuda")
    bad[7, 3] = bad[59, 0] = True
    hurt = dev["q"].clone()
    hurt[bad] = float("nan")
    hurt[60] = float("nan")  # its position is in front of the first one: it sees nothing
    out, lse = run(hurt)
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad])
    assert (out[60:62] == 0).all() and torch.isneginf(lse[60:62]).all()


def test_window_prompts_without_pages_leave_the_rows_behind_the_last(K):
    q = torch.randn(6, 4, 64, device="cuda").bfloat16()
    cache = torch.randn(2, 2, 16, 2, 64, device="cuda").bfloat16()
    out, lse = torch.full_like(q, 5.0), torch.full((6, 4), 7.0, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    K.paged_window_prefill(q, cache, _i32([0, 1, 4]), _i32([0, 0, 0]), none, _i32([0, 0]), window=8, sinks=1, out=out,
                           out_lse=lse)
    assert (out[:4] == 0).all() and torch.isneginf(lse[:4]).all()
    assert (out[4:] == 5).all() and (lse[4:] == 7).all()
