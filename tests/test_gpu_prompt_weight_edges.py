"""Attention weight of prompts where a query or a table is not in order, and its
exponentials one by one.

Tolerances of test_gpu_evict.py, except where scores are exact: there a weight
is one exponential.  With s the score and c the log sum, x = s fl(log2 e) -
fl(c fl(log2 e)) is off by at most 2^-24 (|s| log2 e (representation of
log2 e) + 2 |c| log2 e + |x|), times ln 2 in the weight; 2^x by 2 + 2^-22
units in the last place (the multi-function unit's bound; the polynomial's
1.9e-7 is below it), at most 2.01 * 2^-23 relative.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_window_attention import _case, _i32

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _prompt(K, host, dev, edit=None, status=None, lse=None):
    q = dev["q"]
    tables = [dev["qo"], dev["indptr"], dev["indices"], dev["last"]]
    if lse is None:
        lse = torch.empty(q.shape[:2], device="cuda")
        K.paged_prefill(q, dev["cache"], *tables, out_lse=lse)
    if edit is not None:
        edit(tables)
    rows = tables[0].numel() - 1
    weight = torch.zeros(rows, 200, device="cuda")
    K.paged_prefill_weights(q, dev["cache"], *tables, lse, weight, status=status)
    torch.cuda.synchronize()
    return weight


@pytest.mark.parametrize("at", [0, 2, 3, 10, 31, 59])
def test_a_prompt_token_of_nan(K, at):
    """NaN for every position that the token sees, whatever the place of its column; nothing for the others."""

    def edit(q, cache, indptr, indices, lens):
        q[at] = np.nan

    host, dev = _case([100], [60], 1, 1, 64, 16, at, edit)
    weight = _prompt(K, host, dev)
    pos = 40 + at
    assert torch.isnan(weight[0, :pos + 1]).all()
    assert torch.isfinite(weight[0, pos + 1:]).all() and (weight[0, pos + 1:100] > 0).all()


@pytest.mark.parametrize("head", [0, 1, 2, 3])
def test_a_prompt_head_of_nan(K, head):
    def edit(q, cache, indptr, indices, lens):
        q[30, head] = np.nan

    host, dev = _case([100], [60], 4, 1, 64, 16, head, edit)
    weight = _prompt(K, host, dev)
    assert torch.isnan(weight[0, :71]).all() and torch.isfinite(weight[0, 71:]).all()


def _exact_scores(K, score, logsum, at):
    """Weights that prompt token `at` of 128 gives alone; its scores against the positions are given (bf16 values)."""

    q = torch.zeros(128, 1, 64, device="cuda")
    q[:, 0, 5] = 1.0
    cache = torch.zeros(8, 2, 16, 1, 64, device="cuda")
    cache[:, 0, :, 0, 5] = score.view(8, 16)
    lse = torch.full((128, 1), INF, device="cuda")  # the others give exp(-inf)
    lse[at] = logsum
    weight = torch.zeros(1, 128, device="cuda")
    K.paged_prefill_weights(q.bfloat16(), cache.bfloat16(), _i32([0, 128]), _i32([0, 8]), _i32(range(8)), _i32([16]), lse,
                            weight, sm_scale=1.0)
    return weight[0, :at + 1].double().cpu()


def _one_exponential(got, s, c):
    log2e = 1.4426950408889634
    x = (s - c) * log2e
    tol = 2.01 * 2.0 ** -23 + 2.0 ** -24 * 0.6932 * (s.abs() * log2e + 2 * abs(c) * log2e + x.abs())
    want = torch.exp(s - c)
    top = float(torch.finfo(torch.float32).max)
    edge = (want / top - 1).abs() <= tol  # either way
    big = (want > top) & ~edge
    assert torch.isinf(got[big]).all()
    ok = ~big & ~edge & (want > 2.0 ** -125)
    assert ((got - want).abs()[ok] <= tol[ok] * want[ok]).all(), ((got - want).abs()[ok] / (tol[ok] * want[ok])).max()
    assert (got[want <= 2.0 ** -125] <= 2.0 ** -124).all()
    return int(ok.sum()), int(big.sum())


@pytest.mark.parametrize("at", [96, 97, 98, 99, 100, 106, 107, 115, 122, 123, 127])
def test_one_exponential_of_a_prompt(K, at):
    """Columns of the multi-function unit and of the polynomial alike."""

    g = torch.Generator().manual_seed(at)
    s = (torch.rand(128, generator=g) * 2 - 1).bfloat16().float()
    _one_exponential(_exact_scores(K, s.cuda(), 0.0, at), s[:at + 1].double(), 0.0)
    # far from the log sum, on both sides: products that fp32 does not hold are inf or 0
    s = ((torch.rand(128, generator=g) * 2 - 1) * 200).bfloat16().float()
    ok, big = _one_exponential(_exact_scores(K, s.cuda(), 3.0, at), s[:at + 1].double(), 3.0)
    assert ok > 10 and big > 10
    s = torch.linspace(85, 92, 128).bfloat16().float()  # around the largest number
    _one_exponential(_exact_scores(K, s.cuda(), 0.0, at), s[:at + 1].double(), 0.0)
    s = torch.full((128,), -INF)
    s[:64] = -1e30
    assert (_exact_scores(K, s.cuda(), 1.0, at) == 0).all()


# ------------------------------------------------------------------ tables
def _many(seed):
    return _case([20 + i for i in range(40)], [5] * 40, 4, 2, 64, 16, seed)


def test_prompts_behind_the_first_requests_report_bad_tables(K):
    host, dev = _many(3)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = _prompt(K, host, dev, status=status)
    assert int(status.item()) == 0 and (good[:, :20] > 0).all()

    def past(tables):
        tables[1] = tables[1].clone()
        tables[1][36] = 100000  # the end of request 35, the beginning of request 36

    got = _prompt(K, host, dev, past, status)
    rest = [r for r in range(40) if r not in (35, 36)]
    assert int(status.item()) == 1
    assert torch.equal(got[rest], good[rest]) and (got[35:37] == 0).all()


def test_prompts_behind_the_first_requests_report_too_many_tokens(K):
    lens = [20 + i for i in range(40)]
    host, dev = _case(lens, [5] * 39 + [59], 4, 2, 64, 16, 3)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = _prompt(K, host, dev, status=status)
    assert int(status.item()) == 0
    tables = [dev["qo"], dev["indptr"], dev["indices"], dev["last"]]
    lse = torch.empty(dev["q"].shape[:2], device="cuda")
    K.paged_prefill(dev["q"], dev["cache"], *tables, out_lse=lse)
    last = dev["last"].clone()
    last[39] = 1  # 49 positions for 59 tokens
    weight = torch.zeros(40, 200, device="cuda")
    K.paged_prefill_weights(dev["q"], dev["cache"], *tables[:3], last, lse, weight, status=status)
    assert int(status.item()) == 1
    assert torch.equal(weight[:39], good[:39]) and (weight[39] == 0).all()


def test_prompts_without_any_page_are_reported(K):
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    cache = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    weight, status = torch.full((2, 10), 3.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    K.paged_prefill_weights(q, cache, _i32([0, 3, 3]), _i32([0, 0, 0]), none, _i32([0, 0]),
                            torch.zeros(3, 4, device="cuda"), weight, status=status)
    assert int(status.item()) == 1 and (weight == 3).all()
