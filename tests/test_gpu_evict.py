"""Accumulated attention weight and the choice of what to keep, against the
oracle (oracle/small_cache.py).

Weights are sums of exponentials of fp32 scores: |err| <= 2^-12 of what the
call adds to a position, and fp32's half step of the sum with what was there.
Kept positions and moved weights are equal.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import small_cache as o
from tests.test_gpu_window_attention import _case, _check, _i32

pytestmark = pytest.mark.gpu

F = 2.0 ** -12


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _weights_ok(got, before, added, lens):
    got, before = got.double().cpu().numpy(), before.double().cpu().numpy()
    for b, n in enumerate(lens):
        want = before[b, :n] + added[b]
        tol = F * added[b] + 2.0 ** -23 * np.abs(want) + 1e-12
        assert (np.abs(got[b, :n] - want) <= tol).all(), b
        assert (got[b, n:] == before[b, n:]).all()


LENS = [1, 16, 17, 0, 300, 1500, 161, 700]


@pytest.mark.parametrize("hq,hkv,d,ps", [(32, 8, 128, 16), (8, 8, 64, 32), (28, 4, 128, 64), (16, 1, 64, 128),
                                         (10, 5, 128, 16), (9, 1, 128, 32)])
def test_decode_weights(K, hq, hkv, d, ps):
    host, dev = _case(LENS, [1] * len(LENS), hq, hkv, d, ps, hq)
    wide = torch.rand(len(LENS), 2000, device="cuda")
    weight = wide[:, :1700]
    before = wide.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.empty(len(LENS), hq, device="cuda")
    args = (dev["q"], dev["cache"], dev["indptr"], dev["indices"], dev["last"])
    out = K.paged_decode_weights(*args, weight, out_lse=lse, status=status)
    assert int(status.item()) == 0
    _check(out, lse, host, None, 0, d ** -0.5)
    added = o.paged(host["q"], host["cache"], host["qo"], host["indptr"], host["indices"], host["last"], d ** -0.5)[2]
    _weights_ok(wide, before, added, LENS)
    # again without a log sum of the caller's: the same bits
    wide2 = before.clone()
    assert torch.equal(K.paged_decode_weights(*args, wide2[:, :1700]), out) and torch.equal(wide2, wide)


def test_decode_weights_capacity_and_nan(K):
    host, dev = _case([100, 40], [1, 1], 4, 2, 64, 16, 3)
    weight = torch.zeros(2, 50, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.paged_decode_weights(dev["q"], dev["cache"], dev["indptr"], dev["indices"], dev["last"], weight, status=status)
    assert int(status.item()) == 12
    added = o.paged(host["q"], host["cache"], host["qo"], host["indptr"], host["indices"], host["last"], 64 ** -0.5)[2]
    _weights_ok(weight, torch.zeros(2, 50), [added[0][:50], added[1]], [50, 40])


@pytest.mark.parametrize("hq,hkv,d,ps", [(32, 8, 128, 16), (8, 8, 64, 32), (28, 4, 128, 64), (16, 1, 64, 128),
                                         (10, 5, 128, 16), (34, 1, 128, 16), (128, 1, 64, 16)])
def test_prompt_weights(K, hq, hkv, d, ps):
    n = [1, 16, 5, 0, 300, 130, 161, 64]
    lens = [1, 16, 17, 40, 300, 900, 161, 700]
    host, dev = _case(lens, n, hq, hkv, d, ps, hq)
    weight = torch.rand(8, 900, device="cuda")
    before = weight.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.empty(sum(n), hq, device="cuda")
    wide = torch.zeros(sum(n), hq, d + 8, dtype=torch.bfloat16, device="cuda")
    q = wide[:, :, :d]
    q.copy_(dev["q"])
    tables = (dev["qo"], dev["indptr"], dev["indices"], dev["last"])
    K.paged_prefill(q, dev["cache"], *tables, out_lse=lse, status=status)
    K.paged_prefill_weights(q, dev["cache"], *tables, lse, weight, status=status)
    assert int(status.item()) == 0
    added = o.paged(host["q"], host["cache"], host["qo"], host["indptr"], host["indices"], host["last"], d ** -0.5)[2]
    _weights_ok(weight, before, added, lens)


def test_prompt_weights_of_empty_log_sums_and_bad_tables(K):
    host, dev = _case([200, 90], [70, 90], 4, 2, 64, 16, 4)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.empty(160, 4, device="cuda")
    tables = [dev["qo"], dev["indptr"], dev["indices"], dev["last"]]
    K.paged_prefill(dev["q"], dev["cache"], *tables, out_lse=lse)
    lse[70:] = -float("inf")
    weight = torch.zeros(2, 200, device="cuda")
    K.paged_prefill_weights(dev["q"], dev["cache"], *tables, lse, weight, status=status)
    assert int(status.item()) == 0 and (weight[1] == 0).all() and (weight[0] > 0).all()
    first = weight[0].clone()
    weight.zero_()
    tables[1] = _i32([0, 13, 500])
    K.paged_prefill_weights(dev["q"], dev["cache"], *tables, lse, weight, status=status)
    assert int(status.item()) == 1 and torch.equal(weight[0], first) and (weight[1] == 0).all()
    status.zero_()
    weight = torch.zeros(2, 150, device="cuda")
    tables[1] = dev["indptr"]
    K.paged_prefill_weights(dev["q"], dev["cache"], *tables, lse, weight, status=status)
    assert int(status.item()) == 12 and torch.equal(weight[0], first[:150])


def _select(K, weight, lens, budget, sinks, recent, width=None):
    rows = len(lens)
    width = budget - sinks if width is None else width
    kf, kc = _i32([-5] * rows), _i32([-5] * rows)
    keep = torch.full((rows, width), -9, dtype=torch.int32, device="cuda")
    out = torch.full_like(weight, 9.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.evict_select(weight, _i32(lens), budget, sinks=sinks, recent=recent, keep_from=kf, keep=keep, keep_count=kc,
                   out_weight=out, status=status)
    torch.cuda.synchronize()
    return kf.cpu().numpy(), keep.cpu().numpy(), kc.cpu().numpy(), out.cpu().numpy(), int(status.item())


def _check_select(got, weight, lens, budget, sinks, recent):
    kf, keep, kc, out, status = got
    assert status == 0
    w = weight.cpu().numpy()
    for r, n in enumerate(lens):
        pos = o.select(w[r, :n], n, budget, sinks, recent)
        if n <= budget:
            assert kf[r] == n and kc[r] == 0 and (keep[r] == -1).all()
        else:
            assert kf[r] == sinks and kc[r] == budget - sinks
            assert (keep[r, :kc[r]] == pos[sinks:]).all() and (keep[r, kc[r]:] == -1).all()
        assert np.array_equal(out[r, :len(pos)], w[r, pos], equal_nan=True)
        assert (out[r, len(pos):] == 0).all()


@pytest.mark.parametrize("cap", [700, 40000])
@pytest.mark.parametrize("budget,sinks,recent", [(64, 4, 10), (64, 64, 0), (64, 0, 64), (1, 0, 0), (300, 3, 100), (65, 0, 1)])
def test_select(K, cap, budget, sinks, recent):
    rng = np.random.default_rng(budget + sinks)
    lens = [0, 1, budget, budget + 1, 65, 300, 699, cap, cap - 1, 512]
    w = rng.random((len(lens), cap)).astype(np.float32) ** 8
    w[4] = 0.25                                       # all equal
    w[5] = rng.integers(0, 3, cap)                    # many ties
    w[6, ::3], w[6, 1::3] = 0.0, -0.0                 # equal zeros
    w[7] = rng.normal(size=cap)                       # negative ones too
    w[8, :200:7] = np.nan
    w[9, ::5], w[9, 1::5] = np.inf, -np.inf
    weight = torch.as_tensor(w).cuda()
    _check_select(_select(K, weight, lens, budget, sinks, recent, max(budget - sinks, 1) + 3), weight, lens, budget,
                  sinks, recent)


def test_select_of_strided_rows_and_bad_lengths(K):
    wide = torch.rand(3, 1000, device="cuda")
    weight = wide[:, 10:510]
    got = _select(K, weight, [500, 300, 20], 100, 2, 5)
    _check_select(got, weight, [500, 300, 20], 100, 2, 5)
    kf, keep, kc, out, status = _select(K, weight, [501, -3, 20], 100, 2, 5)
    assert status == 1 and list(kf) == [501, 0, 20] and list(kc) == [0, 0, 0] and (keep == -1).all()


def test_a_cache_that_evicts(K):
    """Prompt, its weights, decode steps with weights, eviction, and the attention over what stays."""

    rng = np.random.default_rng(41)
    ps, hq, hkv, d, rows, cap = 16, 8, 2, 64, 3, 20
    pool = torch.zeros(1, 60, 2, ps, hkv, d, dtype=torch.bfloat16, device="cuda")
    count = torch.zeros(60, dtype=torch.int32, device="cuda")
    table = torch.zeros(rows, cap, dtype=torch.int32, device="cuda")
    num, last = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    indptr, indices = _i32([0] * (rows + 1)), _i32([0] * rows * cap)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    weight, spare = torch.zeros(rows, cap * ps, device="cuda"), torch.zeros(rows, cap * ps, device="cuda")
    ref = [np.zeros((0, 2, hkv, d)) for _ in range(rows)]
    wref = [np.zeros(0) for _ in range(rows)]

    def grow(n):
        t = sum(n)
        page, off = _i32([0] * t), _i32([0] * t)
        qo = _i32(np.cumsum([0] + n))
        K.page_reserve(count, table, num, last, qo, ps, slot_page=page, slot_offset=off, out_indptr=indptr,
                       out_indices=indices, status=status)
        x = torch.as_tensor(rng.normal(size=(t, 2, hkv, d)).astype(np.float32)).to(torch.bfloat16).cuda()
        K.kv_append(x[:, 0].contiguous(), x[:, 1].contiguous(), pool[0], page, off, status)
        at = 0
        for r, k in enumerate(n):
            ref[r] = np.concatenate([ref[r], x[at:at + k].double().cpu().numpy()])
            wref[r] = np.concatenate([wref[r], np.zeros(k)])
            at += k
        q = torch.as_tensor(2 * rng.normal(size=(t, hq, d)).astype(np.float32)).to(torch.bfloat16).cuda()
        return q, qo

    def note(q, n):
        at = 0
        for r, k in enumerate(n):
            length = len(ref[r])
            for i in range(k):
                p = o.attend(q[at].double().cpu().numpy(), ref[r][:, 0], ref[r][:, 1],
                             o.visible(length - k + i, length, None, 0), d ** -0.5)[2]
                wref[r] += p.sum(0)
                at += 1

    n = [120, 33, 250]
    q, qo = grow(n)
    lse = torch.empty(sum(n), hq, device="cuda")
    K.paged_prefill(q, pool[0], qo, indptr, indices, last, out_lse=lse, status=status)
    K.paged_prefill_weights(q, pool[0], qo, indptr, indices, last, lse, weight, status=status)
    note(q, n)
    kf, kc = _i32([0] * rows), _i32([0] * rows)
    keep = torch.zeros(rows, 90, dtype=torch.int32, device="cuda")
    for _ in range(3):
        for _ in range(5):
            q, _ = grow([1] * rows)
            out = K.paged_decode_weights(q, pool[0], indptr, indices, last, weight, status=status)
            note(q, [1] * rows)
            for r in range(rows):
                want, _, _, spread = o.attend(q[r].double().cpu().numpy(), ref[r][:, 0], ref[r][:, 1],
                                              np.ones(len(ref[r]), bool), d ** -0.5)
                err = np.abs(out[r].double().cpu().numpy() - want)
                assert (err <= 2.0 ** -8 * (np.abs(want) + spread) + F * spread).all()
        lens = _i32([len(x) for x in ref])
        for r in range(rows):
            assert np.allclose(weight[r, :len(ref[r])].cpu().numpy(), wref[r], rtol=2.0 ** -11, atol=1e-9)
        K.evict_select(weight, lens, 92, sinks=2, recent=20, keep_from=kf, keep=keep, keep_count=kc, out_weight=spare,
                       status=status)
        K.cache_compact(pool, count, table, num, last, kf, keep, kc, status=status)
        for r in range(rows):  # the choice is exact for the weights that the device holds
            pos = o.select(weight[r].cpu().numpy(), len(ref[r]), 92, 2, 20)
            ref[r], wref[r] = ref[r][pos], wref[r][pos]
        weight, spare = spare, weight
    assert int(status.item()) == 0
    assert [len(x) for x in ref] == [92, 48, 92]


def test_prompt_weights_stay_apart(K):
    """A request's weights do not depend on its neighbours' queries or on unused memory."""

    def edit(q, cache, indptr, indices, lens):
        q[70:130] = np.nan  # request 1, beside tiles of requests 0 and 2

    host, dev = _case([200, 90, 77], [70, 60, 37], 14, 2, 64, 16, 6, edit)
    tables = [dev["qo"], dev["indptr"], dev["indices"], dev["last"]]
    lse = torch.empty(167, 14, device="cuda")
    K.paged_prefill(dev["q"], dev["cache"], *tables, out_lse=lse)
    weight = torch.zeros(3, 200, device="cuda")
    K.paged_prefill_weights(dev["q"], dev["cache"], *tables, lse, weight)
    added = o.paged(host["q"][:70], host["cache"], host["qo"][:2], host["indptr"], host["indices"], host["last"][:1],
                    64 ** -0.5)[2]
    _weights_ok(weight[:1], torch.zeros(1, 200), added, [200])
    assert torch.isnan(weight[1, :90]).all() and torch.isfinite(weight[2]).all() and (weight[2, :77] > 0).all()


@pytest.mark.parametrize("n,length,hq,hkv", [(1500, 1500, 4, 2), (700, 1300, 6, 1), (40, 3000, 8, 2)])
def test_prompt_weights_over_many_runs(K, n, length, hq, hkv):
    host, dev = _case([length], [n], hq, hkv, 64, 16, n)
    tables = [dev["qo"], dev["indptr"], dev["indices"], dev["last"]]
    lse = torch.empty(n, hq, device="cuda")
    K.paged_prefill(dev["q"], dev["cache"], *tables, out_lse=lse)
    weight = torch.zeros(1, length, device="cuda")
    ws = torch.full((K._prefill_weights_workspace_bytes(hkv, 16, dev["indices"].numel()),), 255, dtype=torch.uint8,
                    device="cuda")
    K.paged_prefill_weights(dev["q"], dev["cache"], *tables, lse, weight, workspace=ws)
    added = o.paged(host["q"], host["cache"], host["qo"], host["indptr"], host["indices"], host["last"], 64 ** -0.5)[2]
    _weights_ok(weight, torch.zeros(1, length), added, [length])


def test_select_of_more_positions_than_shared_memory_holds(K):
    rng = np.random.default_rng(77)
    w = (rng.random((2, 500_000)) ** 6).astype(np.float32)
    w[1, ::2] = 0.5
    weight = torch.as_tensor(w).cuda()
    lens = [500_000, 450_001]
    _check_select(_select(K, weight, lens, 30_000, 7, 1000), weight, lens, 30_000, 7, 1000)
