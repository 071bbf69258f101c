"""How near the 4-bit decode is, and a prompt's attention over a 4-bit cache.

Tight bound: p is rounded to bf16 (half a step is 2^-8 relative) and enters
all sums of a position alike, p x scale as a bf16 value and its exact
remainder, the result is rounded, sums are fp32: with value = minimum + scale
code, |err| <= 2^-8 (|o| + sum p |value|) + 2^-12 sum p (|minimum| + 16 scale).
(test_gpu_kv4_cache.py's bound also has room for a rounded p x scale.)
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import small_cache as o
from tests.test_gpu_kv4_cache import LENS, _bf16, _case, _i32, _run

U, F = 2.0 ** -8, 2.0 ** -12


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _bounds(q, val, scale, code, scale_qk):
    """(o, bound) [Hq, D] of one query over all positions."""

    n, hkv, d = val[0].shape
    want, _, p, spread = o.attend(q, *val, np.ones(n, bool), scale_qk)
    group = q.shape[0] // hkv
    parts = np.stack([p[h] @ (np.abs(val[1][:, h // group] - scale[:, h // group] * (code[:, h // group] + 8)) +
                              16 * scale[:, h // group]) for h in range(q.shape[0])])
    return want, U * (np.abs(want) + spread) + F * parts, p


def _tight(out, host, ulp=1e-30):
    val, scale, code = o.unpack4(host["rec"])
    got = out.double().cpu().numpy()
    for b in range(len(host["q"])):
        at = (host["indices"], host["indptr"][b], host["indptr"][b + 1], host["last"][b])
        kv = tuple(o.row_tokens(val, *at))
        if len(kv[0]) == 0:
            continue
        want, tol, _ = _bounds(host["q"][b], kv, list(o.row_tokens(scale, *at))[1], list(o.row_tokens(code, *at))[1],
                               host["q"].shape[2] ** -0.5)
        err = np.abs(got[b] - want)
        assert (err <= tol + ulp).all(), (b, (err / (tol + ulp)).max())


def _outliers(rng, n, hkv, d):
    """K and V [n, 2, hkv, d] whose V groups have one large channel each: scale x code far above most values."""

    x = rng.normal(size=(n, 2, hkv, d))
    x[:, 1] *= 0.01
    x[:, 1, :, 20:24] = 40 + rng.normal(size=(n, hkv, 4))
    return _bf16(x).float().numpy()


def _outlier_case(lens, hq, hkv, d, seed):
    host, dev = _case(lens, hq, hkv, d, 16, seed)
    rng = np.random.default_rng(seed)
    rec = host["rec"]
    for b, n in enumerate(lens):
        x = _outliers(rng, n, hkv, d)
        pos = np.arange(n)
        rec[host["indices"][host["indptr"][b] + pos // 16], :, pos % 16] = o.record_bytes(*o.pack4(x))
    dev["cache"] = torch.as_tensor(rec).cuda()
    return host, dev


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,ps", [(32, 8, 128, 16), (8, 8, 64, 32), (16, 1, 64, 128), (10, 5, 128, 16), (3, 3, 128, 16)])
def test_decode(K, hq, hkv, d, ps):
    host, dev = _case(LENS, hq, hkv, d, ps, hq + ps)
    _tight(_run(K, dev)[0], host)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (12, 1, 128)])
def test_decode_of_groups_with_one_large_channel(K, hq, hkv, d):
    host, dev = _outlier_case([2, 3, 5, 7, 11, 40], hq, hkv, d, hq)
    _tight(_run(K, dev)[0], host)


def test_the_bound_tells_a_rounded_product_from_an_exact_one():
    """Without a GPU: p x scale rounded to bf16 leaves the tight bound on such rows, the exact product stays within it."""

    rng = np.random.default_rng(3)
    beyond = 0
    for n in (3, 5, 7, 11) * 8:
        x = _outliers(rng, n, 1, 64)
        val, scale, code = o.unpack4(o.record_bytes(*o.pack4(x)))
        q = _bf16(rng.normal(size=(1, 64))).float().numpy()
        want, tol, p = _bounds(q, (val[:, 0], val[:, 1]), scale[:, 1], code[:, 1], 0.125)
        e = o.to_bf16(p[0] / p[0].max()).astype(np.float64)  # what the tensor core takes
        total = (p[0] / p[0].max()).sum()
        s, c, low = scale[:, 1, 0], code[:, 1, 0], val[:, 1, 0] - scale[:, 1, 0] * (code[:, 1, 0] + 8)
        rest = e @ low + 8 * (e @ s)
        exact = (((e[:, None] * s) * c).sum(0) + rest) / total
        rounded = ((o.to_bf16(e[:, None] * s).astype(np.float64) * c).sum(0) + rest) / total
        assert (np.abs(exact - want[0]) <= tol[0]).all()
        beyond += (np.abs(rounded - want[0]) > tol[0]).any()
    assert beyond >= 16


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** 40])
def test_the_range_of_values(K, size):
    """V's values times their number within 2^55, down to 2^-30: sums carry 2^-73 of what they stand for, so their
    subnormals are absolute steps of 2^-76; K's size is q's to undo."""

    rng = np.random.default_rng(5)
    x = _bf16(rng.normal(size=(9, 2, 16, 2, 64)) * size).float().numpy()
    host, dev = _case([140], 4, 2, 64, 16, 7)
    host["rec"] = o.record_bytes(*o.pack4(x))
    host["q"] = _bf16(rng.normal(size=(1, 4, 64)) / size).float().numpy()
    host["indices"] = np.arange(9)
    dev.update(cache=torch.as_tensor(host["rec"]).cuda(), q=_bf16(host["q"]).cuda(), indices=_i32(host["indices"]))
    _tight(_run(K, dev)[0], host, 140 * 2.0 ** -76)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 30])
def test_a_prompt_over_a_4_bit_cache(K, window):
    """Chunks of a prompt: quantised, expanded, and attended to over the expanded pages, then a decode step over the records."""

    rng = np.random.default_rng(19)
    ps, hq, hkv, d, chunks = 16, 8, 2, 64, [50, 1, 37, 90]
    pages = -(-sum(chunks) // ps)
    ids = rng.permutation(pages + 3)[:pages]
    cache = torch.zeros(pages + 3, 2, ps, hkv, d // 2 + 16, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    n, stored = 0, np.zeros((0, 2, hkv, d))
    for c in chunks:
        x = _bf16(rng.normal(size=(c, 2, hkv, d)))
        at = np.arange(n, n + c)
        K.kv4_append(x[:, 0].contiguous().cuda(), x[:, 1].contiguous().cuda(), cache, _i32(ids[at // ps]), _i32(at % ps),
                     status)
        val = o.unpack4(o.record_bytes(*o.pack4(x.float().numpy())))[0]
        stored = np.concatenate([stored, val])
        n += c
        held = -(-n // ps)
        pool = torch.full((held, 2, ps, hkv, d), float("nan"), dtype=torch.bfloat16, device="cuda")
        K.kv4_expand(cache, _i32(ids[:held]), out=pool, status=status)
        q = _bf16(rng.normal(size=(c, hq, d)))
        table = (_i32([0, c]), _i32([0, held]), _i32(range(held)), _i32([n - (held - 1) * ps]))
        if window is None:
            out = K.paged_prefill(q.cuda(), pool, *table, status=status)
        else:
            out = K.paged_window_prefill(q.cuda(), pool, *table, window=window, sinks=3, status=status)
        assert int(status.item()) == 0
        kv = _bf16(stored).double().numpy()  # the expanded values, rounded once
        for i in range(c):
            see = o.visible(n - c + i, n, window, 3)
            want, _, _, spread = o.attend(q[i].double().numpy(), kv[:, 0], kv[:, 1], see, d ** -0.5)
            err = np.abs(out[i].double().cpu().numpy() - want)
            assert (err <= U * (np.abs(want) + spread) + F * spread).all(), i
    host = dict(q=q[-1:].float().numpy(), rec=cache.cpu().numpy(), indptr=np.array([0, pages]), indices=ids, last=[n - (pages - 1) * ps])
    if window is None:
        dev = dict(q=q[-1:].cuda(), cache=cache, indptr=_i32([0, pages]), indices=_i32(ids), last=_i32(host["last"]))
        _tight(_run(K, dev)[0], host)


@pytest.mark.gpu
def test_values_below_the_range_of_the_sums(K):
    """All of V is below 2^-53 in size: O is exact to a step of 2^-76 for each of its sums' terms."""

    rng = np.random.default_rng(6)
    x = _bf16(rng.normal(size=(9, 2, 16, 2, 64)) * 2.0 ** -58).float().numpy()
    host, dev = _case([140], 4, 2, 64, 16, 7)
    host["rec"] = o.record_bytes(*o.pack4(x))
    host["indices"] = np.arange(9)
    dev.update(cache=torch.as_tensor(host["rec"]).cuda(), indices=_i32(host["indices"]))
    _tight(_run(K, dev)[0], host, 140 * 2.0 ** -76)
