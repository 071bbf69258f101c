"""The 4-bit cache against the oracle (oracle/small_cache.py).

Records are equal byte for byte (single fp32 operations).  Attention: p and
then p x scale are rounded to bf16 (half a step is 2^-8 relative), the result
too, sums are fp32: with value = minimum + scale code,
|err| <= 2^-8 (|o| + sum p |value| + (1 + 2^-8) sum p scale |code - 8|)
         + 2^-12 sum p (|minimum| + 16 scale); LSE within 2^-12 (1 + |lse|).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import small_cache as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
F = 2.0 ** -12


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64).reshape(-1), dtype=torch.int32, device="cuda")


def _bf16(x):
    return torch.as_tensor(np.asarray(x, np.float32)).to(torch.bfloat16)


@pytest.mark.parametrize("d,ps,hkv,t", [(128, 16, 8, 50), (64, 32, 3, 33), (128, 64, 1, 1), (64, 16, 5, 200)])
def test_append(K, d, ps, hkv, t):
    rng = np.random.default_rng(d + t)
    x = rng.normal(size=(2, t, hkv, d)) * np.exp2(rng.integers(-20, 20, size=(2, t, 1, 1)))
    x[0, 0] = 0.0
    x[1, t // 2] = -1.5          # constant groups
    x[0, t // 3, :, 5] = 3e38    # a difference that fp32 does not hold
    x[0, t // 3, :, 9] = -3e38
    x[1, 0] = rng.normal(size=(hkv, d)) * 2.0 ** -125  # a spread that no scale is given for
    x[1, t - 1] = rng.normal(size=(hkv, d)) * 2.0 ** -110
    xt = _bf16(x)
    wide = torch.zeros(t, 2, hkv * d, dtype=torch.bfloat16, device="cuda")  # strided rows
    wide[:, 0].copy_(xt[0].reshape(t, -1))
    wide[:, 1].copy_(xt[1].reshape(t, -1))
    k, v = wide[:, 0].view(t, hkv, d), wide[:, 1].view(t, hkv, d)
    pages = -(-t // ps) + 3
    slots = rng.permutation(pages * ps)[:t]
    cache = torch.full((pages, 2, ps, hkv, d // 2 + 16), 77, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.kv4_append(k, v, cache, _i32(slots // ps), _i32(slots % ps), status)
    assert int(status.item()) == 0
    got = cache.cpu().numpy()
    want = np.full_like(got, 77)
    for kv in range(2):
        xs = xt[kv].float().numpy()
        rec = o.record_bytes(*o.pack4(xs))
        want[slots // ps, kv, slots % ps] = rec
        val, scale, _ = o.unpack4(rec)
        # Half a code, and 15 codes times the scale's rounding.  A group whose spread / 15 is below 2^-120 has scale 0 and
        # comes back as its minimum: off by its spread at most, which is below 15 * 2^-120.
        assert (np.abs(val - xs) <= scale * (0.5 + 15 * 2.0 ** -9) + 15 * 2.0 ** -120).all()
    assert (got == want).all()
    # expanded: the values, rounded once
    ids = np.concatenate([np.unique(slots // ps)[::-1], [-1]])
    out = torch.full((len(ids), 2, ps, hkv, d), 9.0, dtype=torch.bfloat16, device="cuda")
    K.kv4_expand(cache, _i32(ids), out=out, status=status)
    assert int(status.item()) == 0 and (out[-1] == 9).all()
    val = o.unpack4(got)[0][ids[:-1]]
    written = (want != 77).any(-1)[ids[:-1]]
    have = out[:-1].float().cpu().numpy()
    assert (np.abs(have - val)[written] <= U * np.abs(val)[written] + 1e-38).all()


def test_append_of_inf_and_nan_and_bad_slots(K):
    x = torch.randn(4, 2, 64, dtype=torch.bfloat16)
    x[0, 0, 5] = float("nan")   # group 1
    x[1, 1, 62] = float("inf")  # group 2
    x[2, 0, 0] = float("-inf")  # group 0
    cache = torch.zeros(3, 2, 16, 2, 48, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.kv4_append(x.cuda(), x.cuda(), cache, _i32([1, 1, 1, 1]), _i32([0, 1, 2, 3]), status)
    assert int(status.item()) == 0
    out = torch.empty(1, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    K.kv4_expand(cache, _i32([1]), out=out)
    nan = torch.isnan(out[0, :, :4]).cpu()
    want = torch.zeros_like(nan)
    want[:, 0, 0, 1::4] = want[:, 1, 1, 2::4] = want[:, 2, 0, 0::4] = True
    assert torch.equal(nan, want)
    before = cache.clone()
    K.kv4_append(x.cuda(), x.cuda(), cache, _i32([-1, 3, 0, 0]), _i32([0, 0, 16, -1]), status)
    assert int(status.item()) == 3 and torch.equal(cache, before)
    status.zero_()
    K.kv4_expand(cache, _i32([7]), out=out, status=status)
    assert int(status.item()) == 3


def _case(lens, hq, hkv, d, ps, seed, edit=None):
    rng = np.random.default_rng(seed)
    pages = [-(-x // ps) for x in lens]
    pool = sum(pages) + 4
    x = rng.normal(size=(pool, 2, ps, hkv, d)) * rng.choice([0.5, 1, 3], size=(hkv, d)) + rng.normal(size=(hkv, d))
    rec = o.record_bytes(*o.pack4(_bf16(x).float().numpy()))
    perm = rng.permutation(pool)
    indptr = np.cumsum([0] + pages)
    last = [n - (k - 1) * ps if k else 0 for n, k in zip(lens, pages)]
    indices = perm[: sum(pages)].copy()
    for b, k in enumerate(pages):
        if k:  # slots past the last token: codes of ones, scales and minima of NaN
            rec[indices[indptr[b + 1] - 1], :, last[b]:] = 255
    q = rng.normal(size=(len(lens), hq, d)).astype(np.float32)
    if edit is not None:
        edit(q, rec, indptr, indices)
    qt = _bf16(q)
    host = dict(q=qt.float().numpy(), rec=rec, indptr=indptr, indices=indices, last=last)
    dev = dict(q=qt.cuda(), cache=torch.as_tensor(rec).cuda(), indptr=_i32(indptr), indices=_i32(indices),
               last=_i32(last))
    return host, dev


def _run(K, dev, want=0, **kw):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full(dev["q"].shape[:2], 7.0, device="cuda")
    out = K.paged_kv4_decode(dev["q"], dev["cache"], dev["indptr"], dev["indices"], dev["last"], out_lse=lse,
                             status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == want
    return out, lse


def _check(out, lse, host, window=None, sinks=0):
    val, scale, code = o.unpack4(host["rec"])
    rows, hq, d = host["q"].shape
    group = hq // val.shape[3]
    got, glse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    for b in range(rows):
        lo, hi, last = host["indptr"][b], host["indptr"][b + 1], host["last"][b]
        k, v = o.row_tokens(val, host["indices"], lo, hi, last)
        _, sc = o.row_tokens(scale, host["indices"], lo, hi, last)
        _, cd = o.row_tokens(code, host["indices"], lo, hi, last)
        see = o.visible(len(k) - 1, len(k), window, sinks)
        want, wlse, p, spread = o.attend(host["q"][b], k, v, see, d ** -0.5)
        v, sc, cd, p = v[see], sc[see], cd[see], p[:, see]
        for h in range(hq):
            x = h // group
            codes = p[h] @ (sc[:, x] * np.abs(cd[:, x]))
            parts = p[h] @ (np.abs(v[:, x] - sc[:, x] * (cd[:, x] + 8)) + 16 * sc[:, x])
            tol = U * (np.abs(want[h]) + spread[h] + (1 + U) * codes) + F * parts + 1e-30
            err = np.abs(got[b, h] - want[h])
            assert (err <= tol).all(), (b, h, (err / tol).max())
        empty = np.isneginf(wlse)
        assert (np.isneginf(glse[b]) == empty).all()
        assert (np.abs(np.where(empty, 0, glse[b] - np.where(empty, 0, wlse))) <=
                F * (1 + np.abs(np.where(empty, 0, wlse)))).all()


LENS = [1, 16, 17, 0, 300, 1200, 161, 700]


@pytest.mark.parametrize("hq,hkv,d,ps", [(32, 8, 128, 16), (8, 8, 64, 32), (28, 4, 128, 64), (16, 1, 64, 128),
                                         (10, 5, 128, 16), (9, 1, 128, 32), (12, 12, 64, 16), (36, 9, 128, 16),
                                         (14, 2, 64, 16), (32, 2, 128, 16), (3, 3, 128, 16), (20, 20, 128, 16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (130, 5)])
def test_decode(K, hq, hkv, d, ps, window, sinks):
    host, dev = _case(LENS, hq, hkv, d, ps, hq + ps)
    _check(*_run(K, dev, window=window, sinks=sinks), host, window, sinks)


def test_decode_of_long_and_many_rows(K):
    host, dev = _case([20011, 3, 4999], 8, 2, 128, 16, 2)
    _check(*_run(K, dev), host)
    rng = np.random.default_rng(8)
    host, dev = _case(list(rng.integers(0, 40, 300)), 4, 4, 64, 16, 3)
    _check(*_run(K, dev), host)


def test_hidden_nan_stays_out_and_seen_nan_gets_in(K):
    def edit(q, rec, indptr, indices):
        for pos in range(4, 60):  # scales and minima of NaN in pages that are read
            rec[indices[pos // 16], :, pos % 16, :, -16:] = 255
        indices[indptr[1] + 1: indptr[1] + 3] = -9

    host, dev = _case([100, 100], 8, 2, 128, 16, 4, edit)
    host["indices"] = np.where(host["indices"] < 0, 0, host["indices"])
    _check(*_run(K, dev, window=40, sinks=4), host, 40, 4)

    def one(q, rec, indptr, indices):
        rec[indices[2], 1, 5, 0, -8:-6] = 255  # V's first minimum of one token: group 0
        q[1, 3] = np.nan

    host, dev = _case([100, 100], 8, 2, 128, 16, 5, one)
    out, _ = _run(K, dev)
    nan = torch.isnan(out).cpu()
    want = torch.zeros_like(nan)
    want[0, :4, 0::4] = True
    want[1, 3] = True
    assert torch.equal(nan, want)


def test_large_and_small_values(K):
    def edit(q, rec, indptr, indices):
        q *= 30
        q[1] *= 1e-6

    host, dev = _case([500, 90], 8, 8, 128, 16, 6, edit)
    _check(*_run(K, dev), host)
    rng = np.random.default_rng(1)
    for size in (1e-4, 1e6):
        x = _bf16(rng.normal(size=(9, 2, 16, 2, 64)) * size).float().numpy()
        host, dev = _case([140], 4, 2, 64, 16, 7)
        rec = o.record_bytes(*o.pack4(x[: len(host["rec"])]))
        host["rec"] = np.concatenate([rec, host["rec"][len(rec):]])
        host["q"] = _bf16(host["q"] / size).float().numpy()
        dev.update(cache=torch.as_tensor(host["rec"]).cuda(), q=_bf16(host["q"]).cuda())
        host["indices"][:] = np.arange(9)
        dev["indices"] = _i32(host["indices"])
        _check(*_run(K, dev), host)


def test_strides_streams_graphs_and_status(K):
    host, dev = _case([900, 33, 0, 2048], 8, 2, 128, 16, 14)
    want, wlse = _run(K, dev)
    wide = torch.empty(4, 3, 8, 192, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 1, :, 32:160]
    q.copy_(dev["q"])
    out = torch.full((4, 8, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((K._kv4_decode_workspace_bytes(8, 2, 128),), 255, dtype=torch.uint8, device="cuda")
    args = (q, dev["cache"], dev["indptr"], dev["indices"], dev["last"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.paged_kv4_decode(*args, out=out[:, :, 64:192], workspace=ws)
    side.synchronize()
    assert torch.equal(out[:, :, 64:192], want) and (out[:, :, :64] == 5).all() and (out[:, :, 192:] == 5).all()
    got, lse = torch.empty_like(want), torch.empty_like(wlse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.paged_kv4_decode(*args, out=got, out_lse=lse, workspace=ws)
    for _ in range(2):
        got.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, wlse)
    bad = dict(dev, indices=dev["indices"].clone())
    bad["indices"][3] = -1
    out, _ = _run(K, bad, want=3)
    assert torch.equal(out[1:], want[1:])
    bad = dict(dev, indptr=_i32([0, 57, 60, 60, 999]))
    out, lse = _run(K, bad, want=1)
    assert torch.equal(out[:3], want[:3]) and (out[3] == 0).all() and torch.isneginf(lse[3]).all()


def test_pages_move_like_any_others(K):
    """Append, fork, reserve, append, compact and decode over one 4-bit pool of two layers."""

    rng = np.random.default_rng(31)
    layers, pool, ps, hkv, d, rows, cap = 2, 40, 16, 2, 64, 4, 9
    cache = torch.zeros(layers, pool, 2, ps, hkv, d // 2 + 16, dtype=torch.uint8, device="cuda")
    ref = np.zeros((layers, rows, cap * ps, 2, hkv, d))
    count = torch.zeros(pool, dtype=torch.int32, device="cuda")
    table = torch.zeros(rows, cap, dtype=torch.int32, device="cuda")
    num, last = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    lens = [0] * rows
    indptr, indices = _i32([0] * (rows + 1)), _i32([0] * rows * cap)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def grow(n):
        t = sum(n)
        page, off = _i32([0] * t), _i32([0] * t)
        K.page_reserve(count, table, num, last, _i32(np.cumsum([0] + n)), ps, slot_page=page, slot_offset=off,
                       out_indptr=indptr, out_indices=indices, status=status)
        for li in range(layers):
            x = _bf16(rng.normal(size=(t, 2, hkv, d)))
            K.kv4_append(x[:, 0].contiguous().cuda(), x[:, 1].contiguous().cuda(), cache[li], page, off, status)
            xs, at = x.float().numpy(), 0
            for r, k in enumerate(n):
                ref[li, r, lens[r]:lens[r] + k] = o.unpack4(o.record_bytes(*o.pack4(xs[at:at + k])))[0]
                at += k
        for r, k in enumerate(n):
            lens[r] += k

    grow([40, 0, 21, 0])
    K.page_fork(cache, count, table, num, last, _i32([0]), _i32([3]), status=status)
    ref[:, 3], lens[3] = ref[:, 0], lens[0]
    grow([3, 5, 0, 30])
    keep = [[41, 42], [4], [3, 9, 20], list(range(30, 70, 3))]
    kf = [7, 0, 1, 20]
    mat = np.full((rows, 16), -1)
    for r, k in enumerate(keep):
        mat[r, :len(k)] = k
        ref[:, r, :kf[r] + len(k)] = ref[:, r, list(range(kf[r])) + k]
        lens[r] = kf[r] + len(k)
    K.cache_compact(cache, count, table, num, last, _i32(kf), torch.as_tensor(mat, dtype=torch.int32).cuda(),
                    _i32([len(k) for k in keep]), status=status)
    grow([1, 1, 1, 1])
    assert int(status.item()) == 0
    q = torch.randn(rows, 4, d, dtype=torch.bfloat16, device="cuda")
    tables = dict(indptr=indptr.cpu().numpy(), indices=indices.cpu().numpy(), last=last.cpu().numpy())
    for li in range(layers):
        host = dict(tables, q=q.float().cpu().numpy(), rec=cache[li].cpu().numpy())
        val = o.unpack4(host["rec"])[0]
        for r in range(rows):
            k, v = o.row_tokens(val, tables["indices"], tables["indptr"][r], tables["indptr"][r + 1], tables["last"][r])
            assert (np.stack([k, v], 1) == ref[li, r, :lens[r]]).all()
        _check(*_run(K, dict(q=q, cache=cache[li], indptr=indptr, indices=indices, last=last)), host)
