"""Drafted-token trees on the device: mask, acceptance and attention against
the 64-bit oracle (oracle/tree_attention.py).

Tolerance of the attention, element by element: P is rounded to bf16 as a
tensor-core operand and the result to bf16, each by at most 2^-8 relative
(8 significant bits), so |err| <= 2^-8 (|o| + sum p |v|); fp32 scores of up
to 128 products leave a relative error below 2^-12 in p.  LSE: the same 2^-12
in the sum, and 2^-12 of its size for the fp32 scores.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import tree_attention as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
F = 2.0 ** -12


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64), dtype=torch.int32, device="cuda")


def _tree(rng, n):
    return [-1 if i == 0 or rng.random() < 0.1 else int(rng.integers(max(0, i - 5), i)) for i in range(n)]


def _case(reqs, hq, hkv, d, ps, seed, see=None, kv_fix=None):
    """reqs: (drafted, context) tokens per request.  The pool is NaN wherever no request's token sits."""

    rng = np.random.default_rng(seed)
    lens = [n + c for n, c in reqs]
    n_pages = [-(-x // ps) for x in lens]
    total = sum(n_pages) + 3
    perm = rng.permutation(total)
    cache = np.full((total, 2, ps, hkv, d), np.nan, np.float32)
    kv_indptr, kv_indices, last, at = [0], [], [], 0
    for x, n in zip(lens, n_pages):
        pages = [int(p) for p in perm[at:at + n]]
        at += n
        kv_indices += pages
        kv_indptr.append(len(kv_indices))
        last.append(x - (n - 1) * ps if n else 0)
        for t in range(x):
            cache[pages[t // ps], :, t % ps] = rng.normal(size=(2, hkv, d))
    qo = np.cumsum([0] + [n for n, _ in reqs]).tolist()
    q = rng.normal(size=(qo[-1], hq, d)).astype(np.float32) * 1.5
    trees = [_tree(rng, n) for n, _ in reqs]
    if see is None:
        see = [o.ancestors(t) for t in trees]
    host = dict(qo=qo, kv_indptr=kv_indptr, kv_indices=kv_indices, last=last, see=see, trees=trees, ps=ps, lens=lens)
    if kv_fix is not None:
        kv_fix(cache, host)
    ct, qt = torch.as_tensor(cache).to(torch.bfloat16), torch.as_tensor(q).to(torch.bfloat16)
    host.update(cache=ct.double().numpy(), q=qt.double().numpy())
    words = max(1, -(-max(n for n, _ in reqs) // 32))
    mask = np.concatenate([o.pack_bits(m, words) for m in see]) if qo[-1] else np.zeros((0, words), np.int32)
    dev = dict(q=qt.cuda(), cache=ct.cuda(), qo=_i32(qo), kv_indptr=_i32(kv_indptr), kv_indices=_i32(kv_indices or [0]),
               last=_i32(last), mask=torch.as_tensor(mask).cuda())
    return host, dev


def _run(K, dev, want_status=0, **kw):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full(dev["q"].shape[:2], 7.0, device="cuda")
    out = K.paged_tree_attention(dev["q"], dev["cache"], dev["qo"], dev["kv_indptr"], dev["kv_indices"], dev["last"],
                                 dev["mask"], out_lse=lse, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status.item()) == want_status
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


def _check(got, host, rows=slice(None)):
    want, wlse, spread = o.tree_attention(host["q"], host["cache"], host["qo"], host["kv_indptr"], host["kv_indices"],
                                          host["last"], host["see"])
    out, lse = got
    tol = U * (np.abs(want) + spread) + F * spread + 1e-30
    err = np.abs(out - want)
    assert (err[rows] <= tol[rows]).all(), (err - tol)[rows].max()
    empty = np.isinf(wlse)
    assert (np.isneginf(lse) == empty)[rows].all()
    lerr = np.abs(np.where(empty, 0, lse) - np.where(empty, 0, wlse))
    assert (lerr[rows] <= (F * (1 + np.abs(np.where(empty, 0, wlse))))[rows]).all(), lerr[rows].max()


REQS = [(1, 0), (5, 37), (33, 300), (1, 1), (0, 50), (8, 128), (7, 121), (2, 1000)]


@pytest.mark.parametrize("d,ps", [(128, 16), (64, 32), (128, 64), (64, 128)])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (4, 4), (28, 4), (16, 1)])
def test_matches_oracle(K, d, ps, hq, hkv):
    host, dev = _case(REQS, hq, hkv, d, ps, seed=hq + d + ps)
    _check(_run(K, dev), host)


@pytest.mark.parametrize("reqs,hq,hkv", [
    ([(70, 500)], 8, 2),                    # 280 rows of a kv head: two tiles, twice
    ([(129, 3), (1, 900), (64, 64)], 4, 2),  # ragged, the mean just below / above a tile
    ([(300, 10)], 2, 1),                    # a mask of ten words
    ([(3, 20000)], 2, 1),                   # one long item over many CTAs
    ([(17, 5000), (1, 1), (2, 7000)], 4, 1),
    ([(1, 15), (1, 16), (1, 17), (1, 127), (1, 128), (1, 255), (1, 256)], 4, 4),
])
def test_sizes(K, reqs, hq, hkv):
    host, dev = _case(reqs, hq, hkv, 128, 16, seed=len(reqs))
    _check(_run(K, dev), host)


def test_many_requests(K):
    reqs = [(int(n), int(c)) for n, c in np.random.default_rng(3).integers(0, [4, 200], size=(150, 2))]
    host, dev = _case(reqs, 4, 2, 64, 16, seed=9)
    _check(_run(K, dev), host)


def test_arbitrary_masks_and_empty_rows(K):
    """Any bits, a row that sees nothing (no context), bits behind the request's tokens."""

    rng = np.random.default_rng(5)
    reqs = [(40, 0), (40, 100), (9, 0)]
    see = [rng.random((n, n)) < 0.4 for n, _ in reqs]
    see[0][3] = False
    see[1][0] = False
    see[2][:] = False
    host, dev = _case(reqs, 8, 2, 128, 16, seed=6, see=see)
    dev["mask"] |= torch.tensor([0, -(1 << 31)], dtype=torch.int32, device="cuda")  # bit 63
    out, lse = _run(K, dev)
    _check((out, lse), host)
    assert (out[3] == 0).all() and np.isneginf(lse[3]).all() and (out[80:] == 0).all()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("ctx", [100, 3000])
@pytest.mark.parametrize("which", [0, 1])
def test_inf_and_nan_stay_with_the_rows_that_see_them(K, value, ctx, which):
    """Token 2's K (which = 0) or V (1) holds inf / NaN; rows that mask it are as without it."""

    n = 6
    see = [np.tril(np.ones((n, n), bool))]
    see[0][3:, 2] = False
    see[0][5, 2] = True

    def fix(cache, host):
        pos = ctx + 2
        page = host["kv_indices"][pos // host["ps"]]
        cache[page, which, pos % host["ps"], :, 5] = value

    host, dev = _case([(n, ctx)], 4, 2, 128, 16, seed=1, see=see, kv_fix=fix)
    out, lse = _run(K, dev)
    clean = dict(host, cache=np.nan_to_num(host["cache"], nan=0.0, posinf=0.0, neginf=0.0))
    rows = [0, 1, 3, 4]
    _check((out, lse), clean, rows)
    hit = out[[2, 5]]
    if which == 1:
        assert not np.isfinite(hit[..., 5]).any()
        same = np.isnan(hit[..., 5]) if np.isnan(value) else hit[..., 5] == value
        assert same.all()
        assert np.isfinite(np.delete(hit, 5, axis=-1)).all()
    elif np.isnan(value):
        assert np.isnan(hit).all()


# Requests whose mean fills an even number of 128-row tiles (two per CTA), beside ones that leave a tile or
# a half of it empty, and without a context or without drafts.
WIDE = [
    ([(64, 500)], 8, 2),
    ([(96, 40), (1, 0), (80, 2000), (40, 300)], 8, 2),
    ([(200, 3), (0, 77), (256, 900), (60, 129)], 2, 2),
    ([(37, 700), (33, 0)], 14, 2),
    ([(130, 1000)], 12, 4),
    ([(1, 5000), (70, 10), (20, 128), (33, 127)], 32, 2),
]


@pytest.mark.parametrize("d,ps", [(128, 16), (64, 16), (128, 128)])
@pytest.mark.parametrize("reqs,hq,hkv", WIDE)
def test_two_row_tiles(K, reqs, hq, hkv, d, ps):
    mean = -(-sum(n for n, _ in reqs) * (hq // hkv) // (128 * len(reqs)))
    assert mean % 2 == 0
    host, dev = _case(reqs, hq, hkv, d, ps, seed=len(reqs) + d)
    _check(_run(K, dev), host)


@pytest.mark.parametrize("value", [np.nan, -np.inf])
@pytest.mark.parametrize("which", [0, 1])
def test_two_row_tiles_masks_inf_and_nan(K, value, which):
    """As above with any bits, rows that see nothing, and a drafted token that only some rows see."""

    rng = np.random.default_rng(12)
    n, ctx = 72, 200
    see = [rng.random((n, n)) < 0.4, rng.random((n, n)) < 0.4]
    see[1][5] = False
    see[1][70] = False
    hit = np.flatnonzero(see[0][:, 9])

    def fix(cache, host):
        pos = ctx + 9
        cache[host["kv_indices"][pos // host["ps"]], which, pos % host["ps"], :, 5] = value

    host, dev = _case([(n, ctx), (n, 0)], 8, 2, 128, 16, seed=2, see=see, kv_fix=fix)
    out, lse = _run(K, dev)
    clean = dict(host, cache=np.nan_to_num(host["cache"], nan=0.0, posinf=0.0, neginf=0.0))
    _check((out, lse), clean, np.setdiff1d(np.arange(2 * n), hit))
    assert (out[n + 5] == 0).all() and np.isneginf(lse[n + 70]).all()
    if which == 1:
        assert not np.isfinite(out[hit][..., 5]).any() and np.isfinite(np.delete(out[hit], 5, axis=-1)).all()
    elif np.isnan(value):
        assert np.isnan(out[hit]).all()


@pytest.mark.parametrize("n", [5, 40, 64])
def test_growing_maxima(K, n):
    """Scores whose maximum grows by more than 2^8 from tile to tile, not always in order.  A channel adds up to
    43 to the scores: their fp32 error is at most 128 * 2^-24 * (43 + sum |q k| of the others, about 11)
    < 2^-11, in place of 2^-12."""

    level = [0, 5, 10, 5, 15, 0, 20, 30, 20, 30, 1]

    def fix(cache, host):
        for t in range(host["lens"][0]):
            cache[host["kv_indices"][t // host["ps"]], 0, t % host["ps"], :, 0] = level[t // 128]

    host, dev = _case([(n, 128 * len(level) - n - 20)], 8, 2, 128, 16, seed=n, kv_fix=fix)
    host["q"][..., 0] = 16.0
    dev["q"][..., 0] = 16.0
    out, lse = _run(K, dev)
    want, wlse, spread = o.tree_attention(host["q"], host["cache"], host["qo"], host["kv_indptr"], host["kv_indices"],
                                          host["last"], host["see"])
    assert (np.abs(out - want) <= U * (np.abs(want) + spread) + 2 * F * spread).all()
    assert (np.abs(lse - wlse) <= 2 * F * (1 + np.abs(wlse))).all()


def test_strides_scale_and_streams(K):
    host, dev = _case([(12, 90), (3, 400)], 8, 2, 128, 16, seed=11)
    total = host["qo"][-1]
    packed = torch.full((total, 16, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    packed[:, 2:10] = dev["q"]
    dev["q"] = packed[:, 2:10]
    wide = torch.zeros(total, 5, dtype=torch.int32, device="cuda")
    wide[:, :1] = dev["mask"]
    dev["mask"] = wide[:, :1]
    out = torch.full((8, total, 128), 3.0, dtype=torch.bfloat16, device="cuda").permute(1, 0, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(K, dev, out=out)
    _check(got, host)


def test_long_pool_offsets(K):
    """Page ids whose element offset is past 2^31 (and byte offset past 2^32)."""

    ps, hkv, d, n, ctx = 16, 8, 128, 4, 300
    host, dev = _case([(n, ctx)], 8, hkv, d, ps, seed=2)
    pages = (1 << 31) // (2 * ps * hkv * d) + 64
    big = torch.empty(pages, 2, ps, hkv, d, dtype=torch.bfloat16, device="cuda")
    used = torch.tensor(host["kv_indices"], device="cuda")
    to = pages - 1 - torch.arange(len(used), device="cuda")
    big[to] = dev["cache"][used]
    dev["cache"], dev["kv_indices"] = big, to.to(torch.int32)
    _check(_run(K, dev), host)


def test_graph_replay_repeats(K):
    host, dev = _case([(9, 700), (5, 30)], 8, 2, 128, 16, seed=21)
    out, lse = torch.empty_like(dev["q"]), torch.empty(dev["q"].shape[:2], device="cuda")
    ws = torch.empty(K.tree_workspace_bytes(2, 14, 8, 2, 128), dtype=torch.uint8, device="cuda")
    args = (dev["q"], dev["cache"], dev["qo"], dev["kv_indptr"], dev["kv_indices"], dev["last"], dev["mask"])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        K.paged_tree_attention(*args, out=out, out_lse=lse, workspace=ws)
    torch.cuda.synchronize()
    first = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        K.paged_tree_attention(*args, out=out, out_lse=lse, workspace=ws)
    for _ in range(3):
        out.zero_()
        ws.fill_(255)  # the workspace needs no initialisation
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    _check((out.double().cpu().numpy(), lse.double().cpu().numpy()), host)


def test_one_token_equals_decode(K):
    """A tree of one token is a decode step."""

    host, dev = _case([(1, 700), (1, 16), (1, 0)], 8, 2, 128, 16, seed=8)
    out, _ = _run(K, dev)
    ref = K.paged_decode(dev["q"], dev["cache"], dev["kv_indptr"], dev["kv_indices"], dev["last"], num_splits=1,
                         workspace=torch.zeros(4096, dtype=torch.uint8, device="cuda"))
    _, _, spread = o.tree_attention(host["q"], host["cache"], host["qo"], host["kv_indptr"], host["kv_indices"],
                                    host["last"], host["see"])
    assert (np.abs(out - ref.double().cpu().numpy()) <= 2 * (2 * U + F) * spread).all()


def test_device_refusals(K):
    from pagelora_b200 import _capi

    host, dev = _case([(5, 40)], 8, 2, 128, 16, seed=4)
    # more drafted tokens than cached ones
    short = dict(dev, kv_indptr=_i32([0, 1]), last=_i32([2]))
    _run(K, short, want_status=_capi.PL_ERR_INVALID_ARGUMENT)
    # a table that leaves kv_indices
    _run(K, dict(dev, kv_indptr=_i32([0, 99])), want_status=_capi.PL_ERR_INVALID_ARGUMENT)
    # a page outside the pool: its tokens read as zeros, nothing else is touched
    bad = dev["kv_indices"].clone()
    bad[1] = 10 ** 6
    _run(K, dict(dev, kv_indices=bad), want_status=_capi.PL_ERR_PAGE_OUT_OF_RANGE)


def test_host_refusals(K):
    host, dev = _case([(5, 40)], 8, 2, 128, 16, seed=4)
    args = [dev[k] for k in ("q", "cache", "qo", "kv_indptr", "kv_indices", "last", "mask")]

    def call(i, t, **kw):
        K.paged_tree_attention(*[t if j == i else a for j, a in enumerate(args)], **kw)

    with pytest.raises(TypeError):
        call(0, args[0].half())
    with pytest.raises(TypeError):
        call(6, args[6].long())
    with pytest.raises(ValueError):
        call(6, args[6][:2])
    with pytest.raises(ValueError):
        call(1, args[1].transpose(0, 1))
    with pytest.raises(RuntimeError):
        call(0, args[0].cpu())
    with pytest.raises(RuntimeError, match="unsupported"):
        call(1, torch.zeros(4, 2, 24, 2, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="workspace"):
        call(4, torch.zeros(64, dtype=torch.int32, device="cuda"),
             workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="invalid"):
        call(0, args[0], sm_scale=-1.0)


# ------------------------------------------------------- mask and acceptance
@pytest.mark.parametrize("sizes", [[1], [0, 5, 33, 1, 64], [200, 3], [1024, 0]])
def test_tree_mask(K, sizes):
    rng = np.random.default_rng(len(sizes))
    trees = [_tree(rng, n) for n in sizes]
    if sizes[0] == 1024:
        trees[0] = list(range(-1, 1023))  # one chain
    words = max(1, -(-max(sizes) // 32))
    qo, base = _i32(np.cumsum([0] + sizes)), _i32(rng.integers(0, 5000, len(sizes)))
    total = sum(sizes)
    pos = torch.empty(total, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    mask, depth = K.tree_mask(_i32(sum(trees, [])), qo, words, base_positions=base, positions=pos, status=status)
    see = [o.ancestors(t) for t in trees]
    want = np.concatenate([o.pack_bits(m, words) for m in see if len(m)])
    assert int(status.item()) == 0
    assert (mask.cpu().numpy() == want).all()
    wd = np.concatenate([m.sum(1) - 1 for m in see])
    assert (depth.cpu().numpy() == wd).all()
    assert (pos.cpu().numpy() == wd + np.repeat(base.cpu().numpy(), sizes)).all()


def test_tree_mask_refusals(K):
    from pagelora_b200 import _capi

    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.tree_mask(_i32([-1, 2, 0]), _i32([0, 3]), 1, status=status)  # a child in front of its parent
    assert int(status.item()) == _capi.PL_ERR_INVALID_ARGUMENT
    status.zero_()
    K.tree_mask(_i32([-1] * 40), _i32([0, 40]), 1, status=status)  # 40 tokens in one word
    assert int(status.item()) == _capi.PL_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError):
        K.tree_mask(_i32([-1]), _i32([0, 1]), 0)
    with pytest.raises(TypeError):
        K.tree_mask(_i32([-1]).long(), _i32([0, 1]), 1)


@pytest.mark.parametrize("agree", [0.0, 0.6, 1.0])
def test_tree_accept(K, agree):
    rng = np.random.default_rng(int(10 * agree))
    sizes = [1, 0, 7, 64, 33, 2, 300]
    trees = [_tree(rng, n) for n in sizes]
    targets = [rng.integers(0, 50, n) for n in sizes]
    tokens = [rng.integers(50, 99, n) for n in sizes]
    for t, tok, tgt in zip(trees, tokens, targets):
        for i, p in enumerate(t):
            if p >= 0 and rng.random() < agree:
                tok[i] = tgt[p]
    base = rng.integers(0, 900, len(sizes))
    width = 300
    keep = torch.full((len(sizes), width), 5, dtype=torch.int32, device="cuda")
    count = torch.zeros(len(sizes), dtype=torch.int32, device="cuda")
    nxt = torch.zeros(len(sizes), dtype=torch.int64, device="cuda")
    K.tree_accept(_i32(sum(trees, [])), torch.as_tensor(np.concatenate(tokens)).cuda(),
                  torch.as_tensor(np.concatenate(targets)).cuda(), _i32(np.cumsum([0] + sizes)), _i32(base), keep=keep,
                  keep_count=count, next_token=nxt)
    for b in range(len(sizes)):
        path, choice = o.accept(trees[b], tokens[b], targets[b])
        assert keep[b].tolist() == [int(base[b]) + i for i in path] + [-1] * (width - len(path))
        assert int(count[b]) == len(path) and int(nxt[b]) == choice


def test_tree_accept_refusals(K):
    from pagelora_b200 import _capi

    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = torch.zeros(4, dtype=torch.int64, device="cuda")
    keep, count = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    nxt = torch.zeros(1, dtype=torch.int64, device="cuda")
    K.tree_accept(_i32([-1, 0, 1, 2]), one, one, _i32([0, 4]), _i32([0]), keep=keep, keep_count=count, next_token=nxt,
                  status=status)  # a path of four, room for two
    assert int(status.item()) == _capi.PL_ERR_INVALID_ARGUMENT and int(count.item()) == 0
    with pytest.raises(TypeError):
        K.tree_accept(_i32([-1]), one.int(), one, _i32([0, 1]), _i32([0]), keep=keep, keep_count=count, next_token=nxt)


def test_calls_without_entries(K):
    """No drafted token in any row: nothing to mask or attend to, every row keeps nothing."""

    host, dev = _case([(3, 20), (2, 0)], 8, 2, 128, 16, seed=14)
    none = _i32([0, 0, 0])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    mask, depth = K.tree_mask(none[:0], none, 1, status=status)
    assert mask.shape == (0, 1) and depth.numel() == 0
    out = K.paged_tree_attention(dev["q"][:0], dev["cache"], none, dev["kv_indptr"], dev["kv_indices"], dev["last"], mask,
                                 status=status)
    assert out.shape == (0, 8, 128)
    keep, count = torch.full((2, 4), 9, dtype=torch.int32, device="cuda"), none[:2].clone() + 9
    nxt = torch.zeros(2, dtype=torch.int64, device="cuda")
    K.tree_accept(none[:0], nxt[:0], nxt[:0], none, none[:2], keep=keep, keep_count=count, next_token=nxt, status=status)
    assert count.tolist() == [0, 0] and int(status.item()) == 0


@pytest.mark.parametrize("d", [64, 128])
def test_a_row_of_one_position_is_exact(K, d):
    """Tokens without a context that see themselves alone: the output is their V, the LSE their score."""

    n = 20
    host, dev = _case([(n, 0), (1, 0)], 8, 2, d, 16, seed=5, see=[np.eye(n, dtype=bool), np.eye(1, dtype=bool)])
    out, _ = _run(K, dev)
    want, _, _ = o.tree_attention(host["q"], host["cache"], host["qo"], host["kv_indptr"], host["kv_indices"],
                                  host["last"], host["see"])
    assert (out == np.float64(np.float32(want))).all()
