"""The cache operators without a GPU: what their C entries refuse before they
touch the device, the workspace sizes, and the oracles against brute force."""

from __future__ import annotations

import itertools

import numpy as np
import pytest

from oracle import page_pool, sparse_decode, tree_attention

P = 0x10000  # an aligned address that no refused call reads


@pytest.fixture(scope="module")
def capi():
    from pagelora_b200 import _capi, build

    if build.is_stale():
        build.build()
    return _capi, _capi.load_library()


# argument lists by name, all of them valid
TREE = dict(q=P, q_st=1024, q_sh=128, kv=P, pages=100, qo=P, kvp=P, kvi=P, last=P, total_pages=100, mask=P, mask_stride=1,
            words=1, batch=2, total_q=8, hq=8, hkv=2, d=128, ps=16, scale=0.1, out=P, o_st=1024, o_sh=128, lse=None, ws=P,
            ws_bytes=1 << 40, status=None, stream=None)
SPARSE = dict(q=P, q_sb=1024, q_sh=128, kv=P, pages=100, indptr=P, indices=P, last=P, total_pages=100, max_pages=60,
              bounds=P, scale=P, batch=2, hq=8, hkv=2, d=128, ps=16, sm_scale=0.1, select=20, sink=1, recent=2, out=P,
              o_sb=1024, o_sh=128, lse=None, selected=P, ws=P, ws_bytes=1 << 40, status=None, stream=None)
BOUNDS = dict(kv=P, pages=100, hkv=2, d=128, ps=16, ids=P, lens=None, n=3, bounds=P, scale=P, status=None, stream=None)
MASK = dict(parents=P, qo=P, base=None, batch=2, total_q=8, words=1, mask=P, stride=1, depth=None, positions=None,
            status=None, stream=None)
ACCEPT = dict(parents=P, tokens=P, targets=P, qo=P, base=P, batch=2, total_q=8, max_keep=8, keep=P, keep_stride=8, count=P,
              nxt=P, status=None, stream=None)
TABLE = dict(refcount=P, pages=100, row_pages=P, row_num=P, last=P, rows=4, cap=8)
RELEASE = dict(TABLE, released=P, n=2, status=None, stream=None)
RESERVE = dict(TABLE, ps=16, indptr=P, total=8, slot_page=P, slot_offset=P, positions=None, out_indptr=None, out_indices=None,
               max_indices=0, status=None, stream=None)
POOL = dict(pool=P, layer_stride=1 << 20, layers=2, token_bytes=512)
FORK = dict(POOL, **TABLE, ps=16, src=P, dst=P, n=2, ws=P, ws_bytes=1 << 20, status=None, stream=None)
COMPACT = dict(POOL, **TABLE, ps=16, keep_from=P, keep=P, keep_stride=8, keep_count=P, max_keep=8, ws=P, ws_bytes=1 << 20,
               status=None, stream=None)

INVALID = {
    "pl_paged_tree_attention": (TREE, [
        dict(q=None), dict(kv=None), dict(qo=None), dict(kvp=None), dict(kvi=None), dict(last=None), dict(mask=None),
        dict(out=None), dict(batch=-1), dict(total_q=-1), dict(pages=0), dict(words=0), dict(mask_stride=0), dict(hkv=3),
        dict(hkv=0), dict(scale=0.0), dict(scale=float("nan")), dict(q=P + 2), dict(kv=P + 8), dict(out=P + 4),
        dict(q_st=1023), dict(o_sh=4)]),
    "pl_paged_sparse_decode": (SPARSE, [
        dict(q=None), dict(kv=None), dict(indptr=None), dict(bounds=None), dict(scale=None), dict(selected=None),
        dict(out=None), dict(batch=-1), dict(pages=0), dict(max_pages=-1), dict(hkv=3), dict(sm_scale=-1.0), dict(sink=-1),
        dict(recent=0), dict(select=0), dict(select=2), dict(q=P + 2), dict(bounds=P + 8), dict(q_sb=1001)]),
    "pl_page_bounds": (BOUNDS, [dict(kv=None), dict(bounds=None), dict(scale=None), dict(ids=None), dict(pages=0),
                                dict(hkv=0), dict(ps=0), dict(n=-1), dict(kv=P + 2)]),
    "pl_tree_mask": (MASK, [dict(parents=None), dict(qo=None), dict(mask=None), dict(batch=-1), dict(total_q=-1),
                            dict(words=0), dict(stride=0)]),
    "pl_tree_accept": (ACCEPT, [dict(parents=None), dict(tokens=None), dict(targets=None), dict(base=None), dict(keep=None),
                                dict(count=None), dict(nxt=None), dict(batch=-1), dict(max_keep=0), dict(keep_stride=7)]),
    "pl_page_release": (RELEASE, [dict(refcount=None), dict(row_pages=None), dict(pages=-1), dict(rows=-1), dict(cap=-1),
                                  dict(n=-1), dict(released=None)]),
    "pl_page_reserve": (RESERVE, [dict(refcount=None), dict(row_num=None), dict(last=None), dict(ps=0), dict(indptr=None),
                                  dict(total=-1), dict(slot_page=None), dict(slot_offset=None), dict(max_indices=-1)]),
    "pl_page_fork": (FORK, [dict(pool=None), dict(layers=-1), dict(token_bytes=0), dict(refcount=None), dict(src=None),
                            dict(dst=None), dict(n=-1), dict(n=5), dict(ps=0)]),
    "pl_cache_compact": (COMPACT, [dict(pool=None), dict(token_bytes=24), dict(keep_from=None), dict(keep=None),
                                   dict(keep_count=None), dict(max_keep=-1), dict(keep_stride=7)]),
}


@pytest.mark.parametrize("fn", INVALID)
def test_invalid_arguments(capi, fn):
    c, lib = capi
    args, bad = INVALID[fn]
    for change in bad:
        got = getattr(lib, fn)(*dict(args, **change).values())
        assert got in (c.PL_ERR_INVALID_ARGUMENT, c.PL_ERR_UNSUPPORTED), (change, got)


@pytest.mark.parametrize("fn,args,change", [
    ("pl_paged_tree_attention", TREE, dict(d=96)), ("pl_paged_tree_attention", TREE, dict(ps=24)),
    ("pl_paged_tree_attention", TREE, dict(hq=258)), ("pl_paged_sparse_decode", SPARSE, dict(ps=64)),
    ("pl_paged_sparse_decode", SPARSE, dict(hq=34)), ("pl_paged_sparse_decode", SPARSE, dict(d=80)),
    ("pl_page_bounds", BOUNDS, dict(d=96)), ("pl_paged_sparse_decode", SPARSE, dict(select=24577, max_pages=30000)),
])
def test_unsupported_shapes(capi, fn, args, change):
    c, lib = capi
    assert getattr(lib, fn)(*dict(args, **change).values()) == c.PL_ERR_UNSUPPORTED


def test_workspaces_that_are_too_small(capi):
    c, lib = capi
    small = c.PL_ERR_WORKSPACE_TOO_SMALL
    need = lib.pl_tree_workspace_bytes(2, 8, 8, 2, 128)
    assert need > 0
    for change in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=P + 8)):
        assert lib.pl_paged_tree_attention(*dict(TREE, **change).values()) == small
    need = lib.pl_sparse_workspace_bytes(2, 2, 60)
    assert need >= 2 * 2 * 60 * 4
    for change in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=P + 8)):
        assert lib.pl_paged_sparse_decode(*dict(SPARSE, **change).values()) == small
    for change in (dict(ws=None), dict(ws_bytes=lib.pl_page_fork_workspace_bytes(2) - 1)):
        assert lib.pl_page_fork(*dict(FORK, **change).values()) == small
    for change in (dict(ws=None), dict(ws_bytes=lib.pl_cache_compact_workspace_bytes(4, 8) - 1)):
        assert lib.pl_cache_compact(*dict(COMPACT, **change).values()) == small


def test_empty_calls_do_nothing(capi):
    _, lib = capi
    for fn, args, change in (("pl_paged_tree_attention", TREE, dict(total_q=0)),
                             ("pl_paged_tree_attention", TREE, dict(batch=0)),
                             ("pl_paged_sparse_decode", SPARSE, dict(batch=0)), ("pl_page_bounds", BOUNDS, dict(n=0)),
                             ("pl_tree_mask", MASK, dict(total_q=0)), ("pl_tree_accept", ACCEPT, dict(batch=0)),
                             ("pl_paged_tree_attention", TREE, dict(total_q=0, q=None, mask=None, out=None)),
                             ("pl_tree_mask", MASK, dict(total_q=0, parents=None, mask=None)),
                             ("pl_paged_sparse_decode", SPARSE, dict(batch=0, q=None, last=None, out=None, selected=None)),
                             ("pl_page_release", RELEASE, dict(n=0, released=None)),
                             ("pl_page_fork", FORK, dict(n=0, ws=None))):
        assert getattr(lib, fn)(*dict(args, **change).values()) == 0, fn


def test_status_strings_of_the_pool(capi):
    c, lib = capi
    for code in (c.PL_ERR_POOL_EXHAUSTED, c.PL_ERR_ROW_CAPACITY, c.PL_ERR_PAGE_SHARED, c.PL_ERR_REFCOUNT):
        assert lib.pl_status_string(code) not in (b"", lib.pl_status_string(-1))


def test_wrappers_refuse_cpu_tensors():
    import torch

    from pagelora_b200 import kernels as K

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        K.tree_mask(i32(4), i32(2), 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.page_release(i32(8), i32(2, 4), i32(2), i32(2), i32(1))


# ------------------------------------------------------------------ oracles
def test_oracle_attention_of_a_chain_is_causal():
    """A chain's tree attention is causal attention, computed here as one softmax over a plain sequence."""

    rng = np.random.default_rng(0)
    n, ctx, d = 5, 11, 64
    cache, q = rng.normal(size=(4, 2, 4, 1, d)), rng.normal(size=(n, 2, d))
    pages = [2, 0, 3, 1]
    see = [tree_attention.ancestors([-1, 0, 1, 2, 3])]
    out, lse, _ = tree_attention.tree_attention(q, cache, [0, n], [0, 4], pages, [4], see)
    k, v = (np.concatenate([cache[p, i, :, 0] for p in pages]) for i in (0, 1))
    for i, h in itertools.product(range(n), range(2)):
        s = k[: ctx + i + 1] @ q[i, h] / 8.0
        w = np.exp(s)
        assert np.allclose(out[i, h], w @ v[: ctx + i + 1] / w.sum(), atol=1e-12)
        assert np.isclose(lse[i, h], np.log(w.sum()), atol=1e-12)


def test_oracle_accept_is_the_longest_confirmed_path():
    rng = np.random.default_rng(1)
    for _ in range(200):
        n = int(rng.integers(1, 7))
        parents = [-1] + [int(rng.integers(-1, i)) for i in range(1, n)]
        tokens, targets = rng.integers(0, 2, n), rng.integers(0, 2, n)
        path, nxt = tree_attention.accept(parents, tokens, targets)
        good = [s for k in range(n + 1) for s in itertools.combinations(range(n), k)
                if all((parents[x] == (s[i - 1] if i else -1)) and (i == 0 or tokens[x] == targets[s[i - 1]])
                       for i, x in enumerate(s))]
        assert len(path) == max(map(len, good)) and tuple(path) in good
        assert nxt == (targets[path[-1]] if path else -1)


def test_oracle_bounds_hold_every_key():
    """lo * s <= k <= hi * s, up to the rounding of k / s in fp32, and the score bounds each key's product with the
    quantised queries."""

    rng = np.random.default_rng(2)
    for _ in range(20):
        k = rng.normal(size=(16, 64)).astype(np.float32)
        b, s = sparse_decode.page_bounds(k)
        assert (k >= b[0] * s - 1e-6 * np.abs(k).max()).all() and (k <= b[1] * s + 1e-6 * np.abs(k).max()).all()
        qi = rng.integers(-127, 128, size=64)
        most = np.maximum(qi * b[0].astype(int), qi * b[1].astype(int)).sum()
        assert (k @ qi <= s * most * (1 + 1e-5) + 1e-3).all()


def test_oracle_pool_keeps_its_counts():
    """Whatever a sequence of operations does, refcount[p] is the number of rows that hold p, and a row's tokens are
    those that were written, copied or kept."""

    rng = np.random.default_rng(3)
    pool = page_pool.Pool(np.zeros((1, 40, 2, 4)), np.zeros(40, int), [[] for _ in range(6)], [0] * 6, 8)
    rows: list[list[int]] = [[] for _ in range(6)]  # a number per token
    written = 0
    for step in range(300):
        kind = int(rng.integers(0, 4))
        try:
            if kind == 0:
                counts = [int(rng.integers(0, 5)) for _ in range(6)]
                slots = iter(pool.reserve(counts))
                for r, n in enumerate(counts):
                    for _ in range(n):
                        page, off = next(slots)
                        written += 1
                        pool.data[0, page, :, off] = written
                        rows[r].append(written)
            elif kind == 1:
                a, b = (int(x) for x in rng.choice(6, 2, replace=False))
                pool.fork([a], [b])
                rows[b] = list(rows[a])
            elif kind == 2:
                r = int(rng.integers(0, 6))
                pool.release([r])
                rows[r] = []
            else:
                keep = [sorted(rng.choice(len(t), int(rng.integers(0, len(t) + 1)), replace=False).tolist()) if t else []
                        for t in rows]
                pool.compact([0] * 6, keep)
                rows = [[t[i] for i in k] for t, k in zip(rows, keep)]
        except page_pool.Refused:
            pass
        held = np.bincount([p for row in pool.rows for p in row], minlength=40)
        assert (held == np.asarray(pool.refcount)).all(), step
        for r, t in enumerate(rows):
            assert pool.length(r) == len(t)
            assert [pool.data[0, pool.rows[r][i // 4], 1, i % 4] for i in range(len(t))] == t, step
    assert written > 100
