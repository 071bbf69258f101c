"""TreeDecoder's sparse side: budgets smaller than the rows, bounds that stay
current through drafts, compactions, forks and releases, and steps without a
host synchronisation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_tree_decode_refusals import Run

pytestmark = pytest.mark.gpu


def _bounds_are_current(dec):
    """Those of every held page equal a computation from the cache alone."""

    from pagelora_b200 import kernels as K

    ids, lens = [], []
    for r, n in enumerate(dec.lens.tolist()):
        for i in range(-(-n // 16)):
            ids.append(int(dec.table[r, i]))
            lens.append(min(16, n - 16 * i))
    i32 = dict(dtype=torch.int32, device=dec.lens.device)
    for li in range(dec.e.kv.shape[0]):
        bounds, scale = torch.zeros_like(dec.bounds[li]), torch.zeros_like(dec.bound_scale[li])
        K.page_bounds(dec.e.kv[li], torch.tensor(ids, **i32), bounds, scale, page_len=torch.tensor(lens, **i32))
        assert torch.equal(bounds[ids], dec.bounds[li][ids]) and torch.equal(scale[ids], dec.bound_scale[li][ids])


def _drafts(run, rng, sizes):
    return [(([run.cur[r]] + rng.integers(0, 4096, n - 1).tolist(), [-1] + [int(rng.integers(0, i)) for i in range(1, n)])
             if n else None) for r, n in enumerate(sizes)]


def _after(run, trees, res):
    for r, t in enumerate(trees):
        if t is not None:
            n = len(run.history[r])
            run.history[r] += [t[0][int(p) - n] for p in res.keep[r, : int(res.keep_count[r])]]
            run.cur[r] = int(res.next_token[r])
    assert run.dec.lens.tolist() == [len(h) for h in run.history]


def test_bounds_follow_drafts_forks_and_releases(cuda_device):
    from pagelora_b200.tree_decode import SparsePages

    run = Run(cuda_device, [60, 15, 33, 47], sparse=SparsePages(select=64), max_context=192)
    rng = np.random.default_rng(1)
    for step in range(6):
        trees = _drafts(run, rng, [int(rng.integers(1, 20)) if run.history[r] and rng.random() < 0.8 else 0 for r in range(4)])
        if not any(trees):
            continue
        res = run.verify(trees, 20)
        run.dec.check()
        _after(run, trees, res)
        _bounds_are_current(run.dec)
        if step == 1:
            run.release(3)
            run.dec.fork([0], [3])
            run.history[3], run.cur[3] = list(run.history[0]), run.cur[0] ^ 1
            _bounds_are_current(run.dec)
        if step == 3:
            run.release(1)
            _bounds_are_current(run.dec)
    # with a budget for all pages a sparse step is a dense one
    live = [r for r in range(4) if run.history[r]]
    _, logits = run.dec.step_sparse(torch.tensor(run.cur, dtype=torch.int64, device=cuda_device))
    run.dec.check()
    for r in live:
        assert np.abs(logits[r].float().cpu().numpy() - run.oracle(run.history[r] + [run.cur[r]])).max() < 0.1, r


def test_a_budget_smaller_than_the_rows(cuda_device):
    """The step's attention is that of the selected pages: every layer's call is checked against a dense decode over
    a page list of its own per kv head."""

    from pagelora_b200 import kernels as K
    from pagelora_b200.tree_decode import SparsePages

    run = Run(cuda_device, [180, 15, 93, 170], sparse=SparsePages(select=5, sink=1, recent=2), max_context=192)
    res = run.verify([([c, c ^ 1], [-1, 0]) for c in run.cur], 2)
    run.cur = res.next_token.tolist()
    seen, plain = [], K.paged_sparse_decode

    def watched(q, kv, indptr, indices, last, bounds, scale, **kw):
        sel = torch.full((q.shape[0], kv.shape[3], kw["num_select"]), -9, dtype=torch.int32, device=q.device)
        out = plain(q, kv, indptr, indices, last, bounds, scale, selected=sel, **kw)
        seen.append((q.clone(), kv, indptr.clone(), indices.clone(), last.clone(), sel, out.clone()))
        return out

    K.paged_sparse_decode = watched
    try:
        run.dec.step_sparse(torch.tensor(run.cur, dtype=torch.int64, device=cuda_device))
    finally:
        K.paged_sparse_decode = plain
    run.dec.check()
    assert len(seen) == 2
    lens = run.dec.lens.tolist()
    for q, kv, indptr, indices, last, sel, out in seen:
        for r in range(4):
            pages = indices[int(indptr[r]): int(indptr[r + 1])].long()
            assert len(pages) == -(-lens[r] // 16)
            for h in range(2):
                chosen = [i for i in sel[r, h].tolist() if i >= 0]
                assert len(chosen) == min(5, len(pages)) and chosen == sorted(set(chosen))
                assert chosen[0] == 0 and chosen[-1] == len(pages) - 1
                k, v = (torch.cat([kv[pages[i], j, : (int(last[r]) if i == len(pages) - 1 else 16), h] for i in chosen])
                        .double() for j in (0, 1))
                p = torch.softmax(q[r, 4 * h: 4 * h + 4].double() @ k.T / 128 ** 0.5, -1)
                # P and the output rounded to bf16, fp32 scores
                spread = p @ v.abs()
                err = (out[r, 4 * h: 4 * h + 4].double() - p @ v).abs()
                assert (err <= 2.0 ** -8 * ((p @ v).abs() + spread) + 2.0 ** -12 * spread).all()


def test_steps_do_not_wait_for_the_device(cuda_device):
    from pagelora_b200.tree_decode import SparsePages

    run = Run(cuda_device, [60, 15, 33], sparse=SparsePages(select=4), max_context=192)
    rng = np.random.default_rng(2)
    cur = torch.tensor(run.cur, dtype=torch.int64, device=cuda_device)
    toks = torch.tensor(rng.integers(0, 4096, 9), dtype=torch.int64, device=cuda_device)
    par = torch.tensor([-1, 0, 0] * 3, dtype=torch.int32, device=cuda_device)
    qo = torch.tensor([0, 3, 6, 9], dtype=torch.int32, device=cuda_device)
    run.dec.verify(toks, par, qo, 3)
    run.dec.step_sparse(cur)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        run.dec.verify(toks, par, qo, 3)
        run.dec.step_sparse(cur)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    run.dec.check()


def test_many_drafted_tokens(cuda_device):
    """More than 128 drafted tokens in all: the projections run in blocks."""

    run = Run(cuda_device, [20, 3, 41], max_context=192)
    rng = np.random.default_rng(3)
    trees = _drafts(run, rng, [90, 33, 70])
    res = run.verify(trees, 90)
    run.dec.check()
    at = 0
    for r, (toks, par) in enumerate(trees):
        for i in (0, 1, len(toks) // 2, len(toks) - 1):
            path, j = [], i
            while j >= 0:
                path.append(toks[j])
                j = par[j]
            want = run.oracle(run.history[r] + path[::-1])
            assert np.abs(res.logits[at + i].float().cpu().numpy() - want).max() < 0.1, (r, i)
        at += len(toks)
    _after(run, trees, res)


def test_entries_that_are_left_out(cuda_device):
    """Page -1 of length 0 in a list of page_bounds; any other page outside the pool is reported."""

    from pagelora_b200 import _capi
    from pagelora_b200 import kernels as K

    i32 = dict(dtype=torch.int32, device=cuda_device)
    kv = torch.randn(6, 2, 16, 3, 64, device=cuda_device).bfloat16()
    for ids, lens, want in (([2, -1, 5, -1], [16, 0, 7, 0], 0), ([-1], [1], _capi.PL_ERR_PAGE_OUT_OF_RANGE),
                            ([-2], [0], _capi.PL_ERR_PAGE_OUT_OF_RANGE), ([6], [0], _capi.PL_ERR_PAGE_OUT_OF_RANGE),
                            ([-1], None, _capi.PL_ERR_PAGE_OUT_OF_RANGE)):
        bounds = torch.full((6, 3, 2, 64), 99, dtype=torch.int8, device=cuda_device)
        scale = torch.full((6, 3), -5.0, device=cuda_device)
        status = torch.zeros(1, **i32)
        K.page_bounds(kv, torch.tensor(ids, **i32), bounds, scale,
                      page_len=None if lens is None else torch.tensor(lens, **i32), status=status)
        assert int(status.item()) == want
        for p in range(6):
            if p in ids and want == 0:
                alone, s = torch.zeros_like(bounds), torch.zeros_like(scale)
                K.page_bounds(kv, torch.tensor([p], **i32), alone, s, page_len=torch.tensor([lens[ids.index(p)]], **i32))
                assert torch.equal(bounds[p], alone[p]) and torch.equal(scale[p], s[p])
            else:
                assert (bounds[p] == 99).all() and (scale[p] == -5.0).all()
