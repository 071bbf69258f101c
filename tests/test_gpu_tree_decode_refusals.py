"""TreeDecoder when it runs out of room: a step that cannot be served changes
no row, accepts nothing and is reported; after rows were released the others
go on as if it had not been tried.

Logits against per-row oracle decoders, within the bound of the batch engine's
own tests (max |err| < 0.1 over a small model's logits).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.decoder import OracleDecoder
from pagelora_b200.synthetic import ModelSpec, make_model_weights, random_prompt

pytestmark = pytest.mark.gpu

QWEN = ModelSpec("small-qwen3", 2, 512, 8, 2, 128, 1024, 4096, 1.0e6, 1e-6, qk_norm=True)


class Run:
    """A decoder, and what its rows' contexts should be."""

    def __init__(self, device, lens, sparse=None, **engine):
        from pagelora_b200.batch_engine import BatchDecodeEngine
        from pagelora_b200.tree_decode import TreeDecoder

        self.w = {k: v.bfloat16() for k, v in make_model_weights(QWEN, seed=0, dtype=torch.float32, norm_jitter=0.1).items()}
        eng = BatchDecodeEngine(QWEN, dict(self.w), adapters=None, lora_spec=None, row_adapter=[-1] * len(lens),
                                page_size=16, device=device, **engine)
        self.history = [list(random_prompt(QWEN.vocab, n, seed=10 + i)) for i, n in enumerate(lens)]
        self.cur = eng.prefill(self.history)
        self.dec = TreeDecoder(eng, sparse=sparse)
        self.device = device

    def oracle(self, tokens):
        o = OracleDecoder(QWEN, {k: v.float() for k, v in self.w.items()}, None, 1.0, page_size=16, num_pages=40, bf16=True)
        for t in tokens:
            _, lg = o.step(t)
        return lg

    def verify(self, trees, max_tokens):
        """trees: (tokens, parents) by row; None sits the step out."""

        trees = [t or ([], []) for t in trees]
        i32 = dict(dtype=torch.int32, device=self.device)
        return self.dec.verify(torch.tensor(sum([t for t, _ in trees], []), dtype=torch.int64, device=self.device),
                               torch.tensor(sum([p for _, p in trees], []), **i32),
                               torch.tensor(np.cumsum([0] + [len(t) for t, _ in trees]), **i32), max_tokens)

    def state(self):
        d = self.dec
        torch.cuda.synchronize()
        return [t.clone() for t in (d.num, d.last, d.lens, d.refcount)] + [t.clone() for t in self.contents()]

    def contents(self):
        """Every row's cached K/V, position by position."""

        d = self.dec
        for r, n in enumerate(d.lens.tolist()):
            pos = torch.arange(n, device=self.device)
            yield d.e.kv[:, d.table[r, pos // 16].long(), :, pos % 16]

    def refused(self, res, before, reason):
        assert (res.keep_count == 0).all() and (res.keep == -1).all() and (res.next_token == -1).all()
        self.unchanged(before, reason)

    def unchanged(self, before, reason):
        from pagelora_b200 import _capi

        with pytest.raises(RuntimeError, match=_capi.status_string(getattr(_capi, reason))):
            self.dec.check()
        assert all(torch.equal(a, b) for a, b in zip(before, self.state()))
        self.dec.check()  # reported once

    def good_step(self, rows):
        """A step of two tokens for `rows` (the second one is rejected or taken), its logits against the oracle's."""

        trees = [([self.cur[r], self.cur[r] ^ 1], [-1, 0]) if r in rows else None for r in range(len(self.cur))]
        res = self.verify(trees, 2)
        self.dec.check()
        at = 0
        for r in rows:
            lg = self.oracle(self.history[r] + [self.cur[r]])
            assert np.abs(res.logits[at].float().cpu().numpy() - lg).max() < 0.1, r
            at += 2
            kept = int(res.keep_count[r])
            self.history[r] += [self.cur[r], self.cur[r] ^ 1][:kept]
            self.cur[r] = int(res.next_token[r])
        assert self.dec.lens.tolist() == [len(h) for h in self.history]

    def release(self, r):
        self.dec.release([r])
        self.history[r] = []


def test_a_row_at_its_capacity(cuda_device):
    run = Run(cuda_device, [70, 20, 33], max_context=64)  # 5 pages a row: 80 tokens
    run.good_step([0, 1, 2])
    before = run.state()
    chain = ([run.cur[0]] * 12, list(range(-1, 11)))
    res = run.verify([chain, chain, None], 12)
    run.refused(res, before, "PL_ERR_ROW_CAPACITY")
    run.release(0)
    run.good_step([1, 2])
    run.good_step([1, 2])


def test_a_pool_without_room(cuda_device):
    run = Run(cuda_device, [40, 20, 33], max_context=160, num_pages=9)  # 3 + 2 + 3 pages held
    run.good_step([0, 1, 2])
    before = run.state()
    chain = ([run.cur[0]] * 12, list(range(-1, 11)))
    res = run.verify([chain, chain, chain], 12)  # two more pages
    run.refused(res, before, "PL_ERR_POOL_EXHAUSTED")
    run.release(1)
    run.good_step([0, 2])
    run.good_step([0, 2])


def test_no_room_to_move_the_accepted_tokens(cuda_device):
    """The drafts fit, but the accepted path skips a rejected token and its move needs a page: the step is undone."""

    run = Run(cuda_device, [40, 30], max_context=160, num_pages=5)  # 3 + 2 pages: none is free
    run.good_step([0])
    n = len(run.history[0])
    order = np.argsort(run.oracle(run.history[0] + [run.cur[0]]))
    drafts = [int(order[0]), *(int(t) for t in order[-1:-4:-1])]  # the least likely token, then the three likeliest
    tree = ([run.cur[0], *drafts], [-1, 0, 0, 0, 0])
    assert n % 16 + 5 <= 16  # the drafts need no page
    before = run.state()
    res = run.verify([tree, None], 5)
    run.refused(res, before, "PL_ERR_POOL_EXHAUSTED")
    run.release(1)
    res = run.verify([tree, None], 5)  # the same step again
    run.dec.check()
    taken = int(res.keep[0, 1]) - n
    assert res.keep_count.tolist() == [2, 0] and int(res.keep[0, 0]) == n and 2 <= taken <= 4
    run.history[0] += [run.cur[0], tree[0][taken]]
    run.cur[0] = int(res.next_token[0])
    run.good_step([0])


def test_sparse_steps_without_room(cuda_device):
    from pagelora_b200.tree_decode import SparsePages

    run = Run(cuda_device, [15, 31, 20], sparse=SparsePages(select=16), max_context=160, num_pages=6)  # 1 + 2 + 2 held

    def step():
        nxt, logits = run.dec.step_sparse(torch.tensor(run.cur, dtype=torch.int64, device=cuda_device))
        return nxt.tolist(), logits

    def accept(nxt, logits, rows):
        run.dec.check()
        for r in rows:
            run.history[r].append(run.cur[r])
            assert np.abs(logits[r].float().cpu().numpy() - run.oracle(run.history[r])).max() < 0.1, r
            run.cur[r] = nxt[r]
        assert run.dec.lens.tolist() == [len(h) for h in run.history]

    accept(*step(), [0, 1, 2])  # both short rows are full now
    before = run.state()
    bounds = run.dec.bounds.clone()
    nxt, _ = step()  # two pages for one that is free
    assert nxt == [-1, -1, -1]
    run.unchanged(before, "PL_ERR_POOL_EXHAUSTED")
    assert torch.equal(bounds, run.dec.bounds)
    run.good_step([2])


def test_forks_without_room(cuda_device):
    run = Run(cuda_device, [40, 20, 33], max_context=160, num_pages=8)
    run.release(1)
    run.release(2)
    run.dec.fork([0], [2])  # two shared pages and a copy
    run.history[2], run.cur[2] = list(run.history[0]), run.cur[0] ^ 1
    run.good_step([0, 2])
    before = run.state()
    run.dec.fork([0], [2])  # not empty
    run.unchanged(before, "PL_ERR_INVALID_ARGUMENT")
    run.good_step([0, 2])
