"""TreeDecoder with rows that ended: a released row stays empty until a fork
or a draft fills it, whatever the other rows do."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_tree_decode_refusals import Run

pytestmark = pytest.mark.gpu


def _step(run, rows):
    nxt, logits = run.dec.step_sparse(torch.tensor(run.cur, dtype=torch.int64, device=run.device))
    run.dec.check()
    assert nxt.shape == (len(run.cur),) and logits.shape[0] == len(run.cur)
    for r in range(len(run.cur)):
        if r in rows:
            run.history[r].append(run.cur[r])
            assert np.abs(logits[r].float().cpu().numpy() - run.oracle(run.history[r])).max() < 0.1, r
            run.cur[r] = int(nxt[r])
        else:
            assert int(nxt[r]) == -1 and not logits[r].any()
    assert run.dec.lens.tolist() == [len(h) for h in run.history]
    pages = [-(-len(h) // 16) for h in run.history]
    assert run.dec.num.tolist() == pages


def test_ended_rows_take_no_part_in_sparse_steps(cuda_device):
    from pagelora_b200.tree_decode import SparsePages

    run = Run(cuda_device, [30, 17, 40, 5], sparse=SparsePages(select=16), max_context=160)
    _step(run, [0, 1, 2, 3])
    run.release(1)
    run.release(3)
    for _ in range(3):
        _step(run, [0, 2])
    held = sum(-(-len(h) // 16) for h in run.history)
    assert int(run.dec.refcount.sum()) == held
    run.dec.fork([2], [1])  # into a row that ended some steps ago
    run.history[1], run.cur[1] = list(run.history[2]), run.cur[2] ^ 1
    _step(run, [0, 1, 2])
    # a draft restarts a row from nothing
    run.verify([None, None, None, ([7, 9], [-1, 0])], 2)
    run.dec.check()
    n = int(run.dec.lens[3])
    assert 1 <= n <= 2
    run.history[3], run.cur[3] = [7, 9][:n], 11
    _step(run, [0, 1, 2, 3])
    for r in range(4):
        run.release(r)
    _step(run, [])
