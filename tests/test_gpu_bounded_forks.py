"""Forks of a BoundedDecoder that are refused change no row: its positions and
weights stay with its pages, and the rows go on as if it had not been tried."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_bounded_decode import Bounded

pytestmark = pytest.mark.gpu


def _modes():
    from pagelora_b200.bounded_decode import EvictBudget, Window

    return dict(window=dict(window=Window(1000)), evict=dict(evict=EvictBudget(40, sinks=3, recent=10)), kv4=dict(kv4=True))


def _rows(dec):
    torch.cuda.synchronize()
    return [dec.pos.clone()] + ([dec.weight.clone()] if dec.budget is not None else [])


def _refused(run, src, dst, reason):
    before, rows = run.state(), _rows(run.dec)
    run.dec.fork(src, dst)
    run.unchanged(before, reason)
    assert all(torch.equal(a, b) for a, b in zip(rows, _rows(run.dec)))


@pytest.mark.parametrize("mode", ["window", "evict", "kv4"])
def test_onto_a_live_row(cuda_device, mode):
    run = Bounded(cuda_device, [40, 20, 40, 33], engine=dict(max_context=192), **_modes()[mode])
    run.step()
    _refused(run, [0], [1], "PL_ERR_INVALID_ARGUMENT")  # of another length
    _refused(run, [0], [2], "PL_ERR_INVALID_ARGUMENT")  # of the same length
    run.release(3)
    _refused(run, [0, 0], [3, 1], "PL_ERR_INVALID_ARGUMENT")  # an empty row and a live one
    _refused(run, [0, 1], [3, 3], "PL_ERR_INVALID_ARGUMENT")  # one row twice
    assert int(run.dec.pos[3]) == 0
    logits = run.step()
    if mode != "kv4":
        for r in range(3):
            assert np.abs(logits[r].float().cpu().numpy() - run.oracle(run.history[r])).max() < 0.1, r


def test_onto_a_row_of_the_same_length_at_another_position(cuda_device):
    run = Bounded(cuda_device, [100, 39], engine=dict(max_context=192), **_modes()["evict"])
    run.step()
    run.dec.evict()
    run.dec.check()
    assert run.dec.lens.tolist() == [40, 40] and run.dec.pos.tolist() == [101, 40]
    _refused(run, [0], [1], "PL_ERR_INVALID_ARGUMENT")
    _refused(run, [1], [0], "PL_ERR_INVALID_ARGUMENT")
    run.step()


@pytest.mark.parametrize("mode", ["window", "evict", "kv4"])
def test_without_room(cuda_device, mode):
    run = Bounded(cuda_device, [40, 5, 45], engine=dict(max_context=192, num_pages=7), **_modes()[mode])
    run.release(1)
    for _ in range(4):
        run.step()  # the last one takes the page that was given back
    _refused(run, [0], [1], "PL_ERR_POOL_EXHAUSTED")
    assert run.dec.pos.tolist() == [44, 0, 49]
    run.step()


@pytest.mark.parametrize("mode", ["window", "evict", "kv4"])
def test_into_empty_rows(cuda_device, mode):
    run = Bounded(cuda_device, [40, 5, 45, 9], engine=dict(max_context=192), **_modes()[mode])
    run.step()
    run.release(1)
    run.release(3)
    run.dec.fork([0, 2], [3, 1])
    run.dec.check()
    for s, d in ((0, 3), (2, 1)):
        run.history[d], run.cur[d] = list(run.history[s]), run.cur[s] ^ 1
    assert run.dec.pos.tolist() == [41, 46, 46, 41]
    if mode == "evict":
        assert torch.equal(run.dec.weight[3], run.dec.weight[0]) and torch.equal(run.dec.weight[1], run.dec.weight[2])
    run.step()
