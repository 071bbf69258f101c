"""BoundedDecoder: windows, eviction by weight and the 4-bit cache over a batch
engine's rows.

Every layer's attention is checked against the oracle of its operator over the
cache that it was given (tolerances of test_gpu_window_attention.py and
test_gpu_kv4_cache.py); where nothing is bounded away, the logits against
per-row oracle decoders (max |err| < 0.1, the batch engine's own bound).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_kv4_cache as kv4_tests
import test_gpu_window_attention as window_tests
from oracle import small_cache as o
from test_gpu_tree_decode_refusals import QWEN, Run

pytestmark = pytest.mark.gpu


class Bounded(Run):
    def __init__(self, device, lens, engine=None, **kw):
        from pagelora_b200.bounded_decode import BoundedDecoder

        super().__init__(device, lens, **(engine or {}))
        self.dec = BoundedDecoder(self.dec.e, **kw)

    def step(self):
        nxt, logits = self.dec.step(torch.tensor(self.cur, dtype=torch.int64, device=self.device))
        self.dec.check()
        for r, h in enumerate(self.history):
            if h:
                h.append(self.cur[r])
                self.cur[r] = int(nxt[r])
            else:
                assert int(nxt[r]) == -1 and (logits[r] == 0).all()
        assert self.dec.pos.tolist() == [len(h) for h in self.history]
        return logits


def _host(q, cache, indptr, indices, last):
    return dict(q=q.float().cpu().numpy(), qo=np.arange(q.shape[0] + 1), indptr=indptr.cpu().numpy(),
                indices=indices.cpu().numpy(), last=last.cpu().numpy(),
                cache=cache.float().cpu().numpy() if cache.dtype == torch.bfloat16 else None)


def test_a_wide_window_is_the_whole_context(cuda_device):
    from pagelora_b200.bounded_decode import Window

    run = Bounded(cuda_device, [60, 15, 33], window=Window(1000), engine=dict(max_context=192))
    for _ in range(3):
        logits = run.step()
        for r in range(3):
            assert np.abs(logits[r].float().cpu().numpy() - run.oracle(run.history[r])).max() < 0.1, r
    assert run.dec.lens.tolist() == [63, 18, 36]


def test_a_window(cuda_device, monkeypatch):
    from pagelora_b200 import kernels as K
    from pagelora_b200.bounded_decode import Window

    run = Bounded(cuda_device, [100, 15, 33], window=Window(24, 2), engine=dict(max_context=192))
    seen, plain = [], K.paged_window_decode

    def watched(q, kv, indptr, indices, last, *, window, sinks, status):
        lse = torch.empty(q.shape[:2], device=q.device)
        out = plain(q, kv, indptr, indices, last, window=window, sinks=sinks, out_lse=lse, status=status)
        window_tests._check(out, lse, _host(q, kv, indptr, indices, last), window, sinks, q.shape[2] ** -0.5)
        seen.append((window, sinks))
        return out

    monkeypatch.setattr(K, "paged_window_decode", watched)
    run.step()
    run.release(1)
    run.step()
    run.dec.fork([0], [1])
    run.history[1], run.cur[1] = list(run.history[0]), run.cur[0] ^ 1
    run.step()
    assert seen == [(24, 2)] * 3 * QWEN.num_layers


def test_weights_and_eviction(cuda_device):
    from pagelora_b200.bounded_decode import EvictBudget

    budget = EvictBudget(40, sinks=3, recent=10)
    run = Bounded(cuda_device, [100, 15, 37], evict=budget, engine=dict(max_context=192))
    given = QWEN.num_layers * QWEN.num_qo_heads  # what a step's softmaxes add up to
    for i in range(1, 4):
        logits = run.step()
        for r in range(3):
            assert np.abs(logits[r].float().cpu().numpy() - run.oracle(run.history[r])).max() < 0.1, r
        # sums of fp32 rounded weights, each within 2^-12 of its part
        assert torch.allclose(run.dec.weight.sum(1), torch.full((3,), float(i * given), device=cuda_device), rtol=2.0 ** -11)
    before, cache = run.dec.weight.cpu(), [c.cpu() for c in run.contents()]  # [position, layer, ...]
    run.dec.evict()
    run.dec.check()
    assert run.dec.lens.tolist() == [40, 18, 40] and run.dec.pos.tolist() == [103, 18, 40]
    after = run.dec.weight.cpu()
    for r, (old, new, n) in enumerate(zip(cache, run.contents(), [103, 18, 40])):
        pos = o.select(before[r].numpy(), n, 40, 3, 10)
        assert torch.equal(new.cpu(), old[pos]) and torch.equal(after[r, :len(pos)], before[r, pos])
        assert (after[r, len(pos):] == 0).all()
    run.step()  # over what stays, at the positions that follow
    assert run.dec.lens.tolist() == [41, 19, 41]
    run.release(0)
    run.dec.fork([2], [0])
    run.history[0], run.cur[0] = list(run.history[2]), run.cur[2] ^ 1
    assert torch.equal(run.dec.weight[0], run.dec.weight[2])
    run.step()
    run.dec.evict()
    run.dec.check()
    assert run.dec.lens.tolist() == [40, 20, 40]


def test_a_refused_step_and_a_refused_eviction_change_nothing(cuda_device):
    from pagelora_b200.bounded_decode import EvictBudget

    run = Bounded(cuda_device, [96, 96], evict=EvictBudget(50, recent=0), engine=dict(max_context=96, num_pages=14))
    run.step()  # 14 pages: all taken
    before, weight = run.state(), run.dec.weight.clone()
    run.dec.evict()  # no page to move the kept tokens to
    run.unchanged(before, "PL_ERR_POOL_EXHAUSTED")
    assert torch.equal(run.dec.weight, weight)
    nxt = None
    for _ in range(16):
        nxt, _ = run.dec.step(torch.tensor(run.cur, dtype=torch.int64, device=cuda_device))
        if int(nxt[0]) == -1:
            break
        run.dec.check()
        before, weight = run.state(), run.dec.weight.clone()
    assert (nxt == -1).all()
    torch.cuda.synchronize()
    assert torch.equal(run.dec.weight, weight) and all(torch.equal(a, b) for a, b in zip(before, run.state()))


@pytest.mark.parametrize("window", [None, (20, 2)])
def test_a_4_bit_cache(cuda_device, monkeypatch, window):
    from pagelora_b200 import kernels as K
    from pagelora_b200.bounded_decode import Window

    run = Bounded(cuda_device, [100, 15, 33], window=window and Window(*window), kv4=True, engine=dict(max_context=192))
    dec = run.dec
    # the prompts' records
    for li in range(QWEN.num_layers):
        want = o.record_bytes(*o.pack4(dec.e.kv[li].float().cpu().numpy()))
        got = dec.kv4[li].cpu().numpy()
        for r, n in enumerate([100, 15, 33]):
            pos = np.arange(n)
            page = dec.table[r].cpu().numpy()[pos // 16]
            assert (got[page, :, pos % 16] == want[page, :, pos % 16]).all()
    seen, plain, append = [], K.paged_kv4_decode, K.kv4_append

    def appended(k, v, cache, page, off, status=None):
        append(k, v, cache, page, off, status)
        rec = cache.cpu().numpy()[page.cpu().numpy(), :, off.cpu().numpy()]
        for i, x in enumerate((k, v)):
            assert (rec[:, i] == o.record_bytes(*o.pack4(x.float().cpu().numpy()))).all()

    def watched(q, cache, indptr, indices, last, *, window, sinks, status):
        lse = torch.empty(q.shape[:2], device=q.device)
        out = plain(q, cache, indptr, indices, last, window=window, sinks=sinks, out_lse=lse, status=status)
        host = dict(_host(q, cache, indptr, indices, last), rec=cache.cpu().numpy())
        kv4_tests._check(out, lse, host, window, sinks)
        seen.append(window)
        return out

    monkeypatch.setattr(K, "paged_kv4_decode", watched)
    monkeypatch.setattr(K, "kv4_append", appended)
    run.step()
    run.release(1)
    run.step()
    run.dec.fork([0], [1])
    run.history[1], run.cur[1] = list(run.history[0]), run.cur[0] ^ 1
    run.step()
    assert len(seen) == 3 * QWEN.num_layers and run.dec.lens.tolist() == [103, 103, 36]


def test_arguments(cuda_device):
    from pagelora_b200.bounded_decode import BoundedDecoder, EvictBudget, Window

    run = Run(cuda_device, [20])
    for kw in (dict(), dict(evict=EvictBudget(64), kv4=True), dict(evict=EvictBudget(64), window=Window(5)),
               dict(window=Window(0)), dict(window=Window(5, -1)), dict(evict=EvictBudget(10, sinks=4, recent=7))):
        with pytest.raises(ValueError):
            BoundedDecoder(run.dec.e, **kw)
    dec = BoundedDecoder(run.dec.e, window=Window(5))
    with pytest.raises(ValueError):
        dec.evict()
    with pytest.raises(ValueError):
        dec.verify(None, None, None, 1)
    with pytest.raises(ValueError):
        dec.step(torch.zeros(2, dtype=torch.int64, device=cuda_device))
