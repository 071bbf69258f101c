"""What a BoundedDecoder's rows hold: budgets, windows that give back what no
later token sees, and the pool that a 4-bit cache leaves unused."""

from __future__ import annotations

import pytest
import torch

from test_gpu_bounded_decode import Bounded
from test_gpu_tree_decode_refusals import Run

pytestmark = pytest.mark.gpu


def test_a_budget_keeps_a_token(cuda_device):
    """A row that keeps nothing would be one without a context, which takes no part in steps."""

    from pagelora_b200.bounded_decode import BoundedDecoder, EvictBudget

    run = Run(cuda_device, [20])
    with pytest.raises(ValueError):
        BoundedDecoder(run.dec.e, evict=EvictBudget(0, sinks=0, recent=0))
    BoundedDecoder(run.dec.e, evict=EvictBudget(1, sinks=0, recent=0))


def _held(dec):
    """Every row's cached tokens [position, layer, ...] of the pool that the decoder reads."""

    pool = dec.e.kv if dec.kv4 is None else dec.kv4
    for r, n in enumerate(dec.lens.tolist()):
        pos = torch.arange(n, device=pool.device)
        yield pool[:, dec.table[r, pos // 16].long(), :, pos % 16].clone()


@pytest.mark.parametrize("kv4", [False, True])
def test_trim_keeps_sinks_and_window(cuda_device, kv4):
    from pagelora_b200.bounded_decode import Window

    run = Bounded(cuda_device, [100, 15, 33, 26, 70], window=Window(24, 2), kv4=kv4, engine=dict(max_context=192))
    run.step()
    run.release(1)
    run.release(4)
    run.dec.fork([0], [4])  # shared pages
    run.history[4], run.cur[4] = list(run.history[0]), run.cur[0] ^ 1
    run.step()
    old, lens, pos = list(_held(run.dec)), run.dec.lens.tolist(), run.dec.pos.clone()
    assert lens == [102, 0, 35, 28, 102]
    run.dec.trim()
    run.dec.check()
    assert run.dec.lens.tolist() == [26, 0, 26, 26, 26] and torch.equal(run.dec.pos, pos)
    for n, a, b in zip(lens, old, _held(run.dec)):
        keep = list(range(min(n, 2))) + list(range(max(2, n - 24), n))
        assert torch.equal(b, a[keep])
    assert int((run.dec.refcount > 0).sum()) == 2 * 4  # two pages a row
    again = list(_held(run.dec))
    run.dec.trim()
    run.dec.check()
    assert all(torch.equal(a, b) for a, b in zip(again, _held(run.dec)))
    run.step()
    assert run.dec.lens.tolist() == [27, 0, 27, 27, 27]


def test_a_text_longer_than_the_rows(cuda_device):
    """With trim() now and then a window's decoder goes on in seven pages a row as one does that keeps them all."""

    from pagelora_b200.bounded_decode import Window

    lens = [60, 15, 33]
    small = Bounded(cuda_device, lens, window=Window(24, 2), engine=dict(max_context=96))
    large = Bounded(cuda_device, lens, window=Window(24, 2), engine=dict(max_context=400))
    for i in range(300):
        small.cur = list(large.cur)
        a, b = small.step(), large.step()
        assert (a.float() - b.float()).abs().max() < 0.1, i
        if i % 40 == 39:
            small.dec.trim()
            small.dec.check()
            assert small.dec.lens.tolist() == [26, 26, 26]
    assert small.dec.pos.tolist() == [360, 315, 333] == large.dec.lens.tolist()


def test_a_refused_trim_changes_nothing(cuda_device):
    from pagelora_b200.bounded_decode import EvictBudget, Window

    run = Bounded(cuda_device, [96, 96], window=Window(50, 2), engine=dict(max_context=96, num_pages=14))
    run.step()  # 14 pages: all taken
    before, pos = run.state(), run.dec.pos.clone()
    run.dec.trim()  # no page to move the kept tokens to
    run.unchanged(before, "PL_ERR_POOL_EXHAUSTED")
    assert torch.equal(run.dec.pos, pos)
    run.step()
    with pytest.raises(ValueError):
        Bounded(cuda_device, [20], evict=EvictBudget(64)).dec.trim()
    run = Bounded(cuda_device, [20], window=Window(2 ** 31 - 1), engine=dict(max_context=96))
    run.dec.trim()  # no row can be longer
    run.dec.check()
    assert run.dec.lens.tolist() == [20]


def test_a_4_bit_cache_without_the_bf16_pool(cuda_device):
    from pagelora_b200.bounded_decode import Window

    runs = [Bounded(cuda_device, [40, 15, 33], window=Window(24, 2), kv4=True, engine=dict(max_context=4000))
            for _ in range(2)]
    gone = runs[1].dec.e
    pool = gone.kv.numel() * 2
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    gone.kv = None
    assert before - torch.cuda.memory_allocated() >= pool
    for step in range(3):
        a, b = (run.step() for run in runs)
        assert torch.equal(a, b)
        for run in runs:
            if step == 0:
                run.release(1)
                run.dec.fork([0], [1])
                run.history[1], run.cur[1] = list(run.history[0]), run.cur[0] ^ 1
            run.dec.trim()
            run.dec.check()
    for x, y in zip(_held(runs[0].dec), _held(runs[1].dec)):
        assert torch.equal(x, y)


def test_the_records_of_a_large_pool(cuda_device):
    """Pages behind the first run of the quantisation as well."""

    from oracle import small_cache as o
    from pagelora_b200.bounded_decode import BoundedDecoder

    run = Run(cuda_device, [20], num_pages=9000)  # 4096 pages of 16 tokens, 2 heads a call
    kv = run.dec.e.kv
    for p in (4095, 4096, 8191, 8192, 8999):
        kv[:, p].normal_()
    dec = BoundedDecoder(run.dec.e, kv4=True)
    for li in range(kv.shape[0]):
        for p in (0, 4095, 4096, 8191, 8192, 8999):
            assert (dec.kv4[li, p].cpu().numpy() == o.record_bytes(*o.pack4(kv[li, p].float().cpu().numpy()))).all(), (li, p)
    assert (dec.kv4[:, 4097:8191] == 0).all()


@pytest.mark.parametrize("kv4", [False, True])
def test_a_refused_step_changes_nothing(cuda_device, kv4):
    from pagelora_b200.bounded_decode import Window

    run = Bounded(cuda_device, [96, 40], window=Window(24, 2), kv4=kv4, engine=dict(max_context=96, num_pages=10))
    run.step()  # 7 + 3 pages: all taken
    for _ in range(7):
        run.step()  # the second row's last page is full now
    before, pos = run.state() + list(_held(run.dec)), run.dec.pos.clone()
    nxt, _ = run.dec.step(torch.tensor(run.cur, dtype=torch.int64, device=cuda_device))
    assert (nxt == -1).all()
    run.unchanged(before[:-2], "PL_ERR_POOL_EXHAUSTED")
    assert torch.equal(run.dec.pos, pos) and all(torch.equal(a, b) for a, b in zip(before[-2:], _held(run.dec)))
    run.release(1)
    run.step()
    run.dec.trim()
    run.dec.check()
    run.step()
