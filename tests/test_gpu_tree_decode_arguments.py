"""What TreeDecoder refuses on the host it refuses before a row has changed,
and a step without tokens changes nothing."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from pagelora_b200.synthetic import ModelSpec

SPEC = ModelSpec("wide-q", 1, 4096, 160, 10, 64, 1024, 4096, 1.0e6, 1e-6)  # 10240 query features


def _engine(**kw):
    return SimpleNamespace(**{**dict(world=1, cascade=None, lora_rank=0, spec=SPEC, page_size=16), **kw})


def test_lora_rows_that_the_shrink_does_not_take():
    from pagelora_b200.tree_decode import TreeDecoder

    with pytest.raises(ValueError, match="8192"):
        TreeDecoder(_engine(lora_rank=16))


@pytest.mark.parametrize("sink,recent,select", [(1, 2, 2), (0, 0, 4), (-1, 1, 4), (0, 1, 0)])
def test_page_budgets(sink, recent, select):
    from pagelora_b200.tree_decode import SparsePages, TreeDecoder

    with pytest.raises(ValueError, match="budget"):
        TreeDecoder(_engine(), sparse=SparsePages(select=select, sink=sink, recent=recent))


@pytest.mark.parametrize("change", [
    dict(page_size=64), dict(spec=ModelSpec("g32", 1, 512, 32, 1, 128, 1024, 4096, 1.0e6, 1e-6)),
])
def test_shapes_that_sparse_decode_does_not_have(change):
    from pagelora_b200.tree_decode import SparsePages, TreeDecoder

    with pytest.raises(ValueError, match="sparse"):
        TreeDecoder(_engine(**change), sparse=SparsePages(select=8))


@pytest.mark.gpu
def test_steps(cuda_device):
    from pagelora_b200.tree_decode import SparsePages
    from test_gpu_tree_decode_refusals import Run

    run = Run(cuda_device, [20, 3, 41], sparse=SparsePages(select=8), max_context=96)
    before = run.state()
    i64 = lambda *a: torch.tensor(a, dtype=torch.int64, device=cuda_device)  # noqa: E731
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda_device)  # noqa: E731
    tok, par, qo = i64(1, 2, 3), i32(-1, 0, -1), i32(0, 2, 2, 3)
    for args, error in (((tok.int(), par, qo, 2), TypeError), ((tok, par.long(), qo, 2), TypeError),
                        ((tok, par, qo.long(), 2), TypeError), ((tok, par[:2], qo, 2), ValueError),
                        ((tok[:2], par, qo, 2), ValueError), ((tok, par, qo[:3], 2), ValueError),
                        ((tok, par, torch.cat([qo, qo[-1:]]), 2), ValueError), ((tok, par, qo, 0), ValueError),
                        ((tok.cpu(), par, qo, 2), RuntimeError), ((tok[None], par, qo, 2), ValueError)):
        with pytest.raises(error):
            run.dec.verify(*args)
    for tokens, error in ((tok.int(), TypeError), (tok[:2], ValueError), (tok.cpu(), RuntimeError)):
        with pytest.raises(error):
            run.dec.step_sparse(tokens)
    for rows in ([3], [-1], [0, 9]):
        with pytest.raises(ValueError):
            run.dec.release(rows)
    for src, dst in (([0], [3]), ([-1], [1]), ([0, 1], [2])):
        with pytest.raises(ValueError):
            run.dec.fork(src, dst)
    run.dec.check()
    assert all(torch.equal(a, b) for a, b in zip(before, run.state()))
    # no row takes part
    res = run.verify([None, None, None], 4)
    run.dec.check()
    assert res.logits.shape == (0, 4096) and res.targets.shape == (0,) and res.keep_count.tolist() == [0, 0, 0]
    assert (res.keep == -1).all() and res.next_token.tolist() == [-1, -1, -1]
    assert all(torch.equal(a, b) for a, b in zip(before, run.state()))
    run.good_step([0, 1, 2])
