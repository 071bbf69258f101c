"""TreeDecoder (drafted trees, forks, sparse steps over a batch engine's
cache) against per-row oracle decoders.

The logits bound is the one of the batch engine's own tests (max |err| < 0.1
over the small models' logits).  After every step the oracle is fed the
tokens that the decoder accepted, so each step also checks what the last one
left in the cache.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import tree_attention as o_tree
from oracle.decoder import OracleDecoder
from pagelora_b200.synthetic import LoRASpec, ModelSpec, make_lora_weights, make_model_weights, random_prompt

pytestmark = pytest.mark.gpu

QWEN = ModelSpec("small-qwen3", 2, 512, 8, 2, 128, 1024, 4096, 1.0e6, 1e-6, qk_norm=True)
LLAMA = ModelSpec("small-llama2-mha", 2, 512, 8, 8, 64, 1024, 4096, 10000.0, 1e-5)
LORA = LoRASpec(16, 32.0, ("q", "k", "v", "o"), num_adapters=2)


def _engine(spec, row_adapter, lens, device, max_context=192):
    from pagelora_b200.batch_engine import BatchDecodeEngine

    w = {k: v.bfloat16() for k, v in make_model_weights(spec, seed=0, dtype=torch.float32, norm_jitter=0.1).items()}
    adapters = [make_lora_weights(spec, LORA, adapter=a, dtype=torch.bfloat16) for a in range(2)]
    used = adapters if max(row_adapter) >= 0 else None
    eng = BatchDecodeEngine(spec, dict(w), adapters=used, lora_spec=LORA, row_adapter=row_adapter, page_size=16,
                            max_context=max_context, device=device)
    eng.shuffle_free_pages(seed=4)
    prompts = [random_prompt(spec.vocab, n, seed=10 + i) for i, n in enumerate(lens)]
    firsts = eng.prefill(prompts)

    def oracle(row, tokens):
        ad = row_adapter[row]
        lo = None if ad < 0 or used is None else {k: (a.float(), b.float()) for k, (a, b) in adapters[ad].items()}
        o = OracleDecoder(spec, {k: v.float() for k, v in w.items()}, lo, LORA.scale, page_size=16,
                          num_pages=max_context // 16 + 2, bf16=True)
        lg = None
        for t in tokens:
            _, lg = o.step(t)
        return lg

    return eng, prompts, firsts, oracle


def _draft(rng, oracle, row, history, first, n, vocab):
    """A tree under `first`: a chain of the oracle's own choices with wrong siblings in between."""

    toks, par = [first], [-1]
    seq, tip = history + [first], 0
    for _ in range(n - 1):
        if rng.random() < 0.45:
            par.append(int(rng.integers(0, len(toks))))
            toks.append(int(rng.integers(0, vocab)))
        else:
            nxt = int(np.argmax(oracle(row, seq)))
            par.append(tip)
            tip = len(toks)
            toks.append(nxt)
            seq = seq + [nxt]
    return toks, par


@pytest.mark.parametrize("spec,row_adapter,lens", [
    (QWEN, [-1, -1, -1], [33, 5, 62]),
    (LLAMA, [0, 0, 1], [16, 47, 20]),
    (LLAMA, [-1, 0, 0, 0, 0, 0, 1, 1, 1, 1], [9, 3, 31, 16, 17, 2, 40, 8, 15, 1]),
], ids=["qwen", "lora", "10rows-gemm-lora"])
def test_verified_trees_match_the_oracle(cuda_device, spec, row_adapter, lens):
    from pagelora_b200.tree_decode import TreeDecoder

    eng, prompts, firsts, oracle = _engine(spec, row_adapter, lens, cuda_device)
    dec = TreeDecoder(eng)
    rng = np.random.default_rng(3)
    history = [list(p) for p in prompts]
    cur = list(firsts)
    accepted_more = 0
    for step in range(3):
        sizes = [int(rng.integers(1, 9)) for _ in cur]
        if step == 1:
            sizes[1] = 0  # this row sits the step out
        trees = [_draft(rng, oracle, r, history[r], cur[r], n, spec.vocab) if n else ([], []) for r, n in enumerate(sizes)]
        qo = np.cumsum([0] + sizes)
        dev = dict(device=cuda_device)
        res = dec.verify(torch.tensor(sum([t for t, _ in trees], []), dtype=torch.int64, **dev),
                         torch.tensor(sum([p for _, p in trees], []), dtype=torch.int32, **dev),
                         torch.tensor(qo, dtype=torch.int32, **dev), 12)
        dec.check()
        logits, targets = res.logits.float().cpu().numpy(), res.targets.cpu().numpy()
        for r, (toks, par) in enumerate(trees):
            tgt = targets[qo[r]:qo[r + 1]]
            for i in range(len(toks)):  # every drafted token's logits: its own path after the context
                path, j = [], i
                while j >= 0:
                    path.append(toks[j])
                    j = par[j]
                lg = oracle(r, history[r] + path[::-1])
                assert np.abs(logits[qo[r] + i] - lg).max() < 0.1, (step, r, i)
            path, choice = o_tree.accept(par, toks, tgt)
            assert int(res.keep_count[r]) == len(path) and int(res.next_token[r]) == choice
            assert res.keep[r, : len(path)].tolist() == [len(history[r]) + i for i in path]
            accepted_more += max(0, len(path) - 1)
            if toks:
                history[r] += [toks[i] for i in path]
                cur[r] = choice
        assert dec.lens.tolist() == [len(h) for h in history]
        pages = [-(-len(h) // 16) for h in history]
        assert dec.num.tolist() == pages and int(dec.refcount.sum()) == sum(pages)
    assert accepted_more > 0  # the oracle's choices were taken


def test_fork_release_and_sparse_steps(cuda_device):
    """Forked rows go their own ways; a budget that covers all pages equals dense decode."""

    from pagelora_b200.tree_decode import SparsePages, TreeDecoder

    eng, prompts, firsts, oracle = _engine(QWEN, [-1] * 4, [60, 20, 33, 7], cuda_device)
    dec = TreeDecoder(eng, sparse=SparsePages(select=32))
    dec.release([1, 3])
    dec.fork([0, 2], [3, 1])
    history = [list(prompts[0]), list(prompts[2]), list(prompts[2]), list(prompts[0])]
    cur = [firsts[0], firsts[2] ^ 1, firsts[2], firsts[0] ^ 1]
    for _ in range(20):  # every row passes a page boundary
        nxt, logits = dec.step_sparse(torch.tensor(cur, dtype=torch.int64, device=cuda_device))
        for r in range(4):
            history[r].append(cur[r])
        cur = nxt.tolist()
    dec.check()
    for r in range(4):
        assert np.abs(logits[r].float().cpu().numpy() - oracle(r, history[r])).max() < 0.1, r
    assert dec.lens.tolist() == [len(h) for h in history]
    # bounds are current: those of all held pages equal a fresh computation
    want_b, want_s = dec.bounds.clone(), dec.bound_scale.clone()
    dec._refresh_bounds(torch.zeros_like(dec.num), dec.cap)
    assert torch.equal(want_b, dec.bounds) and torch.equal(want_s, dec.bound_scale)
    with pytest.raises(ValueError):
        TreeDecoder(eng).step_sparse(nxt)
