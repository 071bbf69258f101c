"""One GEMM workspace for calls of different shapes, in turn: every call finds
its arrival counters at zero whatever ran before, so its result is, bit for
bit, that of a call with a workspace of its own."""

from __future__ import annotations

import pytest
import torch

from pagelora_b200.synthetic import ModelSpec, make_model_weights, random_prompt

pytestmark = pytest.mark.gpu

# 96 row tiles of the vocabulary and 96 of gate_up beside the 8 tiles of q/k/v, o and down
SPEC = ModelSpec("small-wide", 2, 512, 8, 2, 128, 6144, 12288, 1.0e6, 1e-6, qk_norm=True)
LENS = [33, 5, 62, 16, 17, 2, 40, 8, 15, 1]


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


@pytest.mark.parametrize("tokens", [(32, 32), (9, 64), (128, 16)])
def test_narrow_and_wide_products_share_a_workspace(K, tokens):
    g = torch.Generator(device="cuda").manual_seed(5)
    calls, need = [], 0
    for t, n, k in ((tokens[0], 6144, 1024), (tokens[1], 24576, 1024), (tokens[0], 640, 4096), (tokens[1], 20000, 520)):
        x = torch.randn(t, k, generator=g, device="cuda").bfloat16()
        w = (torch.randn(n, k, generator=g, device="cuda") * 0.03).bfloat16()
        calls.append((x, w, K.linear_lora_gemm(x, w)))
        need = max(need, int(K.gemm_plan(t, k, n).workspace_bytes))
    shared = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        for x, w, want in calls:
            out = torch.full_like(want, float("nan"))
            K.linear_lora_gemm(x, w, out=out, workspace=shared)
            assert torch.equal(out, want), tuple(w.shape)


def _engine(device):
    from pagelora_b200.batch_engine import BatchDecodeEngine

    w = {k: v.bfloat16() for k, v in make_model_weights(SPEC, seed=0, dtype=torch.float32, norm_jitter=0.1).items()}
    eng = BatchDecodeEngine(SPEC, dict(w), adapters=None, lora_spec=None, row_adapter=[-1] * len(LENS), page_size=16,
                            max_context=96, device=device)
    return eng, eng.prefill([random_prompt(SPEC.vocab, n, seed=10 + i) for i, n in enumerate(LENS)])


def _own_workspaces(K, monkeypatch):
    """Every product gets a zeroed workspace of its own from here on."""

    shared = K.linear_lora_gemm
    monkeypatch.setattr(K, "linear_lora_gemm", lambda *a, workspace=None, **kw: shared(*a, **kw))


def test_batch_engine_steps(K, cuda_device, monkeypatch):
    def steps():
        eng, cur = _engine(cuda_device)
        for _ in range(2):
            cur = eng.step_host(cur)
        eng._check_status()
        return eng.logits.clone(), cur

    got = steps()
    _own_workspaces(K, monkeypatch)
    want = steps()
    assert torch.equal(got[0], want[0]) and got[1] == want[1]


def test_tree_decoder_steps(K, cuda_device, monkeypatch):
    from pagelora_b200.tree_decode import TreeDecoder

    def step():
        eng, firsts = _engine(cuda_device)
        dec = TreeDecoder(eng)
        n = len(LENS)
        toks = torch.tensor([[f, f ^ 1, f ^ 2] for f in firsts], dtype=torch.int64, device=cuda_device).flatten()
        par = torch.tensor([-1, 0, 0] * n, dtype=torch.int32, device=cuda_device)
        qo = torch.arange(n + 1, dtype=torch.int32, device=cuda_device) * 3
        dec.verify(toks, par, qo, 3)
        res = dec.verify(toks, par, qo, 3)
        dec.check()
        return res.logits, res.targets

    got = step()
    _own_workspaces(K, monkeypatch)
    want = step()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
