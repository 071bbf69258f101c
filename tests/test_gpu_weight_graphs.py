"""Weights and selections captured into a graph and replayed, over tables that
change between replays, and beside one another on two streams."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_window_attention import _case, _i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


class Calls:
    """A prompt's weights, a decode step's, and the choice after them, with buffers of its own."""

    def __init__(self, K, lens, n, seed):
        self.K, rows = K, len(lens)
        _, self.p = _case(lens, n, 8, 2, 64, 16, seed)
        self.q = torch.randn(rows, 8, 64, device="cuda").bfloat16()
        self.tables = (self.p["indptr"], self.p["indices"], self.p["last"])
        self.lse = torch.empty(sum(n), 8, device="cuda")
        K.paged_prefill(self.p["q"], self.p["cache"], self.p["qo"], *self.tables, out_lse=self.lse)
        self.lens = _i32(lens)
        total = self.p["indices"].numel()
        self.ws = [torch.full((b,), 255, dtype=torch.uint8, device="cuda") for b in
                   (K._prefill_weights_workspace_bytes(2, 16, total), K._decode_weights_workspace_bytes(rows, 8, 2, 64, 16, total))]
        self.weight = torch.zeros(rows, max(lens), device="cuda")
        self.moved, self.out = torch.zeros_like(self.weight), torch.zeros_like(self.q)
        self.keep = torch.zeros(rows, 46, dtype=torch.int32, device="cuda")
        self.keep_from, self.count = torch.zeros_like(self.lens), torch.zeros_like(self.lens)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(self):
        K, p = self.K, self.p
        K.paged_prefill_weights(p["q"], p["cache"], p["qo"], *self.tables, self.lse, self.weight, workspace=self.ws[0],
                                status=self.status)
        K.paged_decode_weights(self.q, p["cache"], *self.tables, self.weight, out=self.out, workspace=self.ws[1],
                               status=self.status)
        K.evict_select(self.weight, self.lens, 50, sinks=4, recent=10, keep_from=self.keep_from, keep=self.keep,
                       keep_count=self.count, out_weight=self.moved, status=self.status)

    def results(self):
        torch.cuda.synchronize()
        assert int(self.status.item()) == 0
        return [t.clone() for t in (self.weight, self.out, self.keep, self.keep_from, self.count, self.moved)]

    def capture(self):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.run()
        return graph

    def replayed(self, graph):
        self.weight.zero_()
        graph.replay()
        return self.results()

    def plainly(self):
        self.weight.zero_()
        self.run()
        return self.results()


def _same(a, b):
    """The same bits (the second lengths reach a row's slots of NaN, and NaN does not equal itself)."""

    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def test_replays_over_other_lengths(K):
    calls = Calls(K, [300, 64, 161], [100, 64, 5], 3)
    first = calls.plainly()
    graph = calls.capture()
    assert _same(calls.replayed(graph), first) and _same(calls.replayed(graph), first)
    calls.p["last"].copy_(_i32([1, 3, 16]))        # 289, 51 and 176 positions
    calls.p["qo"].copy_(_i32([0, 20, 71, 74]))     # 20, 51 and 3 tokens
    calls.lens.copy_(_i32([289, 51, 161]))
    second = calls.replayed(graph)
    assert _same(second, calls.plainly()) and not torch.equal(second[0], first[0])


def test_two_graphs_and_two_streams(K):
    calls = [Calls(K, [300, 64, 161], [100, 64, 5], 3), Calls(K, [700, 90], [512, 1], 4)]
    want = [c.plainly() for c in calls]
    graphs = [c.capture() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for captured in (True, False, True):
        for c in calls:
            c.weight.zero_()
        torch.cuda.synchronize()
        for c, g, s in zip(calls, graphs, streams):
            with torch.cuda.stream(s):
                g.replay() if captured else c.run()
        for c, w in zip(calls, want):
            assert _same(c.results(), w), captured
