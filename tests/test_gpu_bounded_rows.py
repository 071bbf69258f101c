"""What a BoundedDecoder's rows hold: budgets, windows that give back what no
later token sees, and the pool that a 4-bit cache leaves unused."""

from __future__ import annotations

import pytest

from test_gpu_tree_decode_refusals import Run

pytestmark = pytest.mark.gpu


def test_a_budget_keeps_a_token(cuda_device):
    """A row that keeps nothing would be one without a context, which takes no part in steps."""

    from pagelora_b200.bounded_decode import BoundedDecoder, EvictBudget

    run = Run(cuda_device, [20])
    with pytest.raises(ValueError):
        BoundedDecoder(run.dec.e, evict=EvictBudget(0, sinks=0, recent=0))
    BoundedDecoder(run.dec.e, evict=EvictBudget(1, sinks=0, recent=0))
