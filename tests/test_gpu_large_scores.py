"""Tree attention where the scores are large: the reference of the online
softmax has to lie near a row's maximum in absolute terms, not relative to its size.

Scores up to 2^17 are exact here: q and K share one large channel whose
product is a multiple of 1/2, a second channel adds multiples of 1/8 up to 4,
and the sums stay below 2^21 of their last bit, so fp32 holds them whatever
the order.  What is left of the error is the rounding of P and of the output
(2^-8 each) and of the exponentials, as for scores of ordinary size:
|err| <= 2^-8 (|o| + sum p |v|) + 2^-12 sum p |v|, LSE within 2^-12 (1 + |lse|).
Beyond, positions differ by more than the exponential's range: a row is the
mean of the V of its highest positions, the same bounds.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import tree_attention as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
F = 2.0 ** -12


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64), dtype=torch.int32, device="cuda")


def _check(K, n, ctx, d, q0, k0, seed, fine=True):
    """One request of n drafted tokens (causal chain), 8 / 2 heads; q0 [n, 8] and k0 [ctx + n] in channel 0, and the
    small products in channel 1 when `fine`."""

    rng = np.random.default_rng(seed)
    ps, hq, hkv, length = 16, 8, 2, ctx + n
    pages = -(-length // ps)
    cache = np.zeros((pages, 2, ps, hkv, d), np.float32)
    flat = cache.transpose(0, 2, 1, 3, 4).reshape(pages * ps, 2, hkv, d).copy()
    flat[:length, 0, :, 0] = k0[:, None]
    if fine:
        flat[:length, 0, :, 1] = rng.integers(-16, 17, size=(length, hkv)) / 8.0
    flat[:length, 1] = rng.normal(size=(length, hkv, d))
    cache = flat.reshape(pages, ps, 2, hkv, d).transpose(0, 2, 1, 3, 4)
    q = np.zeros((n, hq, d), np.float32)
    q[..., 0], q[..., 1] = q0, rng.integers(1, 3, size=(n, hq))
    ct, qt = torch.as_tensor(cache.copy()).to(torch.bfloat16), torch.as_tensor(q).to(torch.bfloat16)
    assert np.array_equal(qt.double().numpy(), q)  # representable
    see = [o.ancestors(list(range(-1, n - 1)))]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full((n, hq), 7.0, device="cuda")
    table = (_i32([0, pages]), _i32(range(pages)), _i32([length - (pages - 1) * ps]))
    out = K.paged_tree_attention(qt.cuda(), ct.cuda(), _i32([0, n]), *table,
                                 torch.as_tensor(o.pack_bits(see[0], -(-n // 32))).cuda(), sm_scale=1.0, out_lse=lse,
                                 status=status)
    assert int(status.item()) == 0
    want, wlse, spread = o.tree_attention(q.astype(np.float64), ct.double().numpy(), [0, n], [0, pages], range(pages),
                                          [length - (pages - 1) * ps], see, sm_scale=1.0)
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= U * (np.abs(want) + spread) + F * spread).all(), np.nanmax(err)
    assert (np.abs(lse.double().cpu().numpy() - wlse) <= F * (1 + np.abs(wlse))).all()


# one row tile per CTA and two; one CTA for all positions and several
SHAPES = [(5, 200, 128), (5, 3000, 64), (64, 300, 128), (64, 2500, 64), (64, 2000, 128)]


@pytest.mark.parametrize("n,ctx,d", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_same_size_everywhere(K, n, ctx, d, sign):
    """|s| from 2^13 to 2^17 by row, every position of a row nearly the same."""

    rng = np.random.default_rng(n + ctx)
    q0 = rng.integers(128, 256, size=(n, 8)) * np.exp2(rng.integers(-1, 2, size=(n, 8)))
    _check(K, n, ctx, d, q0, np.full(ctx + n, sign * 201.0), seed=1)


@pytest.mark.parametrize("n,ctx,d", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_levels_that_change_from_tile_to_tile(K, n, ctx, d, sign):
    level = np.array([130, 129, 200, 131, 255, 255, 128, 254])
    q0 = np.random.default_rng(n).integers(128, 256, size=(n, 8)) * 2.0
    _check(K, n, ctx, d, q0, sign * level[(np.arange(ctx + n) // 128) % 8], seed=2)


@pytest.mark.parametrize("n,ctx,d", SHAPES)
@pytest.mark.parametrize("power", [12, 20, 36, 60, 100])
def test_scores_beyond_the_resolution(K, n, ctx, d, power):
    """Rows of both signs whose scores reach 2^(power + 8): the highest positions take all."""

    rng = np.random.default_rng(power)
    q0 = rng.choice([-1.0, 1.0], size=(n, 8)) * rng.integers(128, 256, size=(n, 8)) * 2.0 ** (power - 8)
    _check(K, n, ctx, d, q0, rng.integers(128, 256, size=ctx + n) * rng.choice([-1.0, 1.0], size=ctx + n), seed=3,
           fine=False)
