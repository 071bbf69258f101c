"""The operators that keep a cache small, without a GPU: what their C entries
refuse before they touch the device, and the oracles against brute force."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import small_cache as o
from test_cache_ops_host import P, capi  # noqa: F401  (a fixture)

DECODE = dict(q=P, q_sb=1024, q_sh=128, kv=P, pages=100, indptr=P, indices=P, last=P, total_pages=100, batch=2, hq=8, hkv=2,
              d=128, ps=16, scale=0.1, window=50, sinks=2, out=P, o_sb=1024, o_sh=128, lse=None, ws=P, ws_bytes=1 << 40,
              status=None, stream=None)
PREFILL = dict(q=P, q_st=1024, q_sh=128, kv=P, pages=100, qo=P, kvp=P, kvi=P, last=P, batch=2, total_q=8, hq=8, hkv=2, d=128,
               ps=16, scale=0.1, window=50, sinks=2, out=P, o_st=1024, o_sh=128, lse=None, status=None, stream=None)
APPEND = dict(k=P, k_st=256, v=P, v_st=256, kv=P, pages=100, page=P, off=P, n=4, hkv=2, d=128, ps=16, status=None, stream=None)
EXPAND = dict(kv=P, pages=100, ids=P, n=3, hkv=2, d=128, ps=16, out=P, status=None, stream=None)
DWEIGHTS = dict(q=P, q_sb=1024, q_sh=128, kv=P, pages=100, indptr=P, indices=P, last=P, total_pages=100, batch=2, hq=8, hkv=2,
                d=128, ps=16, scale=0.1, out=P, o_sb=1024, o_sh=128, lse=None, weight=P, w_stride=60, cap=60, ws=P,
                ws_bytes=1 << 40, status=None, stream=None)
PWEIGHTS = dict(q=P, q_st=1024, q_sh=128, kv=P, pages=100, qo=P, kvp=P, kvi=P, last=P, total_pages=100, batch=2, total_q=8,
                hq=8, hkv=2, d=128, ps=16, scale=0.1, lse=P, weight=P, w_stride=60, cap=60, ws=P, ws_bytes=1 << 40,
                status=None, stream=None)
SELECT = dict(weight=P, w_stride=60, cap=60, lens=P, rows=3, budget=20, sinks=2, recent=5, keep_from=P, keep=P, k_stride=18,
              k_width=18, count=P, out=2 * P, o_stride=60, status=None, stream=None)

LINE = [dict(q=None), dict(kv=None), dict(indptr=None), dict(indices=None), dict(last=None), dict(out=None), dict(batch=-1),
        dict(pages=0), dict(total_pages=-1), dict(hkv=3), dict(hkv=0), dict(scale=0.0), dict(scale=float("nan")),
        dict(q=P + 2), dict(kv=P + 8), dict(out=P + 4), dict(q_sb=1023), dict(o_sh=4)]
WEIGHT = [dict(weight=None), dict(cap=-1), dict(w_stride=59)]
INVALID = {
    "pl_paged_window_decode": (DECODE, LINE + [dict(window=0), dict(window=-1), dict(sinks=-1)]),
    "pl_paged_kv4_decode": (DECODE, LINE + [dict(window=-1), dict(sinks=-1)]),
    "pl_paged_window_prefill": (PREFILL, [
        dict(q=None), dict(kv=None), dict(qo=None), dict(kvp=None), dict(kvi=None), dict(last=None), dict(out=None),
        dict(batch=-1), dict(total_q=-1), dict(pages=0), dict(hkv=3), dict(scale=0.0), dict(window=0), dict(sinks=-1),
        dict(q=P + 2), dict(q_st=1023)]),
    "pl_kv4_append": (APPEND, [dict(k=None), dict(v=None), dict(kv=None), dict(page=None), dict(off=None), dict(n=-1),
                               dict(pages=0), dict(hkv=0), dict(ps=0), dict(k=P + 2), dict(v_st=255), dict(kv=P + 8)]),
    "pl_kv4_expand": (EXPAND, [dict(kv=None), dict(ids=None), dict(out=None), dict(n=-1), dict(pages=0), dict(out=P + 8)]),
    "pl_paged_decode_weights": (DWEIGHTS, LINE + WEIGHT),
    "pl_paged_prefill_weights": (PWEIGHTS, WEIGHT + [
        dict(q=None), dict(kv=None), dict(qo=None), dict(kvp=None), dict(kvi=None), dict(last=None), dict(lse=None),
        dict(batch=-1), dict(total_q=-1), dict(pages=0), dict(hkv=3), dict(scale=-1.0), dict(q=P + 2), dict(q_st=0),
        dict(q_sh=1)]),
    "pl_evict_select": (SELECT, [
        dict(weight=None), dict(lens=None), dict(keep_from=None), dict(keep=None), dict(count=None), dict(out=None),
        dict(out=P), dict(rows=-1), dict(cap=-1), dict(sinks=-1), dict(recent=-1), dict(recent=19), dict(k_width=17),
        dict(k_stride=17), dict(w_stride=59), dict(o_stride=59), dict(budget=-1)]),
}


@pytest.mark.parametrize("fn", INVALID)
def test_invalid_arguments(capi, fn):  # noqa: F811
    c, lib = capi
    args, bad = INVALID[fn]
    for change in bad:
        got = getattr(lib, fn)(*dict(args, **change).values())
        assert got == c.PL_ERR_INVALID_ARGUMENT, (change, got)


@pytest.mark.parametrize("fn,args", [("pl_paged_window_decode", DECODE), ("pl_paged_kv4_decode", DECODE),
                                     ("pl_paged_decode_weights", DWEIGHTS), ("pl_paged_window_prefill", PREFILL),
                                     ("pl_paged_prefill_weights", PWEIGHTS)])
def test_unsupported_shapes(capi, fn, args):  # noqa: F811
    c, lib = capi
    for change in (dict(d=96), dict(ps=24), dict(ps=256), dict(hq=258)):
        assert getattr(lib, fn)(*dict(args, **change).values()) == c.PL_ERR_UNSUPPORTED, change
    if "total_pages" in args:  # positions that 32 bits do not hold
        assert getattr(lib, fn)(*dict(args, total_pages=1 << 27).values()) == c.PL_ERR_UNSUPPORTED
    assert lib.pl_kv4_append(*dict(APPEND, d=96).values()) == c.PL_ERR_UNSUPPORTED
    assert lib.pl_kv4_expand(*dict(EXPAND, d=256).values()) == c.PL_ERR_UNSUPPORTED


def test_workspaces_that_are_too_small(capi):  # noqa: F811
    c, lib = capi
    for fn, args, need in (
            ("pl_paged_window_decode", DECODE, lib.pl_window_decode_workspace_bytes(8, 2, 128)),
            ("pl_paged_kv4_decode", DECODE, lib.pl_kv4_decode_workspace_bytes(8, 2, 128)),
            ("pl_paged_decode_weights", DWEIGHTS, lib.pl_decode_weights_workspace_bytes(2, 8, 2, 128, 16, 100)),
            ("pl_paged_prefill_weights", PWEIGHTS, lib.pl_prefill_weights_workspace_bytes(2, 16, 100))):
        assert need > 0
        for change in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=P + 8)):
            assert getattr(lib, fn)(*dict(args, **change).values()) == c.PL_ERR_WORKSPACE_TOO_SMALL, (fn, change)


def test_empty_calls_do_nothing(capi):  # noqa: F811
    _, lib = capi
    for fn, args, change in (("pl_paged_window_decode", DECODE, dict(batch=0, q=None, out=None, ws=None)),
                             ("pl_paged_kv4_decode", DECODE, dict(batch=0, q=None, out=None, ws=None)),
                             ("pl_paged_window_prefill", PREFILL, dict(total_q=0)),
                             ("pl_paged_decode_weights", DWEIGHTS, dict(batch=0, q=None, ws=None)),
                             ("pl_paged_prefill_weights", PWEIGHTS, dict(total_q=0, q=None, lse=None, ws=None)),
                             ("pl_kv4_append", APPEND, dict(n=0, k=None, page=None)),
                             ("pl_kv4_expand", EXPAND, dict(n=0, ids=None, out=None)),
                             ("pl_evict_select", SELECT, dict(rows=0, lens=None, keep=None))):
        assert getattr(lib, fn)(*dict(args, **change).values()) == 0, fn


def test_records_of_the_oracle():
    rng = np.random.default_rng(1)
    x = o.to_bf16(rng.normal(size=(5, 3, 64)) * 3)
    code, scale, low = o.pack4(x)
    rec = o.record_bytes(code, scale, low)
    assert rec.shape == (5, 3, 48)
    val, sc, cd = o.unpack4(rec)
    assert (cd + 8 == code).all()
    for c in range(64):  # channel c is of group c % 4
        grp = x[..., c % 4::4]
        assert (sc[..., c] == scale[..., c % 4]).all() and (low[..., c % 4] == grp.min(-1)).all()
        assert (np.abs(sc[..., c] - (grp.max(-1) - grp.min(-1)) / 15) <= sc[..., c] * 2.0 ** -8).all()
    assert (np.abs(val - x) <= sc * (0.5 + 15 * 2.0 ** -9)).all()
    flat = o.pack4(np.full((2, 64), 1.25, np.float32))
    assert (flat[0] == 0).all() and (flat[1] == 0).all() and (o.unpack4(o.record_bytes(*flat))[0] == 1.25).all()


def test_window_of_the_oracle():
    for n in (1, 5, 20):
        for p in range(n):
            for window, sinks in ((1, 0), (3, 2), (50, 0), (2, 50)):
                want = [j <= p and (p - j < window or j < sinks) for j in range(n)]
                assert list(o.visible(p, n, window, sinks)) == want
    q, kv = np.ones((4, 8)), np.arange(2 * 3 * 2 * 8).reshape(2, 3, 2, 8) * 0.01
    out, lse, p, spread = o.attend(q, kv[0], kv[1], np.zeros(3, bool), 1.0)
    assert (out == 0).all() and np.isneginf(lse).all() and (p == 0).all()
    out, lse, p, _ = o.attend(q, kv[0], kv[1], np.array([True, False, True]), 1.0)
    s = kv[0][[0, 2], 0].sum(-1)
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[1], w @ kv[1][[0, 2], 0]) and np.allclose(p[0], [w[0], 0, w[1]])
    assert np.allclose(lse[0], np.log(np.exp(s).sum()))


def test_selection_of_the_oracle():
    w = [9.0, 0.1, 0.5, 0.5, 0.2, np.nan, 0.5, 9.0, 9.0]
    assert list(o.select(w, 9, 9, 1, 2)) == list(range(9))
    assert list(o.select(w, 9, 5, 1, 2)) == [0, 2, 5, 7, 8]  # NaN above all, the lower of equals
    assert list(o.select(w, 9, 3, 1, 2)) == [0, 7, 8]
    assert list(o.select(w, 9, 4, 0, 0)) == [0, 5, 7, 8]
