"""Refusals of the cache operators' C entries, without a GPU (beside those of
test_cache_ops_host.py)."""

from __future__ import annotations

from test_cache_ops_host import RESERVE, capi  # noqa: F401  (a fixture)


def test_a_reservation_of_tokens_for_no_rows(capi):  # noqa: F811
    c, lib = capi
    assert lib.pl_page_reserve(*dict(RESERVE, rows=0, total=0).values()) == 0
    assert lib.pl_page_reserve(*dict(RESERVE, rows=0, total=8).values()) == c.PL_ERR_INVALID_ARGUMENT
