"""What the 4-bit calls refuse at the ends of their ranges, without a GPU."""

from __future__ import annotations

import ctypes

import pytest

from solort_b200 import _lib

AT = 1 << 20  # an address that is never read


def _store(tokens: int) -> int:
    a = _lib.SolortInt4StoreArgs(AT, AT, 1024, 128, 1024, 128, tokens, 1, 128, AT, AT, 20480, 2560, 16, 64)
    return _lib.load().solort_attn_kv_store_int4(ctypes.byref(a), None)


@pytest.mark.parametrize("tokens", [2 ** 30 + 1, 2 ** 31 - 37888, 2 ** 31 - 1])
def test_a_store_of_more_rows_than_its_rounds_can_count_is_refused(tokens):
    """A CTA of the store goes on by its grid's rows, up to 148 * 16 / 2 CTAs of 32 for one KV head: behind
    2^31 less these the next row's index would come out negative and pass for one of the call's. The refusal
    comes before anything looks for a device."""
    assert _store(tokens) == -2

