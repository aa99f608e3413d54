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



@pytest.mark.parametrize("keys,heads,batch", [(2 ** 30 + 1, 1, 1), (2 ** 31 - 31, 1, 1), (2 ** 31 - 1, 1, 1),
                                              (2 ** 30, 33, 1), (2 ** 30, 1, 33), (2 ** 26, 8, 65)])
def test_more_keys_than_a_tile_index_can_count_are_refused(keys, heads, batch):
    """Tiles of a sequence are (keys + 31) / 32 in an int: behind 2^31 - 32 keys their count would be
    negative, and so would be the places of the list that a merge reads from. The refusal comes before a
    device is looked for, from the size query too."""
    a = _lib.SolortInt4DecodeArgs(AT, 4096, 4096, 128, AT, 4096, 4096, 128, AT, 20480, 2560, 1 << 20, 2048, AT, 2048,
                                  AT, None, batch, 1, heads, heads, 128, keys, 0.1, 0, None, 0, 0)
    need = ctypes.c_size_t(0)
    assert _lib.load().solort_attn_decode_int4(ctypes.byref(a), None) == -2
    assert _lib.load().solort_attn_decode_int4_workspace_size(ctypes.byref(a), ctypes.byref(need)) == -2
