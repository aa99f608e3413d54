"""What the HF bridge's mirror refuses, without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from solort_b200 import hf_attention as H
from solort_b200 import ops


@pytest.mark.parametrize("arena", [
    lambda: ops.kv_pages_int4(4, 2, 16, device="cpu"),  # one layer's 4-bit arena
    lambda: torch.stack([ops.kv_pages_int4(4, 2, 16, device="cpu") for _ in range(3)]),  # one for each layer
    lambda: torch.zeros(3, 4, 2, 16, 2, 128, dtype=torch.uint8)])
def test_an_arena_that_the_bridge_cannot_write_is_refused_in_words(arena):
    k = torch.zeros(1, 2, 5, 128, dtype=torch.bfloat16)
    with H.solort_kv_write_context(SimpleNamespace(kv_cache=arena()), [0, 1, 2, 3, 4]):
        with pytest.raises(RuntimeError, match="kv_store_int4"):
            H._mirror_to_solort_kv(SimpleNamespace(layer_idx=0), k, k)


def test_a_forward_without_slots_is_still_skipped():
    k = torch.zeros(1, 2, 5, 128, dtype=torch.bfloat16)
    arena = torch.zeros(3, 4, 2, 16, 2, 128, dtype=torch.bfloat16)
    before = H.attention_snapshot()["mirror_skipped"]
    with H.solort_kv_write_context(SimpleNamespace(kv_cache=arena), []):
        assert H._mirror_to_solort_kv(SimpleNamespace(layer_idx=0), k, k) is None
    assert H.attention_snapshot()["mirror_skipped"] == before + 1
