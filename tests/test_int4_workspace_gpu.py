"""The workspace of 4-bit attention over models of different head counts."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, I32, U8 = torch.bfloat16, torch.int32, torch.uint8


def _ops():
    from solort_b200 import ops

    return ops


@pytest.mark.parametrize("nh,nkv", [(32, 8), (16, 2), (5, 1), (64, 8), (14, 2), (8, 8)])
def test_it_never_shrinks_at_given_head_counts(nh, nkv):
    size = _ops().decode_int4_workspace_bytes
    by = torch.tensor([[[size(b, t, nh, nkv, n) for n in (1, 511, 512, 513, 1400, 5000, 90000)]
                        for t in (1, 2, 3, 5, 9, 17)] for b in (1, 2, 7, 37, 38, 90, 300)])
    for dim in range(3):
        assert (by.diff(dim=dim) >= 0).all()
    assert size(1, 1, nh, nkv, 512) == 0 < size(1, 1, nh, nkv, 513)  # resident at once, up to 512 keys
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    units = 300 * nkv * (1 if nh <= 4 * nkv else -(-nh // nkv // 8))
    assert (size(300, 1, nh, nkv, 512) == 0) == (units <= 2 * sms)


def test_the_greatest_of_two_models_sizes_serves_both_and_a_smaller_one_is_refused():
    ops, g, n = _ops(), torch.Generator("cuda").manual_seed(1), 20000
    models = [(32, 8), (16, 2)]  # four and eight query heads a KV head: the smaller model needs more
    need = [ops.decode_int4_workspace_bytes(1, 1, nh, nkv, n) for nh, nkv in models]
    assert need[0] < need[1]
    ws = torch.empty(max(need), dtype=U8, device="cuda")
    table, pos = torch.arange(n // 16, dtype=I32, device="cuda")[None], torch.tensor([n - 1], device="cuda")
    for nh, nkv in models:
        pages = ops.kv_pages_int4(n // 16, nkv, 16)
        rows = [torch.randn(n, nkv, 128, generator=g, device="cuda").to(BF) for _ in "kv"]
        ops.kv_store_int4(*rows, torch.arange(n, device="cuda"), pages)
        q = torch.randn(1, 1, nh, 128, generator=g, device="cuda").to(BF)
        want = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n)
        assert torch.equal(ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n, workspace=ws), want)
    with pytest.raises(RuntimeError, match="workspace"):
        ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n, workspace=ws[:need[0]])
