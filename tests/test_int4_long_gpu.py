"""4-bit attention over many millions of keys: one page of 4096 tokens, again and again in the block table, so
that the result is that of the page's tokens, each as often as it is listed (in 64 bits). Tolerance: as in
test_int4_range_gpu.py; a warp's sums run over 2^26 / 1776 keys, which in fp32 with truncation lose at most
2^-24 of themselves for each of 2400 products of 16 keys, of codes that weigh up to 15 times |v - mid|: 2^-9
sum p |v - mid|."""

from __future__ import annotations

import pytest
import torch

from oracle import int4 as Q

pytestmark = pytest.mark.gpu

BF, I32, P = torch.bfloat16, torch.int32, 4096


@pytest.mark.parametrize("heads,n", [(4, (1 << 22) + 5), (8, (1 << 24) + 4077), (4, (1 << 26) - 1)])
def test_millions_of_keys(heads, n):
    from solort_b200 import ops

    g = torch.Generator("cuda").manual_seed(heads)
    pages = ops.kv_pages_int4(3, 1, P)
    rows = [torch.randn(P, 1, 128, generator=g, device="cuda").to(BF) for _ in "kv"]
    ops.kv_store_int4(*rows, torch.arange(P, 2 * P, device="cuda"), pages)
    table = torch.ones(1, -(-n // P), dtype=I32, device="cuda")
    q = torch.randn(1, 1, heads, 128, generator=g, device="cuda").to(BF)
    out = ops.gqa_decode_paged_int4(q, pages, table, torch.tensor([n - 1], device="cuda"), max_kv_len=n)
    k, v, m = (x[:, 0] for x in Q.load(pages, torch.arange(P, 2 * P, device="cuda"), mids=True))
    often = n // P + (torch.arange(P, device="cuda") < n % P).double()
    p = torch.softmax(q[0, 0].double() @ k.T * 128 ** -0.5 + often.log(), -1)
    want, near, size = p @ v, p @ (v - m).abs(), p @ v.abs()
    off = (out[0, 0].double() - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -16 + 2.0 ** -9) * near + 2.0 ** -10 * size).all()
    assert ops.device_status() == 0
