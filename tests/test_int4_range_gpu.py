"""4-bit attention over values of any size, and over sizes that differ between tokens.

Tolerance, per element, against the 64-bit sum over the held values: half a bf16 step of the result,
2^-8 |o|; half an f16 step of each p * scale, 2^-11 sum p |v - mid|; those of them that are f16 subnormals,
2^-25 where the row's largest in the group is at least 2^5, for 1024 keys at most 2^-20 of that largest
times 7.5, and a held value lies half a step or more from its mid: 2^-16 sum p |v - mid|; scores and fp32
sums, 2^-10 sum p |v| (derived in test_int4_gpu.py; scores here stay below 100, which the query's group sums,
exact to 2^-17, move by less than 2^-10); a p below 2^-126 counts as zero.
"""

from __future__ import annotations

import pytest
import torch

from oracle import int4 as Q

pytestmark = pytest.mark.gpu

BF, I32, U8 = torch.bfloat16, torch.int32, torch.uint8
P = 16


def _ops():
    from solort_b200 import ops

    return ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _held(g, k, v):
    """An arena with the rows ``k, v [n, nkv, 128]`` as one sequence, its table and slots."""
    n, nkv, _ = k.shape
    pages = _ops().kv_pages_int4(-(-n // P) + 2, nkv, P)
    table = torch.randperm(pages.shape[0], generator=g, device="cuda").to(I32)[None, :-(-n // P)].contiguous()
    slots = Q.slots_of(table[0], n, P)
    _ops().kv_store_int4(k.to(BF), v.to(BF), slots, pages)
    return pages, table, slots


def _check(q, pages, table, slots, scale=128 ** -0.5):
    ops, n, t = _ops(), len(slots), q.shape[1]
    pos = torch.tensor([n - t], device="cuda")
    k, v, m = Q.load(pages, slots, mids=True)
    want, near, size = Q.attention(q[0], k, v, n - t, scale, m)
    tol = (2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -16) * near + 2.0 ** -10 * size +
           2.0 ** -126 * v.abs().amax())
    for ctas in (0, 1, 5):
        out = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n, scale=scale, num_ctas=ctas)
        assert torch.isfinite(out).all(), f"num_ctas {ctas}"
        worst = ((out[0].double() - want).abs() / tol).max().item()
        assert worst <= 1, f"num_ctas {ctas}: {worst:.3g} of the tolerance"
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", [2, 4, 8])
@pytest.mark.parametrize("power", [-100, -60, 60, 100, 103, 106, 110])
def test_values_of_every_magnitude(power, heads):
    g = _gen(power + heads)
    k, v = _randn(g, 300, 1, 128), _randn(g, 300, 1, 128).clamp(-3, 3) * 2.0 ** power
    _check(_randn(g, 1, 1, heads, 128).to(BF), *_held(g, k, v))
