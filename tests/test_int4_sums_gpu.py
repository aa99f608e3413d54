"""The sums of 4-bit attention over many keys a warp keep fp32's accuracy.

Scores are small, so that all keys weigh about the same and every rounding of a key's own is independent of the
others': in the mean they shrink with the number of keys, and what would be left is a sum that is cut off. The
partial results, fp32, are read from the workspace, before the last rounding to bf16.

Tolerance per element, eight standard deviations of each independent error and the whole of the others:
* f16 roundings of p * scale, 2^-11 / sqrt(3) each: 8 * 2^-11 / sqrt(3) * sqrt(sum p^2 (v - mid)^2);
* scores, 2^-13 each (2^-10 for |q| scale <= 8, derived in test_int4_gpu.py; |q| scale is below 1 here):
  8 * 2^-13 * sqrt(sum p^2 v^2);
* the running sums of x c and 7.5 x, N tiles in each of W warps: an addition is off by a step / sqrt(12) of a
  sum that grows to S = 7.5 scale, steps are 2^-23 of it at most, so 2^-23 S sqrt(N) / 6 each, two sums, W warps:
  8 * 2^-23 * 7.5 scale * sqrt(2 N / W) / 6;
* a tile's own sum in the tensor cores, which cut off: 2^-21 * 7.5 scale, twice.
scale: the mean over the keys.
"""

from __future__ import annotations

import pytest
import torch

from oracle import int4 as Q

pytestmark = pytest.mark.gpu

BF, I32, U8 = torch.bfloat16, torch.int32, torch.uint8


@pytest.mark.parametrize("heads,n,ctas", [(4, 60000, 2), (8, 60000, 2), (4, 1 << 20, 2), (8, 1 << 20, 2),
                                          (8, 1 << 20, 20), (2, 300001, 1), (4, 3 << 20, 1), (8, 3 << 20, 1)])
def test_means_of_many_values(heads, n, ctas):
    from solort_b200 import ops

    g, P = torch.Generator("cuda").manual_seed(n + heads), 64
    held = 937 * P  # tokens in the arena; the block table lists its pages again and again
    pages = ops.kv_pages_int4(held // P, 1, P)
    k, v = (torch.randn(held, 1, 128, generator=g, device="cuda").to(BF) for _ in "kv")
    ops.kv_store_int4(k, v, torch.arange(held, device="cuda"), pages)
    of = torch.arange(-(-n // P), dtype=I32, device="cuda") % pages.shape[0]
    q = (torch.randn(1, 1, heads, 128, generator=g, device="cuda") / 8).to(BF)
    ws = torch.zeros(ops.decode_int4_workspace_bytes(1, 1, heads, 1, n, num_ctas=ctas), dtype=U8, device="cuda")
    out = ops.gqa_decode_paged_int4(q, pages, of[None], torch.tensor([n - 1], device="cuda"), max_kv_len=n,
                                    num_ctas=ctas, workspace=ws)
    torch.cuda.synchronize()

    hk, hv, mid = (x[:, 0] for x in Q.load(pages, torch.arange(held, device="cuda"), mids=True))
    times = torch.bincount(torch.arange(n, device="cuda") % held, minlength=held).double()
    p = torch.softmax(q[0, 0].double() @ hk.T * 128 ** -0.5 + times.log(), -1)
    want = p @ hv
    scale = Q.quantise(v[:, 0])[1].double().mean(0).repeat_interleave(32)
    tiles, warps = n / 32 / (6 * ctas), 6 * ctas
    tol = (8 * 2.0 ** -11 / 3 ** 0.5 * (p ** 2 @ (hv - mid) ** 2).sqrt() + 8 * 2.0 ** -13 * (p ** 2 @ hv ** 2).sqrt() +
           8 * 2.0 ** -23 * 7.5 * scale * (2 * tiles / warps) ** 0.5 / 6 + 2.0 ** -20 * 7.5 * scale)
    if ctas > 1:
        rows = 4 if heads <= 4 else 8
        o = ws[:2 * ctas * rows * 512].view(torch.float32).view(2 * ctas, rows, 128)[::2, :heads].double()
        ml = ws[2 * ctas * rows * 512:][:2 * ctas * rows * 8].view(torch.float32).view(2 * ctas, rows, 2)[::2, :heads].double()
        got = (o * ml[..., :1].exp2()).sum(0) / (ml[..., 1:] * ml[..., :1].exp2()).sum(0)
    else:  # one CTA writes the rows itself
        got = out[0, 0].double()
        tol = tol + 2.0 ** -8 * want.abs()
    worst = ((got - want).abs() / tol).max().item()
    print(f"{worst:.3g} of the tolerance")
    assert worst <= 1, f"{worst:.3g} of the tolerance"
    assert ops.device_status() == 0


def test_no_bias_in_any_place_of_a_code():
    """The mean error over the dims of one place in a half word, over 8 heads, against eight deviations of it: an
    element's is 2^-11 / sqrt(3) sqrt(sum p^2 (v - mid)^2) from f16 and 2^-10 sqrt(sum p^2 v^2) from its scores
    (|q| scale <= 8), dims are independent of each other but for the two or three nibbles of a group that share
    the f16 rounding, times factors (v - mid) of either sign."""
    from solort_b200 import ops

    g, P, n, heads, ctas = torch.Generator("cuda").manual_seed(7), 64, 1 << 19, 8, 60
    pages = ops.kv_pages_int4(n // P, 1, P)
    k, v = (torch.randn(n, 1, 128, generator=g, device="cuda").to(BF) for _ in "kv")
    at = torch.arange(n, device="cuda")
    ops.kv_store_int4(k, v, at, pages)
    q = (torch.randn(1, 1, heads, 128, generator=g, device="cuda") * 1.5).to(BF)  # weights e^(1.5 x), x normal
    ws = torch.zeros(ops.decode_int4_workspace_bytes(1, 1, heads, 1, n, num_ctas=ctas), dtype=U8, device="cuda")
    ops.gqa_decode_paged_int4(q, pages, (at[:n // P]).to(I32)[None], torch.tensor([n - 1], device="cuda"), max_kv_len=n,
                              num_ctas=ctas, workspace=ws)
    torch.cuda.synchronize()
    o = ws[:2 * ctas * 8 * 512].view(torch.float32).view(2 * ctas, 8, 128)[::2].double()
    ml = ws[2 * ctas * 8 * 512:][:2 * ctas * 8 * 8].view(torch.float32).view(2 * ctas, 8, 2)[::2].double()
    w = (ml[..., :1] - ml[..., :1].amax(0)).exp2()
    got = (o * w).sum(0) / (ml[..., 1:] * w).sum(0)
    hk, hv, mid = (x[:, 0] for x in Q.load(pages, at, mids=True))
    p = torch.softmax(q[0, 0].double() @ hk.T * 128 ** -0.5, -1)
    off = (got - p @ hv).view(heads, 32, 4)
    each = 2.0 ** -11 / 3 ** 0.5 * (p ** 2 @ (hv - mid) ** 2).sqrt() + 2.0 ** -10 * (p ** 2 @ hv ** 2).sqrt()
    tol = 8 * each.view(heads, 32, 4).square().mean((0, 1)).sqrt() / (heads * 32) ** 0.5
    mean = off.mean((0, 1))
    print(mean.tolist(), tol.tolist())
    assert (mean.abs() <= tol).all()
