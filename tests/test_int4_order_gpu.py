"""Flagged 4-bit attention behind the calls that write its keys, with no synchronisation in between.

The cache is filled with NaN scales first, so that a key read before it was written shows in the output;
the flag changes when loads are issued and not what is computed, so the outputs have the bits of the same
calls without it.
"""

from __future__ import annotations

import pytest
import torch

from oracle import attention as A
from oracle import int4 as Q

pytestmark = pytest.mark.gpu

BF, I32, I64, U8 = torch.bfloat16, torch.int32, torch.int64, torch.uint8
EPS, P = 1e-6, 16


def _ops():
    from solort_b200 import ops

    return ops


def _setup(seed, batch, top, nh, nkv):
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-top // P)
    table = torch.randperm(batch * per, generator=g, device="cuda").to(I32).view(batch, per)
    qn, kn = ((1 + 0.1 * torch.randn(128, generator=g, device="cuda")).to(BF) for _ in "qk")
    cos, sin = A.cos_sin(torch.arange(top, device="cuda"), A.inv_freq(128, 1e6, "cuda"), BF)
    return g, table, qn, kn, cos, sin


@pytest.mark.parametrize("n,nh,nkv", [(32, 2, 1), (96, 8, 2), (1024, 32, 8), (6016, 32, 8)])
def test_a_stored_prefix_an_append_and_a_flagged_call(n, nh, nkv):
    """``n`` rows are stored, one token is appended, and the call reads them all: the store is the kernel
    before the one before it."""
    ops = _ops()
    g, table, qn, kn, cos, sin = _setup(n, 1, n + 1, nh, nkv)
    slots = Q.slots_of(table[0], n + 1, P)
    pages = ops.kv_pages_int4(table.numel(), nkv, P)
    pos = torch.tensor([n], device="cuda")
    ws = torch.empty(ops.decode_int4_workspace_bytes(1, 1, nh, nkv, n + 1), dtype=U8, device="cuda")
    rows = [[torch.randn(n, nkv, 128, generator=g, device="cuda").to(BF) for _ in "kv"] for _ in range(3)]
    qkv = [torch.randn(1, (nh + 2 * nkv) * 128, generator=g, device="cuda").to(BF) for _ in range(3)]
    q = torch.zeros(1, nh, 128, dtype=BF, device="cuda")
    first, last, outs = slots[:n].contiguous(), slots[n:].contiguous(), {}
    for flag in (False, True):
        got = outs[flag] = [torch.zeros(1, 1, nh, 128, dtype=BF, device="cuda") for _ in range(30)]
        torch.cuda.synchronize()
        for i, out in enumerate(got):
            pages.fill_(0xFF)
            k, v = rows[i % 3]
            ops.kv_store_int4(k, v, first, pages)
            ops.qk_norm_rope_append_int4(qkv[i % 3], qn, kn, EPS, cos, sin, pos, last, pages, num_qo_heads=nh,
                                         num_kv_heads=nkv, q_out=q)
            ops.gqa_decode_paged_int4(q[:, None], pages, table, pos, max_kv_len=n + 1, out=out, workspace=ws,
                                      stable_prefix=flag)
        torch.cuda.synchronize()
    for a, b in zip(outs[False], outs[True]):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert ops.device_status() == 0


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("batch,nh,nkv", [(1, 2, 1), (3, 16, 8)])
def test_steps_back_to_back(batch, nh, nkv, captured):
    """Appends and flagged calls in turn, with nothing between the steps: where ``q_pos`` is a multiple of
    32, the last token of the tile that is read first was appended by the step before."""
    ops = _ops()
    first, steps = 61, 70
    top = first + steps
    g, table, qn, kn, cos, sin = _setup(batch, batch, top, nh, nkv)
    slots = torch.stack([Q.slots_of(table[b], top, P) for b in range(batch)])
    pages = ops.kv_pages_int4(table.numel(), nkv, P)
    k, v = (torch.randn(batch * first, nkv, 128, generator=g, device="cuda").to(BF) for _ in "kv")
    qkv = torch.randn(steps, batch, (nh + 2 * nkv) * 128, generator=g, device="cuda").to(BF)
    at = [torch.full((batch,), first + i, dtype=I64, device="cuda") for i in range(steps)]
    to = [slots[:, first + i].contiguous() for i in range(steps)]
    q = torch.zeros(batch, nh, 128, dtype=BF, device="cuda")
    ws = torch.empty(ops.decode_int4_workspace_bytes(batch, 1, nh, nkv, top), dtype=U8, device="cuda")
    outs = {f: torch.zeros(steps, batch, 1, nh, 128, dtype=BF, device="cuda") for f in (False, True)}
    before = slots[:, :first].reshape(-1)

    def run(flag):
        for i in range(steps):
            ops.qk_norm_rope_append_int4(qkv[i], qn, kn, EPS, cos, sin, at[i], to[i], pages, num_qo_heads=nh,
                                         num_kv_heads=nkv, q_out=q)
            ops.gqa_decode_paged_int4(q[:, None], pages, table, at[i], max_kv_len=top, out=outs[flag][i],
                                      workspace=ws, stable_prefix=flag)

    for flag in (False, True):
        call = lambda: run(flag)  # noqa: E731
        if captured:
            call()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                run(flag)
            call = graph.replay
        for _ in range(3):
            pages.fill_(0xFF)
            outs[flag].zero_()
            ops.kv_store_int4(k, v, before, pages)
            torch.cuda.synchronize()
            call()
        torch.cuda.synchronize()
    assert torch.isfinite(outs[False]).all() and torch.equal(outs[False], outs[True])
    held_k, held_v, mid = Q.load(pages, slots[0], mids=True)
    want, near, size = Q.attention(q[:1], held_k, held_v, top - 1, 128 ** -0.5, mid)
    # the last step of the first sequence: a bf16 rounding and what test_int4_gpu.py derives
    off = (outs[True][-1, :1, 0].double() - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * near + 2.0 ** -10 * size + 1e-30).all()
    assert ops.device_status() == 0
