"""The paged 4-bit KV cache on the GPU against ``oracle.int4`` in 64 bits.

* Store and append write the oracle's bytes, all of them and no others: the steps that decide a code
  are IEEE fp32 operations in a fixed order on both sides, and the mean of squares is fp64.
* Load returns the held values rounded to bf16 exactly (``mid + scale * (code - 7.5)`` has one fp32
  rounding before the bf16 one).
* Attention, per element, against the 64-bit sum over the held values: half a bf16 step of the result,
  2^-8 |o|; half an f16 step of each p * scale, in all at most 2^-11 sum p |v - mid| (below 2^-14 of the
  tile's largest the step is 2^-25 of that, 2^-33 of the row's, which a thousand keys do not add up to
  2^-22); and the fp32 parts. Of these a score's error enters p relatively: a score is a sum of four
  groups, each of products up to 143 |q| scale whose fp32 accumulation loses at most 2^-20 of the largest
  partial sum over its 32 terms, scaled by 128^-0.5: below 2^-9 * 2^-3 for |q| scale <= 8 -- the inputs
  here stay below -- and the accumulation of p scale * code loses 2^-24 of partial sums below 143 / 7.5
  times sum p |v - mid|'s bound per 16-token step. Both are covered by 2^-10 sum p |v|.
"""

from __future__ import annotations

import pytest
import torch

from oracle import attention as A
from oracle import int4 as Q

pytestmark = pytest.mark.gpu

BF, I32, I64, U8 = torch.bfloat16, torch.int32, torch.int64, torch.uint8
EPS = 1e-6


def _ops():
    from solort_b200 import ops

    return ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _garbage(pages):
    """Fill an arena with bytes whose scales and mids are NaN."""
    pages.fill_(0xFF)
    return pages


def _filled(g, lengths, nkv, P, spare=3, k_gain=1.0):
    """Arena, table and per-sequence slots of sequences of ``lengths`` held tokens; every byte that
    holds none of them is NaN garbage."""
    ops = _ops()
    counts = [max(1, -(-n // P)) for n in lengths]
    pages = _garbage(ops.kv_pages_int4(sum(counts) + spare, nkv, P))
    order = torch.randperm(sum(counts) + spare, generator=g, device="cuda")
    table = torch.full((len(lengths), max(counts)), -7, dtype=I32, device="cuda")  # never looked at
    slots, at = [], 0
    for b, (n, c) in enumerate(zip(lengths, counts)):
        table[b, :c] = order[at:at + c]
        at += c
        slots.append(Q.slots_of(table[b], n, P))
        if n:
            Q.store(pages, slots[-1], (_randn(g, n, nkv, 128) * k_gain).to(BF), _randn(g, n, nkv, 128).to(BF))
    return pages, table, slots


def _check(out, q, pages, slots, q_pos, scale=128 ** -0.5, q_lens=None, kept=None):
    for b, sl in enumerate(slots):
        t = q.shape[1] if q_lens is None else int(q_lens[b])
        if kept is not None and t < q.shape[1]:
            assert torch.equal(out[b, t:], kept[b, t:]), f"sequence {b}: rows past q_lens were written"
        if t == 0:
            continue
        k, v, m = Q.load(pages, sl, mids=True)
        ref, near, size = Q.attention(q[b, :t], k, v, int(q_pos[b]), scale, m)
        off = (out[b, :t].double() - ref).abs()
        tol = 2.0 ** -8 * ref.abs() + 2.0 ** -11 * near + 2.0 ** -10 * size + 1e-30
        assert torch.isfinite(out[b, :t]).all(), f"sequence {b}"
        worst = (off / tol).max().item() if off.numel() else 0.0
        assert worst <= 1, f"sequence {b} of {len(sl)} keys: {worst:.3g} of the tolerance"


def _run(lengths, nh, nkv, P, q_len=1, seed=0, q_lens=None, k_gain=1.0, pos=None, **kw):
    g = _gen(seed)
    pages, table, slots = _filled(g, lengths, nkv, P, k_gain=k_gain)
    q = _randn(g, len(lengths), q_len, nh, 128).to(BF)
    q_pos = torch.tensor(pos if pos is not None else [n - (q_len if q_lens is None else q_lens[b])
                                                      for b, n in enumerate(lengths)], dtype=I64, device="cuda")
    ql = None if q_lens is None else torch.tensor(q_lens, dtype=I32, device="cuda")
    out = _randn(g, *q.shape).to(BF)
    kept = out.clone()
    most = kw.pop("max_kv_len", max(1, max(lengths)))
    got = _ops().gqa_decode_paged_int4(q, pages, table, q_pos, max_kv_len=most, out=out, q_lens=ql, **kw)
    torch.cuda.synchronize()
    assert got is out and _ops().device_status() == 0
    _check(out, q, pages, [s[:most] for s in slots], q_pos, q_lens=q_lens, kept=kept,
           scale=kw.get("scale") or 128 ** -0.5)


# ---------------------------------------------------------------------------------------------
# rows in and out
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("P", [8, 16, 64])
@pytest.mark.parametrize("n,nkv", [(1, 1), (5, 8), (77, 3)])
def test_store_writes_the_oracles_bytes_and_load_returns_them(P, n, nkv):
    ops, g = _ops(), _gen(n + P)
    pages = torch.randint(0, 256, (-(-n // P) + 2, nkv, 160 * P), generator=g, device="cuda", dtype=U8)
    ref = pages.clone()
    k, v = (_randn(g, n, nkv, 128).to(BF) for _ in "kv")
    k[..., 3] *= 50
    k[0] = 7.25
    v[-1] = 0
    slots = torch.randperm(pages.shape[0] * P, generator=g, device="cuda")[:n]
    ops.kv_store_int4(k, v, slots, pages)
    Q.store(ref, slots, k, v)
    torch.cuda.synchronize()
    assert torch.equal(pages, ref)
    gk, gv = ops.kv_load_int4(pages, slots)
    hk, hv = Q.load(ref, slots)
    assert torch.equal(gk, hk.float().to(BF)) and torch.equal(gv, hv.float().to(BF))
    assert ops.device_status() == 0


def test_exact_halves_between_two_codes_round_as_the_oracles():
    ops, g = _ops(), _gen(2)
    # integers and quarters: scales and quotients that are exact, with many ties
    v = (torch.randint(-15, 16, (200, 2, 128), generator=g, device="cuda") / 4).to(BF)
    pages = ops.kv_pages_int4(13, 2, 16)
    ref, slots = pages.clone(), torch.arange(200, device="cuda")
    ops.kv_store_int4(v, -v, slots, pages)
    Q.store(ref, slots, v, -v)
    assert torch.equal(pages, ref)


def test_rows_of_every_magnitude_give_the_oracles_bytes():
    """Steps from the least subnormal to the greatest bf16 number, groups of one value and of two. A mid of
    zero counts without its sign: of +0 and -0 either is the least (IEEE 754), and both hold the same value
    (here the oracle's own bytes differ between devices)."""
    ops, g = _ops(), _gen(24)
    x = torch.rand(272, 1, 128, generator=g, device="cuda", dtype=torch.float64) * 2 - 1
    x = (x * 2.0 ** torch.arange(-143, 129, device="cuda", dtype=torch.float64)[:, None, None])
    x = x.clamp(-3.3895e38, 3.3895e38).to(BF)
    x[:, 0, 32:64] = x[:, 0, 32:33]
    x[:, 0, 64:96] = torch.where(torch.arange(32, device="cuda") % 3 == 0, x[:, 0, 64:65], x[:, 0, 65:66])
    y = x.roll(1, 2)  # a group takes one value of its neighbour's
    pages = ops.kv_pages_int4(34, 1, 8)
    ref, slots = pages.clone(), torch.arange(272, device="cuda")
    ops.kv_store_int4(x, y, slots, pages)
    Q.store(ref, slots, x, y)
    for block in (pages, ref):
        words = block.view(34, 1280).view(torch.int16)
        for at in (256, 576):  # scales and mids of the keys, of the values
            mids = words[:, at + 1:at + 64:2]
            mids.masked_fill_(mids == -0x8000, 0)
    assert torch.equal(pages, ref)


def test_rows_with_strides_padding_and_arena_views():
    ops, g = _ops(), _gen(4)
    n, nkv, P = 19, 4, 16
    big = ops.kv_pages_int4(6, 2 * nkv, P)
    pages = big[:, nkv:]  # heads of a wider arena
    hf = _randn(g, nkv, 40, 128).to(BF)  # head-major rows, as HF has them
    k, v = hf.transpose(0, 1)[:n], hf.transpose(0, 1)[n:2 * n]
    slots = torch.randperm(96, generator=g, device="cuda")[:n]
    slots[::5] = -1
    ops.kv_store_int4(k, v, slots, pages)
    live = slots >= 0
    ref = ops.kv_pages_int4(6, nkv, P)
    Q.store(ref, slots[live], k[live], v[live])
    assert torch.equal(pages, ref) and not big[:, :nkv].any()
    out = [torch.full((nkv, n, 128), 3.0, dtype=BF, device="cuda") for _ in "kv"]
    ops.kv_load_int4(pages, slots, key=out[0].transpose(0, 1), value=out[1].transpose(0, 1))
    hk, hv = Q.load(ref, slots[live])
    assert torch.equal(out[0].transpose(0, 1)[live], hk.float().to(BF))
    assert torch.equal(out[1].transpose(0, 1)[live], hv.float().to(BF))
    assert (out[0][:, ~live] == 3).all() and (out[1][:, ~live] == 3).all()
    assert ops.device_status() == 0


def test_slots_outside_the_arena_are_skipped_and_reported():
    ops, g = _ops(), _gen(5)
    pages = ops.kv_pages_int4(2, 2, 8)
    k = _randn(g, 4, 2, 128).to(BF)
    slots = torch.tensor([3, 16, -2, 1 << 40], device="cuda")
    ops.kv_store_int4(k, k, slots, pages)
    ref = ops.kv_pages_int4(2, 2, 8)
    Q.store(ref, slots[:1], k[:1], k[:1])
    assert torch.equal(pages, ref)
    assert ops.device_status() == 1 << 4
    out = torch.zeros(4, 2, 128, dtype=BF, device="cuda")
    ops.kv_load_int4(pages, slots, key=out, value=torch.zeros_like(out))
    assert not out[1:].any() and ops.device_status() == 1 << 4 and ops.device_status() == 0


def test_broken_rows_read_back_as_nan_in_their_group_only():
    ops, g = _ops(), _gen(6)
    k = _randn(g, 3, 1, 128).to(BF)
    k[0, 0, 5], k[1, 0, 40], k[2, 0, 127] = float("nan"), float("inf"), float("-inf")
    pages = ops.kv_pages_int4(1, 1, 8)
    ops.kv_store_int4(k, k, torch.arange(3, device="cuda"), pages)
    gk, gv = ops.kv_load_int4(pages, torch.arange(3, device="cuda"))
    for x in (gk, gv):
        bad = x.view(3, 4, 32).isnan()
        assert [(i, j) for i in range(3) for j in range(4) if bad[i, j].all()] == [(0, 0), (1, 1), (2, 3)]
        assert bad.sum() == 96


def test_no_rows():
    ops = _ops()
    pages, none = ops.kv_pages_int4(2, 2, 8), torch.zeros(0, dtype=I64, device="cuda")
    k = torch.zeros(0, 2, 128, dtype=BF, device="cuda")
    ops.kv_store_int4(k, k, none, pages)
    gk, _ = ops.kv_load_int4(pages, none)
    assert gk.shape == (0, 2, 128) and not pages.any()


def _append_inputs(g, t, nh, nkv, rows):
    qkv = (_randn(g, t, (nh + 2 * nkv) * 128) * 2).to(BF)
    qn, kn = ((1 + 0.1 * _randn(g, 128)).to(BF) for _ in "qk")
    cos, sin = A.cos_sin(torch.arange(rows, device="cuda"), A.inv_freq(128, 1e6, "cuda"), BF)
    return qkv, qn, kn, cos, sin


@pytest.mark.parametrize("t,nh,nkv,P", [(1, 32, 8, 16), (7, 16, 8, 8), (64, 32, 8, 16), (33, 5, 1, 64),
                                        (515, 14, 2, 16)])
def test_append_matches_the_oracle(t, nh, nkv, P):
    ops, g = _ops(), _gen(t + nh)
    qkv, qn, kn, cos, sin = _append_inputs(g, t, nh, nkv, 4000)
    positions = torch.randint(0, 4000, (t,), generator=g, device="cuda")
    pages = torch.randint(0, 256, (-(-t // P) + 3, nkv, 160 * P), generator=g, device="cuda", dtype=U8)
    ref = pages.clone()
    slots = torch.randperm(pages.shape[0] * P, generator=g, device="cuda")[:t]
    if t > 5:
        slots[2::7] = -1
    q_out = torch.full((t, nh, 128), 9.0, dtype=BF, device="cuda")
    got = ops.qk_norm_rope_append_int4(qkv, qn, kn, EPS, cos, sin, positions, slots, pages, num_qo_heads=nh,
                                       num_kv_heads=nkv, q_out=q_out)
    torch.cuda.synchronize()
    live = slots >= 0
    q, k, v = Q.prologue(qkv, qn, kn, EPS, cos, sin, positions, nh, nkv)
    Q.store(ref, slots[live], k[live], v[live])
    assert torch.equal(pages, ref)
    # queries: half a bf16 step, and fp32's sum of squares and products (below 2^-19 of the pair's size)
    size = (q[live].abs() + torch.roll(q[live], 64, -1).abs())
    off = (got[live].float() - q[live]).abs()
    assert (off <= 2.0 ** -8 * q[live].abs() + 2.0 ** -18 * size).all()
    assert (got[~live] == 9).all() and ops.device_status() == 0


def test_append_without_a_row_in_the_tables_or_the_arena():
    ops, g = _ops(), _gen(8)
    qkv, qn, kn, cos, sin = _append_inputs(g, 5, 4, 2, 50)
    pages = ops.kv_pages_int4(2, 2, 8)
    q_out = torch.full((5, 4, 128), 9.0, dtype=BF, device="cuda")
    positions = torch.tensor([49, 50, -1, 3, 4], device="cuda")
    slots = torch.tensor([0, 1, 2, 16, -1], device="cuda")
    ops.qk_norm_rope_append_int4(qkv, qn, kn, EPS, cos, sin, positions, slots, pages, num_qo_heads=4,
                                 num_kv_heads=2, q_out=q_out)
    assert (q_out[1:] == 9).all() and not (q_out[0] == 9).all() and ops.device_status() == 1 << 4
    assert not pages[1].any()


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
LENGTHS = [1, 7, 8, 9, 15, 16, 17, 100, 255, 256, 257, 1000, 3001]


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("P", [8, 16, 64])
def test_decode_of_one_sequence(n, P):
    _run([n], 32, 8, P, seed=n)


@pytest.mark.parametrize("nh,nkv", [(1, 1), (8, 8), (4, 2), (5, 1), (14, 2), (8, 1), (9, 1), (16, 1), (32, 1), (64, 2)])
@pytest.mark.parametrize("n", [40, 777])
def test_decode_of_every_group(nh, nkv, n):
    _run([n, n // 2], nh, nkv, 16, seed=nh)


@pytest.mark.parametrize("q_len", [2, 4, 5, 8, 17, 40])
@pytest.mark.parametrize("lengths", [[60], [40, 300, 1001]])
def test_verify_rows_see_their_own_prefix(q_len, lengths):
    _run(lengths, 16, 4, 16, q_len=q_len, seed=q_len)


@pytest.mark.parametrize("num_ctas", [0, 1, 2, 13, 296, 1000])
def test_ragged_batches_over_any_number_of_ctas(num_ctas):
    _run(LENGTHS + [0, 2222, 64] + list(range(1, 30)), 8, 2, 16, seed=num_ctas, num_ctas=num_ctas)


@pytest.mark.parametrize("num_ctas", [0, 5])
def test_query_counts_and_rows_without_keys(num_ctas):
    # counts of 0, and sequences whose first rows, or all rows, see no key
    _run([500, 300, 20, 0, 3, 700], 8, 2, 8, q_len=5, q_lens=[5, 0, 3, 4, 5, 1], num_ctas=num_ctas,
         pos=[495, 10, 17, -9, -2, 699])


def test_short_batches_in_the_direct_form():
    _run([0, 1, 5, 16, 100, 256], 8, 2, 16, q_len=3, q_lens=[3, 1, 3, 0, 2, 3], pos=[-3, 0, 2, 1, 98, 253])


def test_keys_past_max_kv_len_are_not_read():
    _run([900, 300], 8, 2, 16, q_len=2, max_kv_len=512)
    _run([900, 30], 8, 2, 16, q_len=2, max_kv_len=100)


@pytest.mark.parametrize("scale", [0.5, -0.1, 1e-9])
def test_other_scales(scale):
    _run([400], 8, 2, 16, scale=scale, k_gain=0.5)


def test_scores_far_apart_and_rising_along_the_sequence():
    ops, g = _ops(), _gen(3)
    n, P = 2000, 16
    pages, table, _ = _filled(g, [n], 1, P)
    slots = Q.slots_of(table[0], n, P)
    k = _randn(g, n, 1, 128).to(BF)
    k += (torch.arange(n, device="cuda")[:, None, None] / 400).to(BF)  # the maximum is raised again and again
    Q.store(pages, slots, k, _randn(g, n, 1, 128).to(BF))
    q = (1 + 0.1 * _randn(g, 1, 1, 8, 128)).to(BF)
    pos = torch.tensor([n - 1], device="cuda")
    for ctas in (1, 30):
        out = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n, num_ctas=ctas)
        _check(out, q, pages, [slots], pos)


def test_strided_queries_outputs_tables_and_pages():
    ops, g = _ops(), _gen(9)
    nh, nkv, P, n = 8, 2, 16, 333
    pages, table, slots = _filled(g, [n, n - 50], nkv, P)
    wide = torch.zeros(pages.shape[0], 2 * nkv, pages.shape[2], dtype=U8, device="cuda")
    wide[:, 1::2] = pages  # every other head of a wider arena
    tables = torch.full((2, 2 * table.shape[1]), -1, dtype=I32, device="cuda")
    tables[:, :table.shape[1]] = table
    q = _randn(g, 2, nh, 3, 136).to(BF)[..., :128].transpose(1, 2)  # [2, 3, nh, 128]
    out = torch.zeros(3, 2, nh, 132, dtype=BF, device="cuda").transpose(0, 1)[..., :128]
    pos = torch.tensor([n - 3, n - 53], device="cuda")
    ops.gqa_decode_paged_int4(q, wide[:, 1::2], tables, pos, max_kv_len=n, out=out)
    _check(out, q, pages, slots, pos)


def test_pages_past_32_bits():
    ops, g = _ops(), _gen(10)
    nkv, P, n = 8, 64, 900
    num = (5 << 30) // (nkv * P * 160)  # 5 GiB of pages
    pages = torch.empty(num, nkv, 160 * P, dtype=U8, device="cuda")
    table = (num - 1 - torch.arange(15, device="cuda", dtype=I32))[None]
    slots = Q.slots_of(table[0], n, P)
    k, v = (_randn(g, n, nkv, 128).to(BF) for _ in "kv")
    ops.kv_store_int4(k, v, slots, pages)
    gk, gv = ops.kv_load_int4(pages, slots)
    assert torch.equal(gk, Q.held(k).float().to(BF)) and torch.equal(gv, Q.held(v).float().to(BF))
    q, pos = _randn(g, 1, 1, 32, 128).to(BF), torch.tensor([n - 1], device="cuda")
    out = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n)
    _check(out, q, pages[-15:].contiguous(), [slots - (num - 15) * P], pos)


def test_table_entries_outside_the_arena_count_as_absent_keys():
    ops, g = _ops(), _gen(11)
    for P, n in ((8, 203), (16, 500)):
        pages, table, _ = _filled(g, [n], 2, P)
        q, pos = _randn(g, 1, 1, 8, 128).to(BF), torch.tensor([n - 1], device="cuda")
        good = Q.slots_of(table[0], n, P)
        table[0, 3], table[0, 7] = pages.shape[0], -5
        at = torch.arange(n, device="cuda") // P
        good = good[(at != 3) & (at != 7)]
        for ctas in (0, 6):
            out = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n, num_ctas=ctas)
            torch.cuda.synchronize()
            assert ops.device_status() == 1 << 5
            _check(out, q, pages, [good], pos)


def test_broken_keys_reach_the_rows_that_see_them_and_no_others():
    ops, g = _ops(), _gen(12)
    n, P = 300, 16
    pages, table, slots = _filled(g, [n], 1, P)
    k = torch.full((1, 1, 128), float("nan"), dtype=BF, device="cuda")
    ops.kv_store_int4(k, k, slots[0][298:299], pages)
    q, pos = _randn(g, 1, 4, 2, 128).to(BF), torch.tensor([296], device="cuda")
    for most in (300, 256):
        out = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=most)
        if most == 300:
            assert out[0, 2:].isnan().all()
            _check(out[:, :2], q[:, :2], pages, [slots[0][:298]], pos)
        else:
            assert torch.isfinite(out).all()


@pytest.mark.parametrize("nh", [1, 2, 4])
def test_broken_values_behind_a_row_leave_it_as_it_is(nh):
    """Only V is broken, and 1, 2 or 4 heads of the group put rows with and without it into one warp."""
    ops, g = _ops(), _gen(21)
    n, P = 90, 16
    for P in (8, 16):
        pages, table, slots = _filled(g, [n], 1, P)
        v = torch.full((1, 1, 128), float("nan"), dtype=BF, device="cuda")
        ops.kv_store_int4(_randn(g, 1, 1, 128).to(BF), v, slots[0][88:89], pages)
        q, pos = _randn(g, 1, 3, nh, 128).to(BF), torch.tensor([87], device="cuda")
        for ctas in (0, 1):
            out = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n, num_ctas=ctas)
            assert out[0, 1:].isnan().all()
            _check(out[:, :1], q[:, :1], pages, [slots[0][:88]], pos)


def test_value_scales_far_apart():
    """Groups of values 2^40 apart, tokens too: each is held to its own size."""
    ops, g = _ops(), _gen(22)
    n, P = 700, 16
    pages, table, slots = _filled(g, [n], 2, P)
    v = _randn(g, n, 2, 4, 32) * torch.tensor([1e-18, 1.0, 1e12, 30.0], device="cuda")[:, None]
    v[300:] *= 1e3  # the powers of two are lowered half way
    ops.kv_store_int4(_randn(g, n, 2, 128).to(BF), v.view(n, 2, 128).to(BF), slots[0], pages)
    q, pos = _randn(g, 1, 1, 8, 128).to(BF), torch.tensor([n - 1], device="cuda")
    for ctas in (0, 1):
        _check(ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=n, num_ctas=ctas), q, pages, slots, pos)


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e4, 1e25])
def test_query_rows_of_any_size(size):
    ops, g = _ops(), _gen(23)
    pages, table, slots = _filled(g, [500], 2, 16)
    q = (_randn(g, 1, 1, 8, 128) * size).to(BF)
    q[0, 0, 3] = 0
    pos, scale = torch.tensor([499], device="cuda"), 0.1 / size
    _check(ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=500, scale=scale), q, pages, slots, pos, scale=scale)


def test_a_call_gives_the_same_bits_every_time():
    ops, g = _ops(), _gen(13)
    pages, table, _ = _filled(g, [3000, 17, 800], 8, 16)
    q, pos = _randn(g, 3, 1, 32, 128).to(BF), torch.tensor([2999, 16, 799], device="cuda")
    first = ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=3000)
    for _ in range(5):
        assert torch.equal(ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=3000), first)


@pytest.mark.parametrize("batch,nkv,n", [(16, 8, 1152), (16, 8, 1153), (37, 8, 192), (38, 8, 192),
                                         (150, 8, 33), (3, 1, 513)])
def test_both_sides_of_the_division_between_ctas(batch, nkv, n):
    _run([n - 7 * (b % 4) for b in range(batch)], 2 * nkv, nkv, 16, max_kv_len=n)


@pytest.mark.parametrize("lengths,most,q_len,q_lens", [
    ([700], 700, 1, None), ([0, 700], 700, 1, None), ([1, 1536], 1536, 1, None), ([1536, 33], 1536, 2, [2, 1]),
    ([700, 5, 0, 64], 700, 5, [5, 3, 0, 1]), ([1] * 9 + [1000] * 7, 1000, 1, None), ([190, 3000], 3000, 3, [3, 0])])
def test_units_of_several_ctas(lengths, most, q_len, q_lens):
    """Caches that a cluster shares: sequences shorter than its warps, rows and sequences that see nothing."""
    _run(lengths, 16, 8, 16, q_len=q_len, q_lens=q_lens, max_kv_len=most)


def test_a_workspace_of_the_largest_call_serves_the_smaller_ones():
    ops, g = _ops(), _gen(25)
    sizes = [[ops.decode_int4_workspace_bytes(b, t, 32, 8, n) for n in (1, 64, 512, 513, 1100, 4000, 70000)]
             for t in (1, 2, 3, 9) for b in (1, 2, 4, 16, 38, 64, 300)]
    by = torch.tensor(sizes).view(4, 7, 7)
    for dim in range(3):
        assert (by.diff(dim=dim) >= 0).all()
    pages, table, slots = _filled(g, [1100] * 4, 8, 16)
    ws = torch.full((ops.decode_int4_workspace_bytes(4, 5, 32, 8, 1100),), 255, dtype=U8, device="cuda")
    for b, t, n in ((4, 5, 1100), (1, 1, 700), (2, 2, 1), (4, 1, 1100), (3, 5, 300), (1, 5, 1000)):
        q = _randn(g, b, t, 32, 128).to(BF)
        pos = torch.full((b,), n - 1, device="cuda")
        out = ops.gqa_decode_paged_int4(q, pages, table[:b], pos, max_kv_len=n, workspace=ws)
        _check(out, q, pages, [x[:n] for x in slots[:b]], pos)


def test_calls_on_two_streams_at_once():
    ops, g = _ops(), _gen(26)
    pages, table, _ = _filled(g, [5000, 900, 2111], 8, 16)
    q = [_randn(g, 3, t, 32, 128).to(BF) for t in (1, 4)]
    pos = torch.tensor([4990, 890, 2101], device="cuda")
    want = [ops.gqa_decode_paged_int4(x, pages, table, pos, max_kv_len=5000) for x in q]
    ws = [torch.empty(ops.decode_int4_workspace_bytes(3, x.shape[1], 32, 8, 5000), dtype=U8, device="cuda")
          for x in q]
    out = [torch.zeros_like(x) for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, w, o, st in zip(q, ws, out, streams):
            with torch.cuda.stream(st):
                ops.gqa_decode_paged_int4(x, pages, table, pos, max_kv_len=5000, out=o, workspace=w)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_two_graphs_that_share_a_workspace_and_sequences_that_share_pages():
    """Two captured calls of different sizes, replayed in turn over one workspace; the second's sequences
    are one prefix at several lengths, the same pages in every table row."""
    ops, g = _ops(), _gen(27)
    pages, table, slots = _filled(g, [3000], 8, 16)
    shared = table.expand(5, -1).contiguous()
    ends = [2999, 2999, 40, 1500, 0]
    q = [_randn(g, b, 1, 32, 128).to(BF) for b in (1, 5)]
    pos = [torch.tensor([2000], device="cuda"), torch.tensor(ends, device="cuda")]
    ws = torch.empty(ops.decode_int4_workspace_bytes(5, 1, 32, 8, 3000), dtype=U8, device="cuda")
    out = [torch.zeros_like(x) for x in q]

    def call(i):
        ops.gqa_decode_paged_int4(q[i], pages, (table, shared)[i], pos[i], max_kv_len=3000, out=out[i], workspace=ws)

    graphs = []
    for i in range(2):
        call(i)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            call(i)
    for _ in range(3):
        for x in out:
            x.fill_(9)
        pos[0] += 1
        for gr in graphs + graphs[::-1]:
            gr.replay()
        torch.cuda.synchronize()
        _check(out[0], q[0], pages, slots, pos[0])
        _check(out[1], q[1], pages, slots * 5, pos[1])


def test_refusals_on_the_device():
    ops, g = _ops(), _gen(14)
    pages, table, _ = _filled(g, [600], 8, 16)
    q, pos = _randn(g, 1, 1, 32, 128).to(BF), torch.tensor([599], device="cuda")
    need = ops.decode_int4_workspace_bytes(1, 1, 32, 8, 600)
    assert need > 0 and ops.decode_int4_workspace_bytes(9, 1, 32, 8, 256) == 0
    with pytest.raises(RuntimeError, match="workspace"):
        ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=600,
                                  workspace=torch.empty(need - 1, dtype=U8, device="cuda"))
    with pytest.raises(RuntimeError, match="workspace"):
        ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=600,
                                  workspace=torch.empty(need + 300, dtype=U8, device="cuda")[8:])
    with pytest.raises(RuntimeError, match="max_kv_len"):
        ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=table.shape[1] * 16 + 1)
    with pytest.raises(RuntimeError, match="KV heads"):
        ops.qk_norm_rope_append_int4(torch.zeros(1, 48 * 128, dtype=BF, device="cuda"), pos, pos, EPS, pos, pos,
                                     pos, pos, pages, num_qo_heads=32, num_kv_heads=4)
    with pytest.raises(RuntimeError, match="cpu"):
        ops.gqa_decode_paged_int4(q, pages, table.cpu(), pos, max_kv_len=600)
    with pytest.raises(RuntimeError, match="solort_attn_decode_int4"):  # a count beyond its field
        ops.gqa_decode_paged_int4(q, pages, table, pos, max_kv_len=600, num_ctas=1 << 40,
                                  workspace=torch.empty(need, dtype=U8, device="cuda"))


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def test_prompt_chunks_and_captured_decode_steps_of_a_batch():
    """Two sequences: a prompt appended whole, the rest of a longer one as a chunk over its cached prefix
    (load + prefill), then decode steps of both, padded to four, replayed from one captured graph on a
    side stream; every result against the oracle's own cache."""
    ops, g = _ops(), _gen(20)
    nh, nkv, P, top = 16, 2, 16, 512
    pages, ref = ops.kv_pages_int4(70, nkv, P), ops.kv_pages_int4(70, nkv, P)
    table = torch.randperm(70, generator=g, device="cuda")[:64].to(I32).view(2, 32)
    table = torch.cat([table, torch.zeros(2, 32, dtype=I32, device="cuda")])
    _, qn, kn, cos, sin = _append_inputs(g, 1, nh, nkv, top)

    def append(qkv, positions, slots, out=None):
        q = ops.qk_norm_rope_append_int4(qkv, qn, kn, EPS, cos, sin, positions, slots, pages, num_qo_heads=nh,
                                         num_kv_heads=nkv, q_out=out)
        live = slots >= 0
        if not torch.cuda.is_current_stream_capturing():
            _, k, v = Q.prologue(qkv[live], qn, kn, EPS, cos, sin, positions[live], nh, nkv)
            Q.store(ref, slots[live], k, v)
        return q

    lengths = [150, 333]
    for b, first in ((0, 0), (1, 0), (1, 200)):  # sequence 1 arrives as 200 tokens and then the rest
        at = torch.arange(first, 200 if (b, first) == (1, 0) else lengths[b], device="cuda")
        slots = table[b].long()[at // P] * P + at % P
        qkv = (_randn(g, len(at), (nh + 2 * nkv) * 128)).to(BF)
        q = append(qkv, at, slots)
        k, v = ops.kv_load_int4(pages, Q.slots_of(table[b], int(at[-1]) + 1, P))
        out = ops.gqa_prefill(q, k, v)
        want = Q.attention(q, k.double(), v.double(), first, 128 ** -0.5)
        assert (out.double() - want).abs().max() <= 2e-2  # the prefill's own tolerance
    assert torch.equal(pages, ref)

    qkv = torch.zeros(4, (nh + 2 * nkv) * 128, dtype=BF, device="cuda")
    pos = torch.tensor([lengths[0], lengths[1], 0, 0], device="cuda")
    slots = torch.full((4,), -1, dtype=I64, device="cuda")
    q_lens = torch.tensor([1, 1, 0, 0], dtype=I32, device="cuda")
    q_out = torch.zeros(4, nh, 128, dtype=BF, device="cuda")
    out = torch.full((4, 1, nh, 128), 5.0, dtype=BF, device="cuda")
    ws = torch.empty(ops.decode_int4_workspace_bytes(4, 1, nh, nkv, top), dtype=U8, device="cuda")

    def step():
        append(qkv, pos, slots, q_out)
        ops.gqa_decode_paged_int4(q_out[:, None], pages, table, pos, max_kv_len=top, out=out, workspace=ws,
                                  q_lens=q_lens, stable_prefix=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(20):
        at = torch.tensor(lengths, device="cuda") + i
        pos[:2].copy_(at)
        slots[:2].copy_(table[:2].long().gather(1, (at // P)[:, None])[:, 0] * P + at % P)
        qkv.copy_(_randn(g, *qkv.shape).to(BF))
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        _, k, v = Q.prologue(qkv[:2], qn, kn, EPS, cos, sin, pos[:2], nh, nkv)
        Q.store(ref, slots[:2], k, v)
        assert torch.equal(pages, ref)
        _check(out[:2], q_out[:2, None], pages, [Q.slots_of(table[b], int(at[b]) + 1, P) for b in (0, 1)], at)
        assert (out[2:] == 5).all()
    assert ops.device_status() == 0
