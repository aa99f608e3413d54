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


def _along(n, score):
    """Keys that score ``score`` (a number each) with queries of ones, scaled by 128^-0.5: constant rows,
    which are held exactly where they are bf16 numbers."""
    return (torch.as_tensor(score, device="cuda", dtype=torch.float32).expand(n) / 128 ** 0.5)[:, None, None].expand(n, 1, 128)


def _ones(g, t, heads):
    return (1 + 0.05 * _randn(g, 1, t, heads, 128)).to(BF)


@pytest.mark.parametrize("heads", [2, 4, 8])
@pytest.mark.parametrize("power", [20, 24, 28, 34, 60, 100])
@pytest.mark.parametrize("at", [0, 333, 699])
def test_a_token_of_large_values_and_no_weight(power, heads, at):
    """Its scale is 2^power times the others', its weight e^-(0.7 power + 4) and less."""
    g, n = _gen(power + heads + at), 700
    k, v = _randn(g, n, 1, 128), _randn(g, n, 1, 128)
    k[at] = _along(1, -0.7 * power - 12.0)[0]
    v[at] *= 2.0 ** power
    _check(_ones(g, 1, heads), *_held(g, k, v))


@pytest.mark.parametrize("heads", [4, 8])
@pytest.mark.parametrize("power", [30, 80])
def test_a_large_token_that_half_of_the_heads_look_at(power, heads):
    """The others' results stay their own, in a group of its own size too."""
    g, n = _gen(power + heads), 500
    k, v = _randn(g, n, 1, 128), _randn(g, n, 1, 128)
    k[200] = _along(1, 60.0)[0]
    v[200, :, :96] *= 2.0 ** power
    q = _ones(g, 1, heads)
    q[:, :, ::2] *= -1
    _check(q, *_held(g, k, v))


@pytest.mark.parametrize("score", [-45.0, 0.0, 30.0])
@pytest.mark.parametrize("q_len,heads", [(2, 1), (2, 4), (5, 2), (4, 8)])
def test_a_large_token_that_only_the_last_row_sees(q_len, heads, score):
    g, n = _gen(q_len + heads), 160
    k, v = _randn(g, n, 1, 128), _randn(g, n, 1, 128)
    k[n - 1] = _along(1, score)[0]
    v[n - 1] *= 2.0 ** 40
    _check(_ones(g, q_len, heads), *_held(g, k, v))


@pytest.mark.parametrize("heads", [2, 4, 8])
@pytest.mark.parametrize("size", [0.0, 1e-20, 1e-3])
@pytest.mark.parametrize("at", [0, 400, 699])
def test_nearly_all_weight_on_a_token_of_small_values(size, heads, at):
    """Heads that look away: the result is what the other tokens give, e^-20 of the weight each."""
    g, n = _gen(heads + at), 700
    k, v = _randn(g, n, 1, 128), _randn(g, n, 1, 128)
    k[at] = _along(1, 20.0)[0]
    v[at] *= size
    _check(_ones(g, 1, heads), *_held(g, k, v))


@pytest.mark.parametrize("heads", [2, 4, 8])
@pytest.mark.parametrize("falling", [False, True])
def test_values_that_shrink_while_scores_grow(heads, falling):
    """From 2^60 with no weight in the end to 1 with all of it, or the other way round; the power of two of
    a row has to follow both ways."""
    g, n = _gen(heads), 960
    steps = torch.linspace(0, 1, n, device="cuda")
    steps = (1 - steps) if falling else steps
    k = _along(n, 90 * steps) + 0.02 * _randn(g, n, 1, 128)
    v = _randn(g, n, 1, 128) * 2.0 ** (60 * (1 - steps))[:, None, None]
    _check(_ones(g, 1, heads), *_held(g, k, v))


def test_broken_values_without_weight_stay_visible():
    """A NaN in V reaches every row that sees it, whatever its weight."""
    ops, g, n = _ops(), _gen(1), 200
    k, v = _randn(g, n, 1, 128), _randn(g, n, 1, 128)
    k[50], v[50] = _along(1, -200.0)[0], float("nan")
    pages, table, _ = _held(g, k, v)
    for heads in (4, 8):
        out = ops.gqa_decode_paged_int4(_ones(g, 1, heads), pages, table, torch.tensor([n - 1], device="cuda"), max_kv_len=n)
        assert out.isnan().all()
