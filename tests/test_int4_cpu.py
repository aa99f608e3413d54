"""The paged 4-bit KV cache without a GPU: the formula's error bound, the layout's addresses, the
argument structs against the header, the registered ops, and what the entry points refuse."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import int4 as Q
from solort_b200 import _calls_int4, _lib, ops, torch_ops_int4
from tests.test_capi import _c_layout

BF, I32, I64, U8 = torch.bfloat16, torch.int32, torch.int64, torch.uint8


def _rows(kind: str) -> torch.Tensor:
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, 128, generator=g)
    if kind == "offset":  # far from zero: the mid's bf16 step is larger than the spread
        x = x * 0.01 + 1000
    elif kind == "outlier":
        x[:, 7] *= 300
    elif kind == "constant":
        x = x[:, :1].expand(64, 128).clone()
    elif kind == "zero":
        x = x * 0
    elif kind == "tiny":
        x = x * 1e-39
    elif kind == "huge":
        x = x.clamp(-3, 3) * 1e38
    elif kind == "bf16":
        x = x.to(BF).float()
    return x


@pytest.mark.parametrize("kind", ["normal", "offset", "outlier", "constant", "zero", "tiny", "huge", "bf16"])
def test_every_held_value_is_within_half_a_step(kind):
    x = _rows(kind)
    codes, scale, mid = Q.quantise(x)
    assert codes.min() >= 0 and codes.max() <= 15 and scale.isfinite().all() and mid.isfinite().all()
    # half a step, and the fp32 roundings of x - mid, of the quotient and of its sum with 7.5: each at
    # most 2^-24 of a number below 16 steps; where the scale is subnormal, its own last bit as well
    step = scale.double().repeat_interleave(32, -1)
    off = (x.double() - Q.held(x)).abs()
    assert (off <= step * (0.5 + 3 * 16 * 2.0 ** -24) + 2.0 ** -149).all()
    if kind in ("zero",):
        assert (off == 0).all()


def test_addresses_of_a_block_cover_it_once():
    rows = torch.arange(8)
    used = torch.zeros(Q.BLOCK * 2, dtype=torch.long)  # nibbles
    for is_value in (False, True):
        byte, shift = Q.code_place(rows, is_value)
        nib = (2 * byte + shift // 4).reshape(-1)
        used.index_add_(0, nib, torch.ones_like(nib))
        meta = Q.meta_place(rows, is_value).reshape(-1)
        for o in range(4):
            for h in range(2):
                used.index_add_(0, 2 * (meta + o) + h, torch.ones_like(meta))
    assert (used == 1).all()


def test_oracle_store_and_load_are_inverse():
    g = torch.Generator().manual_seed(1)
    pages = torch.zeros(5, 3, 160 * 16, dtype=U8)
    slots = torch.randperm(80, generator=g)[:37]
    k, v = (torch.randn(37, 3, 128, generator=g).to(BF) for _ in "kv")
    Q.store(pages, slots, k, v)
    gk, gv = Q.load(pages, slots)
    assert torch.equal(gk, Q.held(k)) and torch.equal(gv, Q.held(v))


@pytest.mark.parametrize("name", ["SolortInt4AppendArgs", "SolortInt4StoreArgs", "SolortInt4LoadArgs",
                                  "SolortInt4DecodeArgs"])
def test_ctypes_struct_matches_header(name):
    cls = getattr(_lib, name)
    c = _c_layout(name, [f[0] for f in cls._fields_])
    assert c["sizeof"] == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert c[f] == getattr(cls, f).offset, f


@pytest.mark.parametrize("name", ["SolortInt4AppendArgs", "SolortInt4StoreArgs", "SolortInt4LoadArgs",
                                  "SolortInt4DecodeArgs"])
def test_packed_fields_are_the_struct(name):
    cls = getattr(_lib, name)
    fields = [0.25 * i if t is ctypes.c_float else (1 << 30) + i for i, (_, t) in enumerate(cls._fields_)]
    assert _calls_int4.packer(cls)(*fields) == bytes(cls(*fields))


def test_ops_are_registered_with_their_outputs_mutated():
    mutated = {"qk_norm_rope_append_int4": {"kv_pages", "q_out"}, "kv_store_int4": {"kv_pages"},
               "kv_load_int4": {"key", "value"}, "gqa_decode_paged_int4": {"out", "workspace"}}
    assert set(torch_ops_int4.OPS) == set(mutated)
    for name, expect in mutated.items():
        schema = getattr(torch.ops.solort_attn, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info and a.alias_info.is_write} == expect
        assert len(schema.returns) == 0


def _decode_struct(**change) -> _lib.SolortInt4DecodeArgs:
    at = 1 << 20  # never read: every call below is refused, or ends for want of a device
    a = _lib.SolortInt4DecodeArgs(at, 4096, 4096, 128, at, 4096, 4096, 128, at, 20480, 2560, 16, 64, at, 64,
                                  at, None, 1, 1, 32, 8, 128, 1024, 0.1, 0, None, 0, 0)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    ({"head_dim": 64}, -2), ({"q": None}, -1), ({"out": None}, -1), ({"kv_pages": None}, -1),
    ({"block_table": None}, -1), ({"q_pos": None}, -1), ({"q": (1 << 20) + 8}, -1),
    ({"q_stride_head": 132}, -1), ({"out_stride_head": 130}, -1), ({"kv_pages": (1 << 20) + 8}, -1),
    ({"kv_stride_head": 2568}, -1), ({"kv_stride_page": -2560}, -1), ({"page_size": 4}, -1),
    ({"page_size": 24}, -1), ({"num_pages": 0}, -1), ({"batch": 0}, -1), ({"q_len": 0}, -1),
    ({"num_qo_heads": 33}, -1), ({"num_kv_heads": 0}, -1), ({"max_kv_len": 0}, -1), ({"num_ctas": -1}, -1),
    ({"batch": 65536}, -2), ({"batch": 60000, "max_kv_len": 1 << 30}, -2),
    ({"q_lens": (1 << 20) + 2}, -1), ({"q_pos": (1 << 20) + 4}, -1)])
def test_decode_refuses_before_it_reaches_a_device(change, code):
    a = _decode_struct(**change)
    assert _lib.load().solort_attn_decode_int4(ctypes.byref(a), None) == code


@pytest.mark.parametrize("change,code", [
    ({"head_dim": 96}, -2), ({"kv_pages": None}, -1), ({"slots": None}, -1), ({"key": None}, -1),
    ({"value": (1 << 20) + 2}, -1), ({"key_stride_token": 4}, -1), ({"value_stride_head": 100}, -1),
    ({"page_size": 0}, -1), ({"num_pages": -3}, -1), ({"num_tokens": -1}, -1), ({"num_kv_heads": 0}, -1),
    ({"kv_stride_head": 8}, -1), ({"num_tokens": 0}, 0)])
@pytest.mark.parametrize("which", ["store", "load"])
def test_store_and_load_refuse(which, change, code):
    at = 1 << 20
    cls = _lib.SolortInt4StoreArgs if which == "store" else _lib.SolortInt4LoadArgs
    a = cls(at, at, 1024, 128, 1024, 128, 5, 8, 128, at, at, 20480, 2560, 16, 64)
    for k, v in change.items():
        setattr(a, k, v)
    assert getattr(_lib.load(), f"solort_attn_kv_{which}_int4")(ctypes.byref(a), None) == code


@pytest.mark.parametrize("change,code", [
    ({"head_dim": 64}, -2), ({"qkv": None}, -1), ({"cos": None}, -1), ({"positions": None}, -1),
    ({"q_out": None}, -1), ({"rope_rows": 0}, -1), ({"num_qo_heads": 0}, -1), ({"qkv_stride_token": 12}, -1),
    ({"sin": (1 << 20) + 8}, -1), ({"rope_stride": 132}, -1), ({"page_size": 12}, -1), ({"num_tokens": 0}, 0)])
def test_append_refuses(change, code):
    at = 1 << 20
    a = _lib.SolortInt4AppendArgs(at, 6144, 2, 32, 8, 128, at, at, 1e-6, at, at, 128, 64, at, at, at, 4096, 128,
                                  at, 20480, 2560, 16, 64)
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.load().solort_attn_qk_norm_rope_append_int4(ctypes.byref(a), None) == code


def _t(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _decode(**change):
    a = dict(q=_t(2, 1, 32, 128), kv_pages=_t(64, 8, 2560, dtype=U8), block_table=_t(2, 64, dtype=I32),
             q_pos=_t(2, dtype=I64), out=_t(2, 1, 32, 128), workspace=_t(1 << 20, dtype=U8), max_kv_len=1024)
    a.update(change)
    torch.ops.solort_attn.gqa_decode_paged_int4(**a)


def _append(**change):
    a = dict(qkv=_t(3, 48 * 128), q_norm_weight=_t(128), k_norm_weight=_t(128), eps=1e-6, cos=_t(64, 128),
             sin=_t(64, 128), positions=_t(3, dtype=I64), slots=_t(3, dtype=I64),
             kv_pages=_t(64, 8, 2560, dtype=U8), q_out=_t(3, 32, 128))
    a.update(change)
    torch.ops.solort_attn.qk_norm_rope_append_int4(**a)


def _store(**change):
    a = dict(key=_t(3, 8, 128), value=_t(3, 8, 128), slots=_t(3, dtype=I64), kv_pages=_t(64, 8, 2560, dtype=U8))
    a.update(change)
    torch.ops.solort_attn.kv_store_int4(**a)


def test_fake_impls_trace_well_formed_calls():
    with FakeTensorMode():
        _decode()
        _decode(q=_t(2, 40, 32, 128), out=_t(2, 40, 32, 128), max_kv_len=1)
        _append()
        _store()
        torch.ops.solort_attn.kv_load_int4(_t(64, 8, 2560, dtype=U8), _t(3, dtype=I64), _t(3, 8, 128), _t(3, 8, 128))


@pytest.mark.parametrize("call,change", [
    (_decode, {"kv_pages": lambda: _t(64, 8, 2550, dtype=U8)}),
    (_decode, {"kv_pages": lambda: _t(64, 8, 160 * 24, dtype=U8)}),
    (_decode, {"kv_pages": lambda: _t(64, 8, 160 * 4, dtype=U8)}),
    (_decode, {"kv_pages": lambda: _t(64, 8, 2560)}),
    (_decode, {"block_table": lambda: _t(2, 64, dtype=I64)}),
    (_decode, {"block_table": lambda: _t(1, 64, dtype=I32)}),
    (_decode, {"q_pos": lambda: _t(2, dtype=I32)}), (_decode, {"q_pos": lambda: _t(3, dtype=I64)}),
    (_decode, {"max_kv_len": lambda: 1025}), (_decode, {"max_kv_len": lambda: 0}),
    (_decode, {"out": lambda: _t(2, 1, 32, 128, dtype=torch.float16)}),
    (_decode, {"q": lambda: _t(2, 1, 32, 64)}), (_decode, {"q": lambda: _t(2, 1, 33, 128)}),
    (_append, {"qkv": lambda: _t(3, 47 * 128)}), (_append, {"slots": lambda: _t(2, dtype=I64)}),
    (_append, {"positions": lambda: _t(3, dtype=I32)}), (_append, {"q_out": lambda: _t(4, 32, 128)}),
    (_append, {"sin": lambda: _t(63, 128)}),
    (_store, {"key": lambda: _t(3, 4, 128)}), (_store, {"value": lambda: _t(2, 8, 128)}),
    (_store, {"slots": lambda: _t(3, 1, dtype=I64)})])
def test_fake_impls_reject_malformed_calls(call, change):
    with FakeTensorMode(), pytest.raises(RuntimeError):
        call(**{k: v() for k, v in change.items()})


def test_cpu_tensors_are_refused():
    pages = ops.kv_pages_int4(4, 8, 16, device="cpu")
    assert pages.shape == (4, 8, 2560) and not pages.any()
    with pytest.raises(RuntimeError, match="power of two"):
        ops.kv_pages_int4(4, 8, 12, device="cpu")
    k, slots = torch.zeros(2, 8, 128, dtype=BF), torch.zeros(2, dtype=I64)
    with pytest.raises(NotImplementedError):
        ops.kv_store_int4(k, k, slots, pages)
    with pytest.raises(NotImplementedError):
        ops.kv_load_int4(pages, slots)
    q = torch.zeros(1, 1, 32, 128, dtype=BF)
    with pytest.raises(RuntimeError):
        ops.gqa_decode_paged_int4(q, pages, torch.zeros(1, 4, dtype=I32), torch.zeros(1, dtype=I64), max_kv_len=64)
