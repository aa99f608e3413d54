"""Tensors with too few dimensions are refused by the 4-bit calls as any other wrong shape: RuntimeError."""

from __future__ import annotations

import pytest
import torch

from solort_b200 import _calls_int4 as C
from solort_b200 import ops

BF, I32, I64 = torch.bfloat16, torch.int32, torch.int64


def _z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _pages(dims: int) -> torch.Tensor:
    pages = ops.kv_pages_int4(1, 1, 16, device="cpu")
    return pages[0, 0, 0] if dims == 0 else pages.view((1,) * (dims - 1) + (2560,))


def _append(body, pages, qkv=None, cos=None):
    qkv = _z(3, 48 * 128) if qkv is None else qkv
    cos, at = _z(4, 128) if cos is None else cos, _z(3, dtype=I64)
    if body:
        C.append_into(qkv, _z(128), _z(128), 1e-6, cos, _z(4, 128), at, at, pages, _z(3, 32, 128))
    else:
        ops.qk_norm_rope_append_int4(qkv, _z(128), _z(128), 1e-6, cos, _z(4, 128), at, at, pages, num_qo_heads=32,
                                     num_kv_heads=8)


def _decode(body, pages, q=None, table=None):
    q = _z(1, 1, 32, 128) if q is None else q
    table = _z(1, 4, dtype=I32) if table is None else table
    if body:
        C.decode_into(q, pages, table, _z(1, dtype=I64), torch.zeros_like(q), _z(0, dtype=torch.uint8), 32)
    else:
        ops.gqa_decode_paged_int4(q, pages, table, _z(1, dtype=I64), max_kv_len=32)


@pytest.mark.parametrize("dims", [0, 1, 2])
@pytest.mark.parametrize("call", [
    lambda p: _append(True, p), lambda p: _append(False, p), lambda p: _decode(True, p), lambda p: _decode(False, p),
    lambda p: ops.kv_load_int4(p, _z(3, dtype=I64)),
    lambda p: C.load_into(p, _z(3, dtype=I64), _z(3, 8, 128), _z(3, 8, 128)),
    lambda p: C.store_into(_z(3, 8, 128), _z(3, 8, 128), _z(3, dtype=I64), p)])
def test_arenas(call, dims):
    pages = _pages(dims)
    assert pages.dim() == dims
    with pytest.raises(RuntimeError, match="arena"):
        call(pages)


@pytest.mark.parametrize("call", [
    lambda p: _append(True, p, qkv=_z()), lambda p: _append(False, p, qkv=_z()), lambda p: _append(False, p, qkv=_z(3)),
    lambda p: _append(True, p, cos=_z()), lambda p: _append(True, p, cos=_z(4)),
    lambda p: _decode(True, p, q=_z()), lambda p: _decode(False, p, q=_z(3, 128)),
    lambda p: _decode(True, p, table=_z(dtype=I32)), lambda p: _decode(False, p, table=_z(4, dtype=I32)),
    lambda p: C.store_into(_z(), _z(3, 8, 128), _z(3, dtype=I64), p),
    lambda p: C.load_into(p, _z(dtype=I64), _z(1, 8, 128), _z(1, 8, 128)),
    lambda p: ops.kv_load_int4(p, _z(dtype=I64))])
def test_other_tensors(call):
    # NotImplementedError, a RuntimeError too, is the dispatcher's for CPU tensors
    with pytest.raises(RuntimeError):
        call(ops.kv_pages_int4(4, 8, 16, device="cpu"))
