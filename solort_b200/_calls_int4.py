"""C-ABI call builders of the paged 4-bit KV cache: the bodies of the ``torch.ops.solort_attn.*_int4``
ops. As ``solort_b200._calls``: each function checks its tensors, packs one argument struct of
``include/solort_attn.h`` and makes one library call on the current stream of the tensors' device; it
writes only the tensors it is given and allocates nothing. Errors raise ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from solort_b200 import _lib
from solort_b200._calls import HEAD_DIM, _stream_at

TOKEN_BYTES = 160  # K and V of one token of one KV head: codes, and a scale and a mid per 32 values
_byref = ctypes.byref
_BF16, _I64, _I32, _U8 = torch.bfloat16, torch.int64, torch.int32, torch.uint8


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def page_size(kv_pages: torch.Tensor) -> int:
    """Tokens of a page of a 4-bit arena ``[num_pages, nkv, 160 * P]`` (uint8), with its checks."""
    _need(kv_pages.dtype is _U8 and kv_pages.dim() == 3 and kv_pages.stride(2) == 1,
          "kv_pages must be a uint8 [num_pages, nkv, 160 * P] arena with contiguous pages")
    n = kv_pages.shape[2]
    P = n // TOKEN_BYTES
    _need(P >= 8 and not P & (P - 1) and P * TOKEN_BYTES == n,
          f"kv_pages holds {n} bytes per page and head: want 160 * P, P a power of two >= 8")
    return P


def _same_device(first: torch.Tensor, *named) -> int:
    dev = first.device
    for name, t in named:
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, not on {dev}")
    if dev.type != "cuda":
        raise RuntimeError(f"the 4-bit KV ops need CUDA tensors, got {dev}")
    return dev.index


def _vector(name: str, t: torch.Tensor, dtype: torch.dtype, n: int) -> None:
    _need(t.dtype is dtype and t.dim() == 1 and t.shape[0] == n and (n < 2 or t.stride(0) == 1),
          f"{name} must be a contiguous {dtype} vector of {n} entries")


def _rows(name: str, t: torch.Tensor, n: int, heads: int) -> None:
    _need(t.dtype is _BF16 and t.shape == (n, heads, HEAD_DIM) and t.stride(2) == 1,
          f"{name} must be bf16 [{n}, {heads}, {HEAD_DIM}] with a contiguous head dim")


# torch's raw getter: what torch.cuda.current_device() returns, less its look at the lazy start (the
# tensors of a call are on the device already).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_CODE = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_uint32: "I",
         ctypes.c_float: "f", ctypes.c_size_t: "N"}
_PROTOTYPE = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)


def packer(args: type[ctypes.Structure]):
    """``pack(*fields)``: the bytes of a struct of that type with these fields, in a third of the time
    that building the struct takes."""
    layout = "@" + "".join(_CODE[t] for _, t in args._fields_)
    return struct.Struct(f"{layout}{ctypes.sizeof(args) - struct.calcsize(layout)}x").pack


def _entry(name: str, args: type[ctypes.Structure]):
    """``call(index, *fields)``: the library's ``name`` on the current stream of device ``index``."""
    pack, fn = packer(args), None

    def call(index: int, *fields) -> None:
        nonlocal fn
        if fn is None:
            fn = _PROTOTYPE((name, _lib.load()))
        try:
            packed = pack(*fields)
        except struct.error as e:
            raise RuntimeError(f"{name}: {e}") from None
        if index == _current_device():
            rc = fn(packed, _stream_at(index))
        else:
            with torch.cuda.device(index):
                rc = fn(packed, _stream_at(index))
        if rc:
            _lib.check(rc, name)

    return call


_append = _entry("solort_attn_qk_norm_rope_append_int4", _lib.SolortInt4AppendArgs)
_store = _entry("solort_attn_kv_store_int4", _lib.SolortInt4StoreArgs)
_load = _entry("solort_attn_kv_load_int4", _lib.SolortInt4LoadArgs)
_decode = _entry("solort_attn_decode_int4", _lib.SolortInt4DecodeArgs)


# The conditions of a call are looked at together first, since a decode step's calls are as short as
# their checks; only where one fails are they gone through one by one, for the error's words.

def append_into(qkv, q_norm_weight, k_norm_weight, eps: float, cos, sin, positions, slots, kv_pages,
                q_out) -> None:
    """The batch attention prologue into the 4-bit cache: the body of
    ``solort_attn::qk_norm_rope_append_int4``. Head counts follow from ``q_out`` and ``kv_pages``."""
    t = qkv.shape[0] if qkv.dim() else 0
    pages, cs, outs = kv_pages.shape, cos.shape, q_out.shape
    index = qkv.get_device()
    sp, so, sc, sx = kv_pages.stride(), q_out.stride(), cos.stride(), qkv.stride()
    P = pages[2] // TOKEN_BYTES if len(pages) == 3 else 0
    if not (P >= 8 and not P & (P - 1) and sp[2] == 1 and kv_pages.dtype is _U8 and
            P * TOKEN_BYTES == pages[2] and len(outs) == 3 and len(cs) == 2 and index >= 0 and
            index == kv_pages.get_device() == q_out.get_device() == cos.get_device() ==
            sin.get_device() == positions.get_device() == slots.get_device() ==
            q_norm_weight.get_device() == k_norm_weight.get_device() and
            _BF16 is qkv.dtype is q_out.dtype is cos.dtype is sin.dtype is q_norm_weight.dtype is
            k_norm_weight.dtype and _I64 is positions.dtype is slots.dtype and
            outs == (t, outs[1], HEAD_DIM) and so[2] == 1 and
            qkv.shape == (t, (outs[1] + 2 * pages[1]) * HEAD_DIM) and sx[1] == 1 and
            q_norm_weight.shape == k_norm_weight.shape == (HEAD_DIM,) and
            q_norm_weight.is_contiguous() and k_norm_weight.is_contiguous() and
            cs == sin.shape and cs[1] == HEAD_DIM and sc == sin.stride() and sc[1] == 1 and
            positions.shape == slots.shape == (t,) and positions.is_contiguous() and
            slots.is_contiguous()):
        page_size(kv_pages)
        _same_device(qkv, ("kv_pages", kv_pages), ("q_out", q_out), ("cos", cos), ("sin", sin),
                     ("positions", positions), ("slots", slots),
                     ("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight))
        _need(q_out.dim() == 3, "q_out must be [tokens, num_qo_heads, 128]")
        _rows("q_out", q_out, t, outs[1])
        _need(qkv.dtype is _BF16 and qkv.dim() == 2 and qkv.stride(1) == 1 and
              qkv.shape[1] == (outs[1] + 2 * pages[1]) * HEAD_DIM,
              f"qkv must be bf16 [tokens, ({outs[1]} + 2 * {pages[1]}) * 128] with contiguous rows")
        for name, w in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
            _need(w.dtype is _BF16 and w.shape == (HEAD_DIM,) and w.stride(0) == 1,
                  f"{name} must be a contiguous bf16 [128] vector")
        _vector("positions", positions, _I64, t)
        _vector("slots", slots, _I64, t)
        raise RuntimeError("cos and sin must be bf16 [rows, 128] tables with equal strides and "
                           "contiguous rows")
    _append(index, qkv.data_ptr(), sx[0], t, outs[1], pages[1], HEAD_DIM, q_norm_weight.data_ptr(),
            k_norm_weight.data_ptr(), eps, cos.data_ptr(), sin.data_ptr(), sc[0], cs[0],
            positions.data_ptr(), slots.data_ptr(), q_out.data_ptr(), so[0], so[1],
            kv_pages.data_ptr(), sp[0], sp[1], P, pages[0])


def _key_value(call, key, value, slots, kv_pages) -> None:
    pages, sp = kv_pages.shape, kv_pages.stride()
    sk, sv, index, n = key.stride(), value.stride(), key.get_device(), slots.numel()
    P = pages[2] // TOKEN_BYTES if len(pages) == 3 else 0
    if not (P >= 8 and not P & (P - 1) and sp[2] == 1 and kv_pages.dtype is _U8 and
            P * TOKEN_BYTES == pages[2] and index >= 0 and
            index == value.get_device() == slots.get_device() == kv_pages.get_device() and
            _BF16 is key.dtype is value.dtype and slots.dtype is _I64 and slots.shape == (n,) and
            slots.is_contiguous() and
            key.shape == value.shape == (n, pages[1], HEAD_DIM) and sk[2] == 1 == sv[2]):
        page_size(kv_pages)
        _same_device(kv_pages, ("key", key), ("value", value), ("slots", slots))
        _vector("slots", slots, _I64, n)
        _rows("key", key, n, pages[1])
        _rows("value", value, n, pages[1])
    call(index, key.data_ptr(), value.data_ptr(), sk[0], sk[1], sv[0], sv[1], n, pages[1], HEAD_DIM,
         slots.data_ptr(), kv_pages.data_ptr(), sp[0], sp[1], P, pages[0])


def store_into(key, value, slots, kv_pages) -> None:
    """Quantise ``key / value [tokens, nkv, 128]`` to ``slots``: ``solort_attn::kv_store_int4``."""
    _key_value(_store, key, value, slots, kv_pages)


def load_into(kv_pages, slots, key, value) -> None:
    """The held values at ``slots`` to ``key / value``: ``solort_attn::kv_load_int4``."""
    _key_value(_load, key, value, slots, kv_pages)


def decode_fields(q, kv_pages, block_table, q_pos, out, max_kv_len: int, scale: float | None, q_lens,
                  num_ctas: int) -> tuple:
    """The device index and the checked fields of a decode call before its workspace."""
    shape, pages, table, st = q.shape, kv_pages.shape, block_table.shape, block_table.stride()
    sq, so, sp, index = q.stride(), out.stride(), kv_pages.stride(), q.get_device()
    P = pages[2] // TOKEN_BYTES if len(pages) == 3 else 0
    if not (P >= 8 and not P & (P - 1) and sp[2] == 1 and kv_pages.dtype is _U8 and
            P * TOKEN_BYTES == pages[2] and len(shape) == 4 and len(table) == 2 and index >= 0 and
            index == kv_pages.get_device() == block_table.get_device() == q_pos.get_device() ==
            out.get_device() and _BF16 is q.dtype is out.dtype and block_table.dtype is _I32 and
            q_pos.dtype is _I64 and shape[3] == HEAD_DIM and sq[3] == 1 and out.shape == shape and
            so[3] == 1 and table[0] == shape[0] and (table[1] < 2 or st[1] == 1) and
            0 < max_kv_len <= table[1] * P and q_pos.shape == shape[:1] and q_pos.is_contiguous()):
        page_size(kv_pages)
        _same_device(q, ("kv_pages", kv_pages), ("block_table", block_table), ("q_pos", q_pos),
                     ("out", out))
        _need(q.dtype is _BF16 and q.dim() == 4 and shape[3] == HEAD_DIM and sq[3] == 1,
              "q must be bf16 [batch, q_len, num_qo_heads, 128] with a contiguous head dim")
        _need(out.dtype is _BF16 and out.shape == shape and so[3] == 1,
              "out must be bf16, of the shape of q, with a contiguous head dim")
        _need(block_table.dtype is _I32 and len(table) == 2 and table[0] == shape[0] and
              (table[1] < 2 or st[1] == 1),
              "block_table must be int32 [batch, max_pages] with contiguous rows")
        _need(0 < max_kv_len <= table[1] * P,
              f"max_kv_len must be in 1..{table[1] * P}, the keys a block-table row can hold, "
              f"got {max_kv_len}")
        _vector("q_pos", q_pos, _I64, shape[0])
    if q_lens is not None:
        _need(q_lens.device == q.device, f"q_lens is on {q_lens.device}, not on {q.device}")
        _vector("q_lens", q_lens, _I32, shape[0])
    return (index, q.data_ptr(), sq[0], sq[1], sq[2], out.data_ptr(), so[0], so[1], so[2],
            kv_pages.data_ptr(), sp[0], sp[1], P, pages[0], block_table.data_ptr(), st[0], q_pos.data_ptr(),
            0 if q_lens is None else q_lens.data_ptr(), shape[0], shape[1], shape[2], pages[1], HEAD_DIM,
            max_kv_len, _SCALE if scale is None else scale, num_ctas)


_SCALE = HEAD_DIM ** -0.5


def decode_into(q, kv_pages, block_table, q_pos, out, workspace, max_kv_len: int,
                scale: float | None = None, q_lens=None, num_ctas: int = 0,
                stable_prefix: bool = False) -> None:
    """``out = attention(q, 4-bit pages)``: the body of ``solort_attn::gqa_decode_paged_int4``. A short
    or misaligned workspace is the library's SOLORT_ERR_WORKSPACE, raised as ``RuntimeError``."""
    fields = decode_fields(q, kv_pages, block_table, q_pos, out, max_kv_len, scale, q_lens, num_ctas)
    at = n = 0
    if workspace.numel():
        _need(workspace.get_device() == fields[0], f"workspace is on {workspace.device}, not on {q.device}")
        _need(workspace.is_contiguous(), "workspace must be contiguous")
        at, n = workspace.data_ptr(), workspace.nbytes
    if q.numel():
        _decode(*fields, at, n, _lib.DECODE_STABLE_PREFIX if stable_prefix else 0)


def decode_workspace_bytes(batch: int, q_len: int, num_qo_heads: int, num_kv_heads: int,
                           max_kv_len: int, num_ctas: int = 0) -> int:
    """Workspace bytes a 4-bit decode call with these sizes needs on the current device."""
    a = _lib.SolortInt4DecodeArgs()
    a.batch, a.q_len, a.num_qo_heads, a.num_kv_heads, a.head_dim = (
        batch, q_len, num_qo_heads, num_kv_heads, HEAD_DIM)
    a.max_kv_len, a.num_ctas = max_kv_len, num_ctas
    need = ctypes.c_size_t(0)
    _lib.check(_lib.load().solort_attn_decode_int4_workspace_size(_byref(a), _byref(need)),
               "solort_attn_decode_int4_workspace_size")
    return int(need.value)
