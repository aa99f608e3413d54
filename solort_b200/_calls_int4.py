"""C-ABI call builders of the paged 4-bit KV cache: the bodies of the ``torch.ops.solort_attn.*_int4``
ops. As ``solort_b200._calls``: each function checks its tensors, packs one argument struct of
``include/solort_attn.h`` and makes one library call on the current stream of the tensors' device; it
writes only the tensors it is given and allocates nothing. Errors raise ``RuntimeError``.
"""

from __future__ import annotations

import ctypes

import torch

from solort_b200 import _lib
from solort_b200._calls import HEAD_DIM, _stream_at

TOKEN_BYTES = 160  # K and V of one token of one KV head: codes, and a scale and a mid per 32 values
_byref, _vp = ctypes.byref, ctypes.c_void_p
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


def _launch(name: str, args, index: int) -> None:
    fn = getattr(_lib.load(), name)
    if index == torch.cuda.current_device():
        rc = fn(_byref(args), _vp(_stream_at(index)))
    else:
        with torch.cuda.device(index):
            rc = fn(_byref(args), _vp(_stream_at(index)))
    if rc:
        _lib.check(rc, name)


def append_into(qkv, q_norm_weight, k_norm_weight, eps: float, cos, sin, positions, slots, kv_pages,
                q_out) -> None:
    """The batch attention prologue into the 4-bit cache: the body of
    ``solort_attn::qk_norm_rope_append_int4``. Head counts follow from ``q_out`` and ``kv_pages``."""
    P = page_size(kv_pages)
    num_pages, nkv, _ = kv_pages.shape
    index = _same_device(qkv, ("kv_pages", kv_pages), ("q_out", q_out), ("cos", cos), ("sin", sin),
                         ("positions", positions), ("slots", slots),
                         ("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight))
    _need(q_out.dim() == 3, "q_out must be [tokens, num_qo_heads, 128]")
    t, nh = qkv.shape[0], q_out.shape[1]
    _rows("q_out", q_out, t, nh)
    _need(qkv.dtype is _BF16 and qkv.dim() == 2 and qkv.stride(1) == 1 and
          qkv.shape[1] == (nh + 2 * nkv) * HEAD_DIM,
          f"qkv must be bf16 [tokens, ({nh} + 2 * {nkv}) * 128] with contiguous rows")
    for name, w in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
        _need(w.dtype is _BF16 and w.shape == (HEAD_DIM,) and w.stride(0) == 1,
              f"{name} must be a contiguous bf16 [128] vector")
    _need(cos.dtype is _BF16 and sin.dtype is _BF16 and cos.dim() == 2 and cos.shape == sin.shape and
          cos.shape[1] == HEAD_DIM and cos.stride() == sin.stride() and cos.stride(1) == 1,
          "cos and sin must be bf16 [rows, 128] tables with equal strides and contiguous rows")
    _vector("positions", positions, _I64, t)
    _vector("slots", slots, _I64, t)
    _launch("solort_attn_qk_norm_rope_append_int4", _lib.SolortInt4AppendArgs(
        qkv.data_ptr(), qkv.stride(0), t, nh, nkv, HEAD_DIM, q_norm_weight.data_ptr(),
        k_norm_weight.data_ptr(), eps, cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0],
        positions.data_ptr(), slots.data_ptr(), q_out.data_ptr(), q_out.stride(0), q_out.stride(1),
        kv_pages.data_ptr(), kv_pages.stride(0), kv_pages.stride(1), P, num_pages), index)


def _key_value(what, key, value, slots, kv_pages):
    P = page_size(kv_pages)
    num_pages, nkv, _ = kv_pages.shape
    index = _same_device(kv_pages, ("key", key), ("value", value), ("slots", slots))
    n = slots.shape[0] if slots.dim() == 1 else -1
    _vector("slots", slots, _I64, n)
    _rows("key", key, n, nkv)
    _rows("value", value, n, nkv)
    return index, what(
        key.data_ptr(), value.data_ptr(), key.stride(0), key.stride(1), value.stride(0),
        value.stride(1), n, nkv, HEAD_DIM, slots.data_ptr(), kv_pages.data_ptr(), kv_pages.stride(0),
        kv_pages.stride(1), P, num_pages)


def store_into(key, value, slots, kv_pages) -> None:
    """Quantise ``key / value [tokens, nkv, 128]`` to ``slots``: ``solort_attn::kv_store_int4``."""
    index, args = _key_value(_lib.SolortInt4StoreArgs, key, value, slots, kv_pages)
    _launch("solort_attn_kv_store_int4", args, index)


def load_into(kv_pages, slots, key, value) -> None:
    """The held values at ``slots`` to ``key / value``: ``solort_attn::kv_load_int4``."""
    index, args = _key_value(_lib.SolortInt4LoadArgs, key, value, slots, kv_pages)
    _launch("solort_attn_kv_load_int4", args, index)


def decode_args(q, kv_pages, block_table, q_pos, out, max_kv_len: int, scale: float | None, q_lens,
                num_ctas: int, stable_prefix: bool):
    """Checked and packed arguments of a decode call without its workspace, and the device index."""
    P = page_size(kv_pages)
    num_pages, nkv, _ = kv_pages.shape
    index = _same_device(q, ("kv_pages", kv_pages), ("block_table", block_table), ("q_pos", q_pos),
                         ("out", out))
    _need(q.dtype is _BF16 and q.dim() == 4 and q.shape[3] == HEAD_DIM and q.stride(3) == 1,
          "q must be bf16 [batch, q_len, num_qo_heads, 128] with a contiguous head dim")
    B, T, H, D = q.shape
    _need(out.dtype is _BF16 and out.shape == q.shape and out.stride(3) == 1,
          "out must be bf16, of the shape of q, with a contiguous head dim")
    _need(block_table.dtype is _I32 and block_table.dim() == 2 and block_table.shape[0] == B and
          (block_table.shape[1] < 2 or block_table.stride(1) == 1),
          "block_table must be int32 [batch, max_pages] with contiguous rows")
    _need(0 < max_kv_len <= block_table.shape[1] * P,
          f"max_kv_len must be in 1..{block_table.shape[1] * P}, the keys a block-table row can hold, "
          f"got {max_kv_len}")
    _vector("q_pos", q_pos, _I64, B)
    if q_lens is not None:
        _need(q_lens.device == q.device, f"q_lens is on {q_lens.device}, not on {q.device}")
        _vector("q_lens", q_lens, _I32, B)
    sq, so = q.stride(), out.stride()
    return index, _lib.SolortInt4DecodeArgs(
        q.data_ptr(), sq[0], sq[1], sq[2], out.data_ptr(), so[0], so[1], so[2], kv_pages.data_ptr(),
        kv_pages.stride(0), kv_pages.stride(1), P, num_pages, block_table.data_ptr(),
        block_table.stride(0), q_pos.data_ptr(), None if q_lens is None else q_lens.data_ptr(), B, T, H,
        nkv, D, max_kv_len, D ** -0.5 if scale is None else scale, num_ctas, None, 0,
        _lib.DECODE_STABLE_PREFIX if stable_prefix else 0)


def decode_into(q, kv_pages, block_table, q_pos, out, workspace, max_kv_len: int,
                scale: float | None, q_lens, num_ctas: int, stable_prefix: bool) -> None:
    """``out = attention(q, 4-bit pages)``: the body of ``solort_attn::gqa_decode_paged_int4``. A short
    or misaligned workspace is the library's SOLORT_ERR_WORKSPACE, raised as ``RuntimeError``."""
    index, a = decode_args(q, kv_pages, block_table, q_pos, out, max_kv_len, scale, q_lens, num_ctas,
                           stable_prefix)
    if workspace.numel():
        _need(workspace.device == q.device, f"workspace is on {workspace.device}, not on {q.device}")
        _need(workspace.is_contiguous(), "workspace must be contiguous")
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if q.numel():
        _launch("solort_attn_decode_int4", a, index)


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
