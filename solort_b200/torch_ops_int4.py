"""The paged 4-bit KV cache's ops registered with torch as ``torch.ops.solort_attn.*_int4``, beside
those of ``solort_b200.torch_ops`` and by its rules: each writes into caller-provided tensors and
returns nothing, has a fake (meta) implementation, and only a CUDA kernel (CPU tensors raise).

* ``qk_norm_rope_append_int4``: a batch's attention prologue, keys and values appended in 4 bits.
* ``kv_store_int4`` / ``kv_load_int4``: rows to and from slots of the arena.
* ``gqa_decode_paged_int4``: decode and verify attention over the arena and a block table.

Reference counterparts are the bf16 ops' (``src/solort/model/cuda_graph_executor.py:168-184,250-263``,
``src/solort/cache/kv_cache.py:86-256``); the reference holds no cache below 16 bits.
"""

from __future__ import annotations

import torch

from solort_b200 import _calls_int4 as C
from solort_b200.torch_ops import NAMESPACE

SCHEMAS = {
    "qk_norm_rope_append_int4": (
        "qk_norm_rope_append_int4(Tensor qkv, Tensor q_norm_weight, Tensor k_norm_weight, float eps, "
        "Tensor cos, Tensor sin, Tensor positions, Tensor slots, Tensor(a!) kv_pages, "
        "Tensor(b!) q_out) -> ()"),
    "kv_store_int4": (
        "kv_store_int4(Tensor key, Tensor value, Tensor slots, Tensor(a!) kv_pages) -> ()"),
    "kv_load_int4": (
        "kv_load_int4(Tensor kv_pages, Tensor slots, Tensor(a!) key, Tensor(b!) value) -> ()"),
    "gqa_decode_paged_int4": (
        "gqa_decode_paged_int4(Tensor q, Tensor kv_pages, Tensor block_table, Tensor q_pos, "
        "Tensor(a!) out, Tensor(b!) workspace, int max_kv_len, float? scale=None, "
        "Tensor? q_lens=None, int num_ctas=0, bool stable_prefix=False) -> ()"),
}

_LIB = torch.library.Library(NAMESPACE, "FRAGMENT")
for _schema in SCHEMAS.values():
    _LIB.define(_schema)


_LIB.impl("qk_norm_rope_append_int4", C.append_into, "CUDA")
_LIB.impl("kv_store_int4", C.store_into, "CUDA")
_LIB.impl("kv_load_int4", C.load_into, "CUDA")
_LIB.impl("gqa_decode_paged_int4", C.decode_into, "CUDA")


# ---- fake (meta) implementations: the same shape / dtype rules, no data access ----

def _fake_append(qkv, q_norm_weight, k_norm_weight, eps, cos, sin, positions, slots, kv_pages, q_out):
    C.page_size(kv_pages)
    nkv = kv_pages.shape[1]
    C._need(q_out.dim() == 3 and qkv.dim() == 2 and
            qkv.shape[1] == (q_out.shape[1] + 2 * nkv) * C.HEAD_DIM,
            "qkv must be [tokens, (num_qo_heads + 2 * nkv) * 128]")
    C._rows("q_out", q_out, qkv.shape[0], q_out.shape[1])
    C._need(cos.shape == sin.shape and cos.dim() == 2 and cos.shape[1] == C.HEAD_DIM,
            "cos and sin must be [rows, 128]")
    C._vector("positions", positions, torch.int64, qkv.shape[0])
    C._vector("slots", slots, torch.int64, qkv.shape[0])


def _fake_key_value(key, value, slots, kv_pages):
    C.page_size(kv_pages)
    C._need(slots.dim() == 1, "slots must be a vector")
    C._vector("slots", slots, torch.int64, slots.shape[0])
    C._rows("key", key, slots.shape[0], kv_pages.shape[1])
    C._rows("value", value, slots.shape[0], kv_pages.shape[1])


def _fake_load(kv_pages, slots, key, value):
    _fake_key_value(key, value, slots, kv_pages)


def _fake_decode(q, kv_pages, block_table, q_pos, out, workspace, max_kv_len, scale=None, q_lens=None,
                 num_ctas=0, stable_prefix=False):
    P = C.page_size(kv_pages)
    C._need(q.dtype == torch.bfloat16 and q.dim() == 4 and q.shape[3] == C.HEAD_DIM,
            "q must be bf16 [batch, q_len, num_qo_heads, 128]")
    C._need(q.shape[2] % kv_pages.shape[1] == 0, "num_qo_heads must be a multiple of num_kv_heads")
    C._need(out.shape == q.shape and out.dtype == torch.bfloat16, "out must match q (bf16)")
    C._need(block_table.dtype == torch.int32 and block_table.dim() == 2 and
            block_table.shape[0] == q.shape[0], "block_table must be int32 [batch, max_pages]")
    C._need(0 < max_kv_len <= block_table.shape[1] * P,
            "max_kv_len exceeds the pages a block-table row can hold")
    C._vector("q_pos", q_pos, torch.int64, q.shape[0])


for _name, _fn in (("qk_norm_rope_append_int4", _fake_append), ("kv_store_int4", _fake_key_value),
                   ("kv_load_int4", _fake_load), ("gqa_decode_paged_int4", _fake_decode)):
    torch.library.register_fake(f"{NAMESPACE}::{_name}", _fn, lib=_LIB)

OPS = tuple(SCHEMAS)
