// Rows into and out of the 4-bit KV cache (layout and formula: int4.cuh).
//
// append_kernel: the attention prologue for a 4-bit cache. Per token, from the fused QKV projection:
// q_out = rope(norm(q)), and the codes of rope(norm(k)) and of v at the token's slot. Reference:
// src/solort/model/cuda_graph_executor.py _rmsnorm :25-28, _cos_sin :95-98, _rope :100-102, and the
// slot-mapped store of src/solort/cache/kv_cache.py:136-149,191-235; one position and one slot per
// token, so one launch serves a batch of sequences, where the reference runs one at a time.
// store_kernel: the codes of given K / V rows. load_kernel: the values of given slots as bf16 rows.
//
// Eight lanes hold a row of 128 dims: lane l takes dims 8l..8l+7 and 64 + 8l..64 + 8l+7, two 16-byte
// accesses, and so both members of its rotate-half pairs; a quantisation group of 32 is four
// adjacent lanes. A warp works on four rows.
//
// All three are bound by the bytes they move, and for a decode step by their launch.
#include <math.h>

#include "host_util.h"
#include "int4.cuh"

namespace solort {

__device__ unsigned g_int4_rows_status;

namespace i4 {

constexpr int kRowThreads = 128;
constexpr int kRowsPerCta = kRowThreads / 8;

struct Arena {
  uint8_t* base;
  int64_t page_stride, head_stride;
  int page_shift, page_mask;
  long long slots;  // num_pages * page_size
};

// The block of `slot`, or nullptr. A slot of -1 is padding and passes silently.
__device__ __forceinline__ uint8_t* slot_block(const Arena& ar, long long slot, int head) {
  const int row = static_cast<int>(slot) & ar.page_mask;
  return ar.base + block_offset(slot >> ar.page_shift, row, head, ar.page_stride, ar.head_stride);
}

struct AppendParams {
  const bf16* qkv;
  int64_t qkv_st;
  int t, nh, nkv;
  const bf16* qn;
  const bf16* kn;
  float eps;
  const bf16* cos;
  const bf16* sin;
  int64_t rope_st;
  int rope_rows;
  const int64_t* positions;
  const int64_t* slots;
  bf16* q_out;
  int64_t qo_st, qo_sh;
  Arena ar;
};

// The norm's sum of squares is fp32 for queries, which are rounded to bf16 at the end, and fp64 for
// keys: a key's last fp32 bit can decide between two codes, and with the sum all but exact its value
// does not depend on the order of the sum. Norm and rotation stay in fp32 with one rounding at the
// end (the bf16 cache's prologue rounds after each step, as the reference's torch ops do).
__global__ void __launch_bounds__(kRowThreads) append_kernel(const AppendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, l8 = lane & 7;
  const unsigned mask = 0xffu << (lane & 24);
  const int heads = p.nh + 2 * p.nkv;
  const int row = blockIdx.x * kRowsPerCta + (threadIdx.x >> 3);
  if (row >= p.t * heads) return;
  const int tok = row / heads, head = row - tok * heads;
  const long long slot = p.slots[tok], pos = p.positions[tok];
  if (slot == -1) return;
  if (slot < 0 || slot >= p.ar.slots || pos < 0 || pos >= p.rope_rows) {
    if (l8 == 0) atomicOr(&g_int4_rows_status, kDevErrSlot);
    return;
  }
  const bf16* src = p.qkv + tok * p.qkv_st + head * kHD + l8 * 8;
  float a[8], b[8];
  unpack8(*reinterpret_cast<const uint4*>(src), a);
  unpack8(*reinterpret_cast<const uint4*>(src + 64), b);
  const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
  if (!is_v) {
    float r;
    if (is_q) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      r = rsqrtf(ss * (1.f / kHD) + p.eps);
    } else {
      double ss = 0.;
#pragma unroll
      for (int i = 0; i < 8; ++i)  // products of bf16 values are exact in fp32
        ss += static_cast<double>(a[i] * a[i]) + static_cast<double>(b[i] * b[i]);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      r = static_cast<float>(rsqrt(ss * (1. / kHD) + static_cast<double>(p.eps)));
    }
    const bf16* wp = (is_q ? p.qn : p.kn) + l8 * 8;
    const int64_t ro = pos * p.rope_st + l8 * 8;
    float w[8], ca[8], cb[8], sa[8], sb[8];
    unpack8(*reinterpret_cast<const uint4*>(wp), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = __fmul_rn(__fmul_rn(a[i], r), w[i]);
    unpack8(*reinterpret_cast<const uint4*>(wp + 64), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __fmul_rn(__fmul_rn(b[i], r), w[i]);
    unpack8(*reinterpret_cast<const uint4*>(p.cos + ro), ca);
    unpack8(*reinterpret_cast<const uint4*>(p.cos + ro + 64), cb);
    unpack8(*reinterpret_cast<const uint4*>(p.sin + ro), sa);
    unpack8(*reinterpret_cast<const uint4*>(p.sin + ro + 64), sb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = __fadd_rn(__fmul_rn(x, ca[i]), __fmul_rn(-y, sa[i]));
      b[i] = __fadd_rn(__fmul_rn(y, cb[i]), __fmul_rn(x, sb[i]));
    }
    if (is_q) {
      bf16* o = p.q_out + tok * p.qo_st + head * p.qo_sh + l8 * 8;
      *reinterpret_cast<uint4*>(o) = pack8(a);
      *reinterpret_cast<uint4*>(o + 64) = pack8(b);
      return;
    }
  }
  uint8_t* blk = slot_block(p.ar, slot, head - p.nh - (is_v ? p.nkv : 0));
  const Group ga = quantise8(a, mask), gb = quantise8(b, mask);
  store_row(blk, static_cast<int>(slot) & 7, l8, is_v, ga, gb);
}

struct StoreParams {
  const bf16* key;
  const bf16* value;
  int64_t k_st, k_sh, v_st, v_sh;
  int t, nkv;
  const int64_t* slots;
  Arena ar;
};

__global__ void __launch_bounds__(kRowThreads) store_kernel(const StoreParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, l8 = lane & 7;
  const unsigned mask = 0xffu << (lane & 24);
  const int row = blockIdx.x * kRowsPerCta + (threadIdx.x >> 3);  // (token, K or V, head)
  if (row >= p.t * p.nkv * 2) return;
  const int tok = row / (2 * p.nkv), rem = row - tok * 2 * p.nkv;
  const bool is_v = rem >= p.nkv;
  const int head = is_v ? rem - p.nkv : rem;
  const long long slot = p.slots[tok];
  if (slot == -1) return;
  if (slot < 0 || slot >= p.ar.slots) {
    if (l8 == 0) atomicOr(&g_int4_rows_status, kDevErrSlot);
    return;
  }
  const bf16* src = (is_v ? p.value + tok * p.v_st + head * p.v_sh
                          : p.key + tok * p.k_st + head * p.k_sh) + l8 * 8;
  float a[8], b[8];
  unpack8(*reinterpret_cast<const uint4*>(src), a);
  unpack8(*reinterpret_cast<const uint4*>(src + 64), b);
  const Group ga = quantise8(a, mask), gb = quantise8(b, mask);
  store_row(slot_block(p.ar, slot, head), static_cast<int>(slot) & 7, l8, is_v, ga, gb);
}

struct LoadParams {
  bf16* key;
  bf16* value;
  int64_t k_st, k_sh, v_st, v_sh;
  int t, nkv;
  const int64_t* slots;
  Arena ar;
};

__global__ void __launch_bounds__(kRowThreads) load_kernel(const LoadParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int l8 = threadIdx.x & 7;
  const int row = blockIdx.x * kRowsPerCta + (threadIdx.x >> 3);  // (head, token)
  if (row >= p.t * p.nkv) return;
  const int head = row / p.t, tok = row - head * p.t;
  const long long slot = p.slots[tok];
  if (slot == -1) return;
  if (slot < 0 || slot >= p.ar.slots) {
    if (l8 == 0) atomicOr(&g_int4_rows_status, kDevErrSlot);
    return;
  }
  const uint8_t* blk = slot_block(p.ar, slot, head);
  const int i = static_cast<int>(slot) & 7, t = l8 & 3, g = l8 >> 2;
  const uint32_t* kc = reinterpret_cast<const uint32_t*>(blk + 64 * i + 16 * t);
  const uint32_t* km = reinterpret_cast<const uint32_t*>(blk + kOffKScale + 16 * i);
  const uint32_t* vm = reinterpret_cast<const uint32_t*>(blk + kOffVScale + 16 * i);
  const uint8_t* pair = blk + kOffV + 128 * (i >> 1) + 4 * g + 2 * (i & 1);
  uint32_t va = 0, vb = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint8_t* unit = pair + 16 * ((2 * t + h) ^ (i & 6));
    va |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(unit)) << (16 * h);
    vb |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(unit + 8)) << (16 * h);
  }
  float x[8];
  bf16* k = p.key + tok * p.k_st + head * p.k_sh + l8 * 8;
  held8(kc[g], km[g], x);
  *reinterpret_cast<uint4*>(k) = pack8(x);
  held8(kc[g + 2], km[g + 2], x);
  *reinterpret_cast<uint4*>(k + 64) = pack8(x);
  bf16* v = p.value + tok * p.v_st + head * p.v_sh + l8 * 8;
  held8(va, vm[g], x);
  *reinterpret_cast<uint4*>(v) = pack8(x);
  held8(vb, vm[g + 2], x);
  *reinterpret_cast<uint4*>(v + 64) = pack8(x);
}

// Checks shared by the three entry points: the arena and the slots.
int make_arena(const void* pages, int64_t page_stride, int64_t head_stride, int32_t page_size,
               int32_t num_pages, int32_t num_kv_heads, int32_t head_dim, const int64_t* slots,
               int32_t num_tokens, Arena* ar) {
  if (head_dim != kHD) return SOLORT_ERR_UNSUPPORTED;
  if (!pages || num_kv_heads <= 0 || num_pages <= 0 || num_tokens < 0 || (num_tokens && !slots))
    return SOLORT_ERR_INVALID_ARGUMENT;
  if (page_size < kBlockTokens || (page_size & (page_size - 1)) != 0)
    return SOLORT_ERR_INVALID_ARGUMENT;
  if (!aligned(pages, 16) || ((page_stride | head_stride) & 15) || !aligned(slots, 8))
    return SOLORT_ERR_INVALID_ARGUMENT;
  if (page_stride < 0 || head_stride < 0) return SOLORT_ERR_INVALID_ARGUMENT;
  ar->base = static_cast<uint8_t*>(const_cast<void*>(pages));
  ar->page_stride = page_stride;
  ar->head_stride = head_stride;
  ar->page_shift = 0;
  while ((1 << ar->page_shift) < page_size) ++ar->page_shift;
  ar->page_mask = page_size - 1;
  ar->slots = static_cast<long long>(num_pages) * page_size;
  return SOLORT_OK;
}

template <typename P>
int launch_rows(void (*kernel)(const P), const P& prm, int64_t rows, void* stream) {
  if (rows > (1ll << 30)) return SOLORT_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + kRowsPerCta - 1) / kRowsPerCta));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, prm) != cudaSuccess) return SOLORT_ERR_CUDA;
  return launch_status();
}

}  // namespace i4

int read_int4_rows_status(unsigned* flags) {
  unsigned v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_int4_rows_status, sizeof(v)) != cudaSuccess) return SOLORT_ERR_CUDA;
  if (v && cudaMemcpyToSymbol(g_int4_rows_status, &zero, sizeof(zero)) != cudaSuccess)
    return SOLORT_ERR_CUDA;
  *flags |= v;
  return SOLORT_OK;
}

}  // namespace solort

using namespace solort;

extern "C" int solort_attn_qk_norm_rope_append_int4(const SolortInt4AppendArgs* a, void* stream) {
  if (!a) return SOLORT_ERR_INVALID_ARGUMENT;
  i4::AppendParams p{};
  int rc = i4::make_arena(a->kv_pages, a->kv_stride_page, a->kv_stride_head, a->page_size,
                          a->num_pages, a->num_kv_heads, a->head_dim, a->slots, a->num_tokens, &p.ar);
  if (rc != SOLORT_OK) return rc;
  if (a->num_qo_heads <= 0 || a->rope_rows <= 0) return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->num_tokens == 0) return SOLORT_OK;
  if (!a->qkv || !a->q_norm_weight || !a->k_norm_weight || !a->cos || !a->sin || !a->positions ||
      !a->q_out)
    return SOLORT_ERR_INVALID_ARGUMENT;
  const int64_t strides =
      a->qkv_stride_token | a->rope_stride | a->q_out_stride_token | a->q_out_stride_head;
  if ((strides & 7) || !aligned(a->qkv, 16) || !aligned(a->q_norm_weight, 16) ||
      !aligned(a->k_norm_weight, 16) || !aligned(a->cos, 16) || !aligned(a->sin, 16) ||
      !aligned(a->q_out, 16) || !aligned(a->positions, 8))
    return SOLORT_ERR_INVALID_ARGUMENT;
  DeviceInfo di;
  rc = current_device_info(&di);
  if (rc != SOLORT_OK) return rc;
  p.qkv = static_cast<const bf16*>(a->qkv);
  p.qkv_st = a->qkv_stride_token;
  p.t = a->num_tokens;
  p.nh = a->num_qo_heads;
  p.nkv = a->num_kv_heads;
  p.qn = static_cast<const bf16*>(a->q_norm_weight);
  p.kn = static_cast<const bf16*>(a->k_norm_weight);
  p.eps = a->eps;
  p.cos = static_cast<const bf16*>(a->cos);
  p.sin = static_cast<const bf16*>(a->sin);
  p.rope_st = a->rope_stride;
  p.rope_rows = a->rope_rows;
  p.positions = a->positions;
  p.slots = a->slots;
  p.q_out = static_cast<bf16*>(a->q_out);
  p.qo_st = a->q_out_stride_token;
  p.qo_sh = a->q_out_stride_head;
  const int64_t rows =
      static_cast<int64_t>(a->num_tokens) * (static_cast<int64_t>(a->num_qo_heads) + 2ll * a->num_kv_heads);
  return i4::launch_rows(i4::append_kernel, p, rows, stream);
}

extern "C" int solort_attn_kv_store_int4(const SolortInt4StoreArgs* a, void* stream) {
  if (!a) return SOLORT_ERR_INVALID_ARGUMENT;
  i4::StoreParams p{};
  int rc = i4::make_arena(a->kv_pages, a->kv_stride_page, a->kv_stride_head, a->page_size,
                          a->num_pages, a->num_kv_heads, a->head_dim, a->slots, a->num_tokens, &p.ar);
  if (rc != SOLORT_OK) return rc;
  if (a->num_tokens == 0) return SOLORT_OK;
  if (!a->key || !a->value) return SOLORT_ERR_INVALID_ARGUMENT;
  const int64_t strides = a->key_stride_token | a->key_stride_head | a->value_stride_token |
                          a->value_stride_head;
  if ((strides & 7) || !aligned(a->key, 16) || !aligned(a->value, 16))
    return SOLORT_ERR_INVALID_ARGUMENT;
  DeviceInfo di;
  rc = current_device_info(&di);
  if (rc != SOLORT_OK) return rc;
  p.key = static_cast<const bf16*>(a->key);
  p.value = static_cast<const bf16*>(a->value);
  p.k_st = a->key_stride_token;
  p.k_sh = a->key_stride_head;
  p.v_st = a->value_stride_token;
  p.v_sh = a->value_stride_head;
  p.t = a->num_tokens;
  p.nkv = a->num_kv_heads;
  p.slots = a->slots;
  return i4::launch_rows(i4::store_kernel, p, 2ll * a->num_tokens * a->num_kv_heads, stream);
}

extern "C" int solort_attn_kv_load_int4(const SolortInt4LoadArgs* a, void* stream) {
  if (!a) return SOLORT_ERR_INVALID_ARGUMENT;
  i4::LoadParams p{};
  int rc = i4::make_arena(a->kv_pages, a->kv_stride_page, a->kv_stride_head, a->page_size,
                          a->num_pages, a->num_kv_heads, a->head_dim, a->slots, a->num_tokens, &p.ar);
  if (rc != SOLORT_OK) return rc;
  if (a->num_tokens == 0) return SOLORT_OK;
  if (!a->key || !a->value) return SOLORT_ERR_INVALID_ARGUMENT;
  const int64_t strides = a->key_stride_token | a->key_stride_head | a->value_stride_token |
                          a->value_stride_head;
  if ((strides & 7) || !aligned(a->key, 16) || !aligned(a->value, 16))
    return SOLORT_ERR_INVALID_ARGUMENT;
  DeviceInfo di;
  rc = current_device_info(&di);
  if (rc != SOLORT_OK) return rc;
  p.key = static_cast<bf16*>(a->key);
  p.value = static_cast<bf16*>(a->value);
  p.k_st = a->key_stride_token;
  p.k_sh = a->key_stride_head;
  p.v_st = a->value_stride_token;
  p.v_sh = a->value_stride_head;
  p.t = a->num_tokens;
  p.nkv = a->num_kv_heads;
  p.slots = a->slots;
  return i4::launch_rows(i4::load_kernel, p, static_cast<int64_t>(a->num_tokens) * a->num_kv_heads,
                         stream);
}
