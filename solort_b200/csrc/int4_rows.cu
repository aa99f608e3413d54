// Rows into and out of the 4-bit KV cache (layout and formula: int4.cuh).
//
// append_kernel: the attention prologue for a 4-bit cache. Per token, from the fused QKV projection:
// q_out = rope(norm(q)), and the codes of rope(norm(k)) and of v at the token's slot. Reference:
// src/solort/model/cuda_graph_executor.py _rmsnorm :25-28, _cos_sin :95-98, _rope :100-102, and the
// slot-mapped store of src/solort/cache/kv_cache.py:136-149,191-235; one position and one slot per
// token, so one launch serves a batch of sequences, where the reference runs one at a time.
// store_kernel: the codes of given K / V rows. load_kernel: the values of given slots as bf16 rows.
//
// Where a row is rotated, eight lanes hold its 128 dims: lane l takes dims 8l..8l+7 and 64 + 8l..64 +
// 8l+7, two 16-byte accesses, and so both members of its rotate-half pairs; a quantisation group of 32
// is four adjacent lanes. Where it is only quantised, four lanes hold it, a group each: what a group
// costs once (its scale, mid and reciprocal) is then paid for 32 values instead of 8, and nothing is
// exchanged. A CTA works on tokens of one head, which share the cache lines that they write; the
// append's query CTAs go over several heads, with the tokens' RoPE rows in registers.
//
// All three are bound by the bytes they move, and for a decode step by their launch. 8 KV heads: storing
// 16380 rows 17.0 us (5.2 TB/s), loading 32001 rows 30.2 us (5.7 TB/s), appending a prompt of 8190 tokens
// with 32 query heads 38.3 us (4.8 TB/s: a token's RoPE rows wait for its position, and 96 registers, with
// 20 bytes a thread spilt, leave 20 warps an SM to hide that); one token's append 2.3 us.
#include <math.h>

#include "host_util.h"
#include "int4.cuh"

namespace solort {

__device__ unsigned g_int4_rows_status;

namespace i4 {

constexpr int kRowThreads = 128;
constexpr int kRowsPerCta = kRowThreads / 8;
constexpr int kGroupRowsPerCta = kRowThreads / 4;  // of four lanes a row
// CTAs per SM from which a CTA takes more than one round of rows, or heads: a prompt of 8190 tokens appended
// 38.4 us with 8 and with 16, 42.2 with 32; 16380 rows stored 16.6 us with 8, 17.0 with 16, 17.8 with 32.
constexpr int kFullCtas = 16;

struct Arena {
  uint8_t* base;
  int64_t page_stride, head_stride;
  int page_shift, page_mask;
  long long slots;  // num_pages * page_size
};

// The block of `slot`, which is one of the arena's (row_there).
__device__ __forceinline__ uint8_t* slot_block(const Arena& ar, long long slot, int head) {
  const int row = static_cast<int>(slot) & ar.page_mask;
  return ar.base + block_offset(slot >> ar.page_shift, row, head, ar.page_stride, ar.head_stride);
}

struct AppendParams {
  const bf16* qkv;
  int64_t qkv_st;
  int t, nh, nkv;
  int heads, q_ctas, kv_ctas;  // heads of a CTA, and CTAs along the query heads and the KV heads
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

__device__ __forceinline__ f2 sum_of_products(f2 a, f2 b, f2 c, f2 d) {
  const float2 x = both(a), y = both(b), u = both(c), v = both(d);
  return pair(__fadd_rn(__fmul_rn(x.x, y.x), __fmul_rn(u.x, v.x)),
              __fadd_rn(__fmul_rn(x.y, y.y), __fmul_rn(u.y, v.y)));
}

// True if `slot` (and `pos`) name a row; a bad one is reported, but for -1, which is padding.
__device__ __forceinline__ bool row_there(long long slot, const Arena& ar, bool report, bool pos_ok = true) {
  if (slot == -1) return false;
  if (slot >= 0 && slot < ar.slots && pos_ok) return true;
  if (report) atomicOr(&g_int4_rows_status, kDevErrSlot);
  return false;
}

// The norm's sum of squares is fp32 for queries, which are rounded to bf16 at the end, and fp64 for
// keys: a key's last fp32 bit can decide between two codes, and with the sum all but exact its value
// does not depend on the order of the sum; its products and sums are each rounded on their own, without
// contraction. Norm and rotation stay in fp32 with one rounding at the end (the bf16 cache's prologue
// rounds after each step, as the reference's torch ops do).
// Grid: (tokens, [query heads | key heads | value heads], p.heads each).
__global__ void __launch_bounds__(kRowThreads, 5) append_kernel(const AppendParams p) {
  pdl_wait();
  const int y = blockIdx.y;
  if (y >= p.q_ctas + p.kv_ctas) {  // values: four lanes a row, two heads at a time
    const int g = threadIdx.x & 3, first = (y - p.q_ctas - p.kv_ctas) * p.heads;
    const int last = min(first + p.heads, p.nkv);
    const int tok = blockIdx.x * kRowsPerCta + (threadIdx.x >> 2 & 15);
    if (tok >= p.t) return;
    const long long slot = p.slots[tok], pos = p.positions[tok];
    const uint4* src = reinterpret_cast<const uint4*>(
        p.qkv + tok * p.qkv_st + static_cast<int64_t>(p.nh + p.nkv) * kHD + g * 32);
    int head = first + (threadIdx.x >> 6);
    uint4 u[4];
    if (head < last)
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = src[head * (kHD / 8) + i];
    if (!row_there(slot, p.ar, g == 0, pos >= 0 && pos < p.rope_rows)) return;
    for (; head < last; head += 2) {
      const uint4 v[4] = {u[0], u[1], u[2], u[3]};
      if (head + 2 < last)
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = src[(head + 2) * (kHD / 8) + i];
      uint32_t codes[4];
      const uint32_t meta = quantise32(v, codes);
      store_group(slot_block(p.ar, slot, head), static_cast<int>(slot) & 7, g, true, codes, meta);
    }
    return;
  }
  const int l8 = threadIdx.x & 7;
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  const int tok = blockIdx.x * kRowsPerCta + (threadIdx.x >> 3);
  if (tok >= p.t) return;
  const long long slot = p.slots[tok], pos = p.positions[tok];
  if (!row_there(slot, p.ar, l8 == 0, pos >= 0 && pos < p.rope_rows)) return;
  const bool is_q = y < p.q_ctas;
  const int first = is_q ? y * p.heads : p.nh + (y - p.q_ctas) * p.heads;
  const int last = min(first + p.heads, is_q ? p.nh : p.nh + p.nkv);
  const bf16* src = p.qkv + tok * p.qkv_st + l8 * 8;
  uint4 ua = *reinterpret_cast<const uint4*>(src + first * kHD);
  uint4 ub = *reinterpret_cast<const uint4*>(src + first * kHD + 64);
  f2 ca[4], cb[4], sa[4], sb[4], wa[4], wb[4];
  const int64_t ro = pos * p.rope_st + l8 * 8;
  const bf16* w = (is_q ? p.qn : p.kn) + l8 * 8;
  unpack_pairs(*reinterpret_cast<const uint4*>(p.cos + ro), ca);
  unpack_pairs(*reinterpret_cast<const uint4*>(p.cos + ro + 64), cb);
  unpack_pairs(*reinterpret_cast<const uint4*>(p.sin + ro), sa);
  unpack_pairs(*reinterpret_cast<const uint4*>(p.sin + ro + 64), sb);
  constexpr f2 kMinus = 0x8000000080000000ull;
  f2 a[4], b[4];
  if (!is_q) {
    for (int head = first; head < last; ++head) {
      unpack_pairs(ua, a);
      unpack_pairs(ub, b);
      if (head + 1 < last) {
        ua = *reinterpret_cast<const uint4*>(src + (head + 1) * kHD);
        ub = *reinterpret_cast<const uint4*>(src + (head + 1) * kHD + 64);
      }
      double ss = 0.;
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // squares of bf16 values are exact in fp32
        const float2 x = both(mul2(a[i], a[i])), z = both(mul2(b[i], b[i]));
        ss += static_cast<double>(x.x) + static_cast<double>(x.y);
        ss += static_cast<double>(z.x) + static_cast<double>(z.y);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      unpack_pairs(*reinterpret_cast<const uint4*>(w), wa);  // of the first-level cache, to save registers
      unpack_pairs(*reinterpret_cast<const uint4*>(w + 64), wb);
      const f2 r = dup(static_cast<float>(rsqrt(ss * (1. / kHD) + static_cast<double>(p.eps))));
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // not packed: the compiler contracts packed products and sums
        const f2 x = mul2(mul2(a[i], r), wa[i]), z = mul2(mul2(b[i], r), wb[i]);
        a[i] = sum_of_products(x, ca[i], z, sa[i] ^ kMinus);
        b[i] = sum_of_products(z, cb[i], x, sb[i]);
      }
      const Group ga = quantise8(a, mask), gb = quantise8(b, mask);
      store_key(slot_block(p.ar, slot, head - p.nh), static_cast<int>(slot) & 7, l8, ga, gb);
    }
    return;
  }
  // out = r (x w cos + partner w sin): the weights join the tables once for all heads.
  unpack_pairs(*reinterpret_cast<const uint4*>(w), wa);
  unpack_pairs(*reinterpret_cast<const uint4*>(w + 64), wb);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ca[i] = mul2(ca[i], wa[i]);
    cb[i] = mul2(cb[i], wb[i]);
    sa[i] = mul2(sa[i], wb[i]) ^ kMinus;
    sb[i] = mul2(sb[i], wa[i]);
  }
  bf16* to = p.q_out + tok * p.qo_st + l8 * 8;
  for (int head = first; head < last; ++head) {
    unpack_pairs(ua, a);
    unpack_pairs(ub, b);
    if (head + 1 < last) {
      ua = *reinterpret_cast<const uint4*>(src + (head + 1) * kHD);
      ub = *reinterpret_cast<const uint4*>(src + (head + 1) * kHD + 64);
    }
    f2 sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fma2(a[i], a[i], fma2(b[i], b[i], sum));
    float ss = both(sum).x + both(sum).y;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    const f2 r = dup(rsqrtf(ss * (1.f / kHD) + p.eps));
    f2 x[4], z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = mul2(fma2(a[i], ca[i], mul2(b[i], sa[i])), r);
      z[i] = mul2(fma2(b[i], cb[i], mul2(a[i], sb[i])), r);
    }
    *reinterpret_cast<uint4*>(to + head * p.qo_sh) = pack_pairs(x);
    *reinterpret_cast<uint4*>(to + head * p.qo_sh + 64) = pack_pairs(z);
  }
}

// Rows of a store, so that the row of a CTA's next round stays inside an int.
constexpr int kMostStored = 1 << 30;

struct StoreParams {
  const bf16* key;
  const bf16* value;
  int64_t k_st, k_sh, v_st, v_sh;
  int t, nkv;
  const int64_t* slots;
  Arena ar;
};

// Eight CTAs an SM: 16380 rows 17.0 us; 17.6 with the 65 registers that the compiler takes, seven CTAs. A
// row is read before its slot is known, a padded one too.
__global__ void __launch_bounds__(kRowThreads, 8) store_kernel(const StoreParams p) {
  pdl_wait();
  const int g = threadIdx.x & 3;
  const bool is_v = static_cast<int>(blockIdx.x) >= p.nkv;  // K heads, then V heads
  const int head = blockIdx.x - (is_v ? p.nkv : 0);
  const bf16* src = (is_v ? p.value + head * p.v_sh : p.key + head * p.k_sh) + g * 32;
  const int64_t st = is_v ? p.v_st : p.k_st;
  const int step = gridDim.y * kGroupRowsPerCta;
  int tok = blockIdx.y * kGroupRowsPerCta + (threadIdx.x >> 2);
  uint4 u[4];
  if (tok < p.t)
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = reinterpret_cast<const uint4*>(src + tok * st)[i];
  for (; tok < p.t; tok += step) {
    const long long slot = p.slots[tok];
    const uint4 v[4] = {u[0], u[1], u[2], u[3]};
    if (tok + step < p.t)  // the next round's rows
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = reinterpret_cast<const uint4*>(src + (tok + step) * st)[i];
    if (!row_there(slot, p.ar, g == 0)) continue;
    uint32_t codes[4];
    const uint32_t meta = quantise32(v, codes);
    store_group(slot_block(p.ar, slot, head), static_cast<int>(slot) & 7, g, is_v, codes, meta);
  }
}

struct LoadParams {
  bf16* key;
  bf16* value;
  int64_t k_st, k_sh, v_st, v_sh;
  int t, nkv;
  const int64_t* slots;
  Arena ar;
};

// Sixteen CTAs an SM, all its warps, with four bytes a thread spilt: 32001 rows 30.3 us; 31.0 with two
// registers more, twelve CTAs.
__global__ void __launch_bounds__(kRowThreads, 16) load_kernel(const LoadParams p) {
  pdl_wait();
  const int l8 = threadIdx.x & 7, t = l8 & 3, g = l8 >> 2;
  const int head = blockIdx.x;
  const int tok = (blockIdx.z * gridDim.y + blockIdx.y) * kRowsPerCta + (threadIdx.x >> 3);
  if (tok >= p.t) return;
  const long long slot = p.slots[tok];
  if (!row_there(slot, p.ar, l8 == 0)) return;
  const uint8_t* blk = slot_block(p.ar, slot, head);
  const int i = static_cast<int>(slot) & 7;
  const uint32_t* kc = reinterpret_cast<const uint32_t*>(blk + 64 * i + 16 * t);
  const uint32_t* km = reinterpret_cast<const uint32_t*>(blk + kOffKScale + 16 * i);
  const uint32_t* vm = reinterpret_cast<const uint32_t*>(blk + kOffVScale + 16 * i);
  const uint8_t* values = blk + kOffV + 128 * (i >> 1) + 4 * g + 2 * (i & 1);
  uint32_t va = 0, vb = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint8_t* unit = values + 16 * ((2 * t + h) ^ (i & 6));
    va |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(unit)) << (16 * h);
    vb |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(unit + 8)) << (16 * h);
  }
  const uint32_t ka = kc[g], kb = kc[g + 2], kma = km[g], kmb = km[g + 2], vma = vm[g], vmb = vm[g + 2];
  bf16* k = p.key + tok * p.k_st + head * p.k_sh + l8 * 8;
  *reinterpret_cast<uint4*>(k) = held8(ka, kma);
  *reinterpret_cast<uint4*>(k + 64) = held8(kb, kmb);
  bf16* v = p.value + tok * p.v_st + head * p.v_sh + l8 * 8;
  *reinterpret_cast<uint4*>(v) = held8(va, vma);
  *reinterpret_cast<uint4*>(v + 64) = held8(vb, vmb);
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
int launch_rows(void (*kernel)(const P), const P& prm, int64_t x, int64_t y, int64_t z, void* stream) {
  if (x > (1ll << 30) || y > 65535) return SOLORT_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(x), static_cast<unsigned>(y), static_cast<unsigned>(z));
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

// CTAs along the tokens, `rows` each, for a grid with `y` heads; fewer, with several rounds each, where
// that would give over kFullCtas per SM.
inline int64_t token_ctas(int tokens, int rows, int64_t y, const DeviceInfo& di) {
  const int64_t all = (static_cast<int64_t>(tokens) + rows - 1) / rows;
  const int64_t cap = static_cast<int64_t>(di.sm_count) * kFullCtas / y;
  return all < cap || cap < 1 ? (cap < 1 ? 1 : all) : cap;
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
  // One head per CTA while the GPU is not full, and up to eight (prompt of 8190 tokens: at most four 41.8
  // us, eight 38.4).
  const int64_t x = (static_cast<int64_t>(a->num_tokens) + i4::kRowsPerCta - 1) / i4::kRowsPerCta;
  const int64_t full = static_cast<int64_t>(di.sm_count) * i4::kFullCtas;
  const int64_t per = x * (a->num_qo_heads + 2ll * a->num_kv_heads) / full;
  p.heads = static_cast<int>(per < 1 ? 1 : per > 8 ? 8 : per);
  p.q_ctas = (a->num_qo_heads + p.heads - 1) / p.heads;
  p.kv_ctas = (a->num_kv_heads + p.heads - 1) / p.heads;
  return i4::launch_rows(i4::append_kernel, p, x, p.q_ctas + 2ll * p.kv_ctas, 1, stream);
}

extern "C" int solort_attn_kv_store_int4(const SolortInt4StoreArgs* a, void* stream) {
  if (!a) return SOLORT_ERR_INVALID_ARGUMENT;
  i4::StoreParams p{};
  int rc = i4::make_arena(a->kv_pages, a->kv_stride_page, a->kv_stride_head, a->page_size,
                          a->num_pages, a->num_kv_heads, a->head_dim, a->slots, a->num_tokens, &p.ar);
  if (rc != SOLORT_OK) return rc;
  if (a->num_tokens > i4::kMostStored) return SOLORT_ERR_UNSUPPORTED;
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
  const int64_t y = 2ll * a->num_kv_heads;
  return i4::launch_rows(i4::store_kernel, p, y, i4::token_ctas(a->num_tokens, i4::kGroupRowsPerCta, y, di),
                         1, stream);
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
  const int64_t wide = 32768;
  const int64_t all = (static_cast<int64_t>(a->num_tokens) + i4::kRowsPerCta - 1) / i4::kRowsPerCta;
  return i4::launch_rows(i4::load_kernel, p, a->num_kv_heads, all < wide ? all : wide,
                         (all + wide - 1) / wide, stream);
}
