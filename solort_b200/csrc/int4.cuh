// The 4-bit KV cache shared by the int4 kernels: its layout, and the two directions of its codes.
//
// A row of 128 values is held in four groups of 32 dims, each as mid + scale * (code - 7.5) with
// codes 0..15 and bf16 mid and scale:
//   mid = bf16((lo + hi) / 2), scale = bf16 rounded up of max(hi - mid, mid - lo) / 7.5,
//   code = rint((x - mid) / scale + 7.5), so |x - held| <= scale / 2 for every value of the group.
// The scale is rounded up and measured from the rounded mid, so no value falls off the ends of the
// code range, however far the group lies from zero. Codes are symmetric about 7.5: a product with
// (code - 7.5) stays as small as the values themselves, which is what bounds the error that the
// attention's bf16 probabilities add.
//
// Layout: pages of P tokens (a power of two >= 8), one KV head of a page contiguous, P / 8 blocks
// of 8 tokens of kBlockBytes. Every byte belongs to one token, so rows are written without a
// read-modify-write. The order inside a block is the order in which the attention's tensor-core
// fragments want the codes (int4_decode.cu): a thread takes its part of a key row, or of a pair of
// value rows, with one 16-byte shared-memory load, free of bank conflicts.
//   keys    token i at 64 i: 16-byte chunk t, word g: nibble j = code of dim 32 g + 8 t + j
//   scales  token i at 512 + 16 i: word g = scale (low half), mid (high half)
//   values  token pair p at 640 + 128 p: 16-byte unit u at place u ^ 2p, word g: the low half holds
//           token 2p and the high half token 2p + 1; nibble j of a half = code of dim 32 g + 4 u + j
//   scales  of the values at 1152 + 16 i, as the keys'
#pragma once

#include "common.cuh"

namespace solort {
namespace i4 {

constexpr int kHD = 128;
constexpr int kBlockTokens = 8;
constexpr int kOffKScale = 512;
constexpr int kOffV = 640;
constexpr int kOffVScale = 1152;
constexpr int kBlockBytes = 1280;
constexpr int kTokenBytes = kBlockBytes / kBlockTokens;  // K and V of one token of one head

// Device status bits of the int4 kernels (bit 0, a wait past its limit, is common.cuh's).
constexpr unsigned kDevErrSlot = 1u << 4;  // a slot outside the arena or a position without a RoPE row
constexpr unsigned kDevErrPage = 1u << 5;  // a block-table entry outside the arena

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ float lo_bf16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  v[0] = lo_bf16(u.x);
  v[1] = hi_bf16(u.x);
  v[2] = lo_bf16(u.y);
  v[3] = hi_bf16(u.y);
  v[4] = lo_bf16(u.z);
  v[5] = hi_bf16(u.z);
  v[6] = lo_bf16(u.w);
  v[7] = hi_bf16(u.w);
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}

// Byte offset of slot row `token` of KV head `head` (its 8-token block) in an arena.
__device__ __forceinline__ int64_t block_offset(int64_t page, int row, int head, int64_t page_stride,
                                                int64_t head_stride) {
  return page * page_stride + head * head_stride +
         static_cast<int64_t>(row / kBlockTokens) * kBlockBytes;
}

// Codes (nibble j = x[j]) and packed scale / mid of one group of 32 values held by four adjacent
// lanes, eight each. Every step is an IEEE fp32 operation in a fixed order, without contraction, so
// a value next to the border of two codes falls on the same side wherever the formula is evaluated
// in fp32; the quotients are true divisions, for which exact halves stay exact halves. A group with
// an infinity or a NaN reads back as NaN throughout: a broken input stays visible.
struct Group {
  uint32_t codes, meta;
};
__device__ __forceinline__ Group quantise8(const float (&x)[8], unsigned mask) {
  float lo = x[0], hi = x[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad |= (__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u;
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
  }
  const unsigned quad = 0xfu << (threadIdx.x & 28);
  bad = (__ballot_sync(mask, bad) & quad) != 0;
  const float mid = __bfloat162float(
      __float2bfloat16_rn(__fadd_rn(__fmul_rn(0.5f, lo), __fmul_rn(0.5f, hi))));
  const float need = __fdiv_rn(fmaxf(__fsub_rn(hi, mid), __fsub_rn(mid, lo)), 7.5f);
  const uint32_t sbits = (__float_as_uint(need) + 0xffffu) & 0xffff0000u;  // need >= 0
  const float step = sbits ? __uint_as_float(sbits) : 1.f;
  Group g;
  g.codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = __float2int_rn(__fadd_rn(__fdiv_rn(__fsub_rn(x[i], mid), step), 7.5f));
    g.codes |= static_cast<uint32_t>(min(max(c, 0), 15)) << (4 * i);
  }
  g.meta = bad ? 0x7fff7fffu : (sbits >> 16) | (__float_as_uint(mid) & 0xffff0000u);
  return g;
}

// Write one row, held by eight adjacent lanes (lane l8: dims 8 l8.. as `a`, 64 + 8 l8.. as `b`), to
// row i of the block at `blk`.
__device__ __forceinline__ void store_row(uint8_t* blk, int i, int l8, bool is_value, const Group& a,
                                          const Group& b) {
  const int t = l8 & 3, g = l8 >> 2;  // `a` is group g, `b` group g + 2
  if (is_value) {
    uint8_t* pair = blk + kOffV + 128 * (i >> 1) + 4 * g + 2 * (i & 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint8_t* unit = pair + 16 * ((2 * t + h) ^ (i & 6));  // place u ^ 2p, p = i / 2
      *reinterpret_cast<uint16_t*>(unit) = static_cast<uint16_t>(a.codes >> (16 * h));
      *reinterpret_cast<uint16_t*>(unit + 8) = static_cast<uint16_t>(b.codes >> (16 * h));
    }
  } else {
    uint32_t* chunk = reinterpret_cast<uint32_t*>(blk + 64 * i + 16 * t);
    chunk[g] = a.codes;
    chunk[g + 2] = b.codes;
  }
  if (t == 0) {
    uint32_t* m = reinterpret_cast<uint32_t*>(blk + (is_value ? kOffVScale : kOffKScale) + 16 * i);
    m[g] = a.meta;
    m[g + 2] = b.meta;
  }
}

// The values of eight codes: mid + scale * (code - 7.5); the product is exact in fp32.
__device__ __forceinline__ void held8(uint32_t codes, uint32_t meta, float (&x)[8]) {
  const float s = lo_bf16(meta), mid = hi_bf16(meta);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = fmaf(s, static_cast<float>((codes >> (4 * i)) & 15u) - 7.5f, mid);
}

}  // namespace i4
}  // namespace solort
