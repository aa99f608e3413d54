// The 4-bit KV cache shared by the int4 kernels: its layout, and the two directions of its codes.
//
// A row of 128 values is held in four groups of 32 dims, each as mid + scale * (code - 7.5) with
// codes 0..15 and bf16 mid and scale:
//   mid = bf16((lo + hi) / 2), scale = bf16 rounded up of max(hi - mid, mid - lo) / 7.5,
//   code = rint((x - mid) / scale + 7.5), so |x - held| <= scale / 2 for every value of the group.
// The scale is rounded up and measured from the rounded mid, so no value falls off the ends of the
// code range, however far the group lies from zero. Codes are symmetric about 7.5: a product with
// (code - 7.5) stays as small as the values themselves, which is what bounds the error that the
// attention's rounded probabilities add.
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

// Wait for the kernels before this one on the stream, and only then let the next one start: a kernel that
// has started thus has finished kernels behind its predecessor. SOLORT_DECODE_STABLE_PREFIX reads before
// the wait what those have written. Were the order the other way round, a chain of short kernels could all
// be resident at once, and such a read could come before the write of the kernel but one.
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;\ngriddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ float lo_bf16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// Byte offset of slot row `token` of KV head `head` (its 8-token block) in an arena.
__device__ __forceinline__ int64_t block_offset(int64_t page, int row, int head, int64_t page_stride,
                                                int64_t head_stride) {
  return page * page_stride + head * head_stride +
         static_cast<int64_t>(row / kBlockTokens) * kBlockBytes;
}

// Pairs of fp32 (the packed instructions take half the issue slots). The compiler contracts a packed
// product and a packed sum of it.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 dup(float a) { return pair(a, a); }

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN goes on
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// a / b, correctly rounded, from y = 1 / b, correctly rounded: Markstein's correction (IBM J. Res. Dev.
// 34(1), 1990). With q = a y and r = a - q b, exact in an fma, the quotient is q + r y as long as
// nothing underflows.
__device__ __forceinline__ f2 quotient2(f2 a, f2 minus_b, f2 y) {
  const f2 q = mul2(a, y);
  return fma2(fma2(q, minus_b, a), y, q);
}

// The scale and mid of a group of 32 values from its least and greatest, and the codes of its pairs.
//
// Every step is an IEEE fp32 operation in a fixed order, without contraction, so a value next to the
// border of two codes falls on the same side wherever the formula is evaluated in fp32; quotients
// are correctly rounded, so that exact halves stay exact halves. A group with an infinity or a NaN
// (lo, hi: with NaN going on) reads back as NaN throughout: a broken input stays visible.
//
// The quotients by the step are quotient2's, its reciprocal from the hardware's approximation and one
// Newton step (correctly rounded for every bf16 step). Where the step is far from 1 values, mid and step
// are scaled by 2^+-64 first, which changes no quotient: mid is then below 2^-60, or what underflows is
// lost in the sum with 7.5 in any case. No code needs clamping: step >= need (1 - 2^-23), so that
// d / step lies within 7.5 (1 + 2^-22) and its sum with 7.5 rounds to 0..15.
struct Quantiser {
  f2 f, m2, s2, y2;
  uint32_t meta;

  __device__ __forceinline__ Quantiser(float lo, float hi) {
    const float mid = __bfloat162float(
        __float2bfloat16_rn(__fadd_rn(__fmul_rn(0.5f, lo), __fmul_rn(0.5f, hi))));
    const float wide = max_nan(__fsub_rn(hi, mid), __fsub_rn(mid, lo));
    constexpr float kSeventh = 1.f / 7.5f;
    const float n0 = __fmul_rn(wide, kSeventh);
    float need = fmaf(fmaf(-n0, 7.5f, wide), kSeventh, n0);
    float by = 1.f;
    if (__builtin_expect(!(wide >= 0x1p-86f && wide <= 0x1p90f), 0)) {
      need = __fdiv_rn(wide, 7.5f);
      by = wide == 0.f ? 1.f : wide < 1.f ? 0x1p64f : 0x1p-64f;
    }
    const uint32_t sbits = (__float_as_uint(need) + 0xffffu) & 0xffff0000u;  // need >= 0
    const float step = (sbits ? __uint_as_float(sbits) : 1.f) * by;
    float y0;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"(step));
    f = dup(by);
    m2 = dup(-mid * by);
    s2 = dup(-step);
    y2 = dup(fmaf(fmaf(-step, y0, 1.f), y0, y0));
    meta = wide < INFINITY ? __byte_perm(sbits, __float_as_uint(mid), 0x7632) : 0x7fff7fffu;
  }
  // The word of eight codes, nibble j = value j. Rounded to an integer, ties to even, by a sum with
  // 1.5 2^23, whose bits add up to one constant for the eight.
  __device__ __forceinline__ uint32_t codes(const f2 (&x)[4]) const {
    uint32_t w = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      const f2 q = quotient2(fma2(x[i], f, m2), s2, y2);
      const float2 r = both(add2(add2(q, dup(7.5f)), dup(12582912.f)));
      w = (w << 4) + __float_as_uint(r.y);
      w = (w << 4) + __float_as_uint(r.x);
    }
    return w - 0x4b400000u * 0x11111111u;
  }
};

__device__ __forceinline__ void unpack_pairs(const uint4& u, f2 (&x)[4]) {
  x[0] = pair(lo_bf16(u.x), hi_bf16(u.x));
  x[1] = pair(lo_bf16(u.y), hi_bf16(u.y));
  x[2] = pair(lo_bf16(u.z), hi_bf16(u.z));
  x[3] = pair(lo_bf16(u.w), hi_bf16(u.w));
}
__device__ __forceinline__ uint4 pack_pairs(const f2 (&x)[4]) {
  const float2 a = both(x[0]), b = both(x[1]), c = both(x[2]), d = both(x[3]);
  return make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(b.x, b.y), pack_bf16x2(c.x, c.y), pack_bf16x2(d.x, d.y));
}

// A group of fp32 values held by four adjacent lanes, eight each: this lane's codes, and the group's
// scale and mid.
struct Group {
  uint32_t codes, meta;
};
__device__ __forceinline__ Group quantise8(const f2 (&x)[4], unsigned mask) {
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = both(x[i]);
    lo = min_nan(lo, min_nan(v.x, v.y));
    hi = max_nan(hi, max_nan(v.x, v.y));
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(mask, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(mask, hi, o));
  }
  const Quantiser q(lo, hi);
  return {q.codes(x), q.meta};
}

// A group of 32 bf16 values in one lane: its codes (word w: values 8 w .. 8 w + 7), scale and mid.
__device__ __forceinline__ uint32_t quantise32(const uint4 (&u)[4], uint32_t (&codes)[4]) {
  __nv_bfloat162 lo, hi;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u[i]);
    const __nv_bfloat162 l = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
    const __nv_bfloat162 g = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    lo = i ? __hmin2_nan(lo, l) : l;
    hi = i ? __hmax2_nan(hi, g) : g;
  }
  const Quantiser q(min_nan(__low2float(lo), __high2float(lo)), max_nan(__low2float(hi), __high2float(hi)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f2 x[4];
    unpack_pairs(u[i], x);
    codes[i] = q.codes(x);
  }
  return q.meta;
}

// Write one key row, held by eight adjacent lanes (lane l8: dims 8 l8.. as `a`, 64 + 8 l8.. as `b`),
// to row i of the block at `blk`.
__device__ __forceinline__ void store_key(uint8_t* blk, int i, int l8, const Group& a, const Group& b) {
  const int t = l8 & 3, g = l8 >> 2;  // `a` is of group g, `b` of group g + 2
  uint32_t* chunk = reinterpret_cast<uint32_t*>(blk + 64 * i + 16 * t);
  chunk[g] = a.codes;
  chunk[g + 2] = b.codes;
  if (t == 0) {
    uint32_t* m = reinterpret_cast<uint32_t*>(blk + kOffKScale + 16 * i);
    m[g] = a.meta;
    m[g + 2] = b.meta;
  }
}
// Write group g of a row, held by one lane.
__device__ __forceinline__ void store_group(uint8_t* blk, int i, int g, bool is_value, const uint32_t (&codes)[4],
                                            uint32_t meta) {
  if (is_value) {
    uint8_t* values = blk + kOffV + 128 * (i >> 1) + 4 * g + 2 * (i & 1);
#pragma unroll
    for (int u = 0; u < 8; ++u)  // place u ^ 2p, p = i / 2
      *reinterpret_cast<uint16_t*>(values + 16 * (u ^ (i & 6))) = static_cast<uint16_t>(codes[u >> 1] >> (16 * (u & 1)));
  } else {
    uint32_t* keys = reinterpret_cast<uint32_t*>(blk + 64 * i) + g;
#pragma unroll
    for (int t = 0; t < 4; ++t) keys[4 * t] = codes[t];
  }
  reinterpret_cast<uint32_t*>(blk + (is_value ? kOffVScale : kOffKScale) + 16 * i)[g] = meta;
}

// The values of eight codes as bf16: mid + scale (code - 7.5), whose product is exact in fp32. Nibble n of
// a word in the low bits of 2^23 is the float 2^23 + 16^n code, and the scale takes 16^-n.
__device__ __forceinline__ uint4 held8(uint32_t codes, uint32_t meta) {
  const f2 s = dup(lo_bf16(meta)), mid = dup(hi_bf16(meta));
  const f2 s12 = mul2(s, pair(0x1p-4f, 0x1p-8f)), s34 = mul2(s, pair(0x1p-12f, 0x1p-16f));
  const f2 centre12 = pair(-0x1p23f - 7.5f * 16, -0x1p23f - 7.5f * 256);
  const f2 centre34 = pair(-0x1p23f - 7.5f * 4096, -0x1p23f - 7.5f * 65536);
  uint32_t o[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = h ? codes >> 12 : codes << 4;  // the half's codes are nibbles 1 to 4
    auto at = [&](uint32_t nibble) { return __uint_as_float(w & nibble | 0x4b000000u); };
    const float2 a = both(fma2(s12, add2(pair(at(0xf0u), at(0xf00u)), centre12), mid));
    const float2 b = both(fma2(s34, add2(pair(at(0xf000u), at(0xf0000u)), centre34), mid));
    o[2 * h] = pack_bf16x2(a.x, a.y);
    o[2 * h + 1] = pack_bf16x2(b.x, b.y);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace i4
}  // namespace solort
