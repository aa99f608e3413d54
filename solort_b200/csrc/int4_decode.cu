// GQA decode / verify attention over the paged 4-bit KV cache (layout and formula: int4.cuh).
//
// With keys held as k = mid + scale (c - 7.5) and values likewise, per group g of 32 dims,
//   q . k       = sum_g scale_g (sum_d q_d c_d - 7.5 sum_d q_d) + mid_g sum_d q_d
//   sum_t p v_d = sum_t (p scale_g) c_d - 7.5 sum_t (p scale_g) + sum_t p mid_g
// so the tensor cores multiply the integer codes and the scales are applied to their fp32 results
// (keys) or to the probabilities (values): the cache is never expanded. A nibble becomes a bf16
// operand in one and-or: 0x4300 | c is the bf16 number 128 + c exactly, and the 128 joins the 7.5
// in the two correction terms (both are taken of exactly the bf16 numbers that the products use, so
// they cancel in the fp32 accumulators). The one rounding on the way is p scale to bf16, the same
// half step as p's in a bf16 attention, against codes symmetric about zero.
//
// Both products are transposed, S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16, tokens or dims as
// the 16 rows, query rows as the 8 columns), so that the few query rows of a decode fill an n8 tile;
// P^T turns into the second product's operand with movmatrix. The rate that the memory asks for
// (0.28 tokens of a head per ns and SM) leaves 27 warp instructions per token and head; this form
// needs about 16. tcgen05 would leave them as they are: the work is unpacking codes, which its
// shared-memory operands would have to be written back for.
//
// Work split: the cache's 16-token tiles, over all sequences, KV heads and blocks of query rows, are
// one list, and CTA c of n takes the tiles [T c / n, T (c + 1) / n): sequences of any lengths load
// every SM alike, and the workspace is two partials per CTA whatever the batch. A CTA's eight warps
// take its tiles in turn, each warp with a ring of kDepth tiles of its own (one bulk copy of 2560
// contiguous bytes a tile, an mbarrier each), so warps meet only at the end of a (sequence, head)
// segment. A segment that is a whole (sequence, head) writes its final rows; parts meet in
// merge_kernel. Lengths are read on the device, and merge_kernel repeats the same division.
//
// Reference semantics: src/solort/model/cuda_graph_executor.py:168,180-184 (keys 0..pos), :250
// (query i at vpos0 + i), src/solort/cache/kv_cache.py:136-149 (slot = bt[pos // P] * P + pos % P).
#include <atomic>
#include <math.h>

#include "host_util.h"
#include "int4.cuh"

namespace solort {

__device__ unsigned g_int4_decode_status;

namespace i4 {

constexpr int kTile = 16;                          // tokens of a tile: two blocks
constexpr int kTileBytes = 2 * kBlockBytes;        // 2560
constexpr int kDepth = 4;                          // tiles in flight per warp
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMinTiles = kWarps;                  // tiles per CTA at least: one per warp
constexpr int kDirectTiles = 2 * kWarps;           // up to this many tiles a (sequence, head) is one CTA
constexpr float kShift = 135.5f;                   // 128 of the bf16 codes and 7.5 of the formula
// A row's running maximum is raised only when a score passes it by 2^8: p stays below 2^8, far
// inside bf16 and fp32, and the accumulators are rescaled a few times per split instead of always.
constexpr float kLazy = 8.f;

template <int NT>  // n8 tiles of query rows
struct Cfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kRing = kWarps * kDepth * kTileBytes;
  static constexpr int kRed = kWarps * kRows * kHD * 4;
  static constexpr int kOffRed = kRing;
  static constexpr int kOffMl = kOffRed + kRed;                  // [warp][row] (max, sum)
  static constexpr int kOffBar = kOffMl + kWarps * kRows * 8;    // [warp][depth]
  static constexpr int kOffFlag = kOffBar + kWarps * kDepth * 8;
  static constexpr int kSmem = kOffFlag + 16;
  static constexpr int kCtasPerSm = NT == 1 ? 2 : 1;
};
static_assert(Cfg<1>::kSmem <= 115712, "two CTAs per SM");

struct Params {
  const bf16* q;
  int64_t q_sb, q_st, q_sh;
  bf16* out;
  int64_t o_sb, o_st, o_sh;
  const uint8_t* pages;
  int64_t page_stride, head_stride;
  const int32_t* block_table;
  int64_t bt_stride;
  int page_size, page_shift, num_pages;
  const int64_t* q_pos;
  const int32_t* q_lens;
  float* part_o;    // [2 * ctas][rows][128], not normalised
  float2* part_ml;  // [2 * ctas][rows] running max (log2 domain) and sum
  int batch, q_len, nh, nkv, group, max_kv_len;
  int direct;  // grid (head and row block, sequence): no parts
  int ctas;
  int stable_prefix;
  float scale_log2;
};

struct Seq {  // one sequence's share of the list
  long long qpos;
  int kv_end, rows, rb, tiles;
  __device__ __forceinline__ int units(int nkv) const { return nkv * rb; }
  __device__ __forceinline__ int total(int nkv) const { return nkv * rb * tiles; }
};

template <int NT>
__device__ __forceinline__ Seq load_seq(const Params& p, int b) {
  Seq s;
  s.qpos = p.q_pos[b];
  const int ql = p.q_lens ? max(0, min(p.q_lens[b], p.q_len)) : p.q_len;
  // Positions far outside the cache are cut before the sum, which then cannot overflow.
  const long long cut = max(-(1ll << 40), min(s.qpos, 1ll << 40));
  s.kv_end = static_cast<int>(max(0ll, min(cut + ql, static_cast<long long>(p.max_kv_len))));
  s.qpos = cut;
  s.rows = ql * p.group;
  s.rb = (s.rows + Cfg<NT>::kRows - 1) / Cfg<NT>::kRows;
  s.tiles = s.rows ? (s.kv_end + kTile - 1) / kTile : 0;
  return s;
}

__device__ __forceinline__ int warp_inclusive(int v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// All tiles of the list; and the tiles before sequence `b` (with the whole warp).
template <int NT>
__device__ __forceinline__ int list_total(const Params& p, int b, int* before) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int c = 0; c < p.batch; c += 32) {
    const int v = c + lane < p.batch ? load_seq<NT>(p, c + lane).total(p.nkv) : 0;
    const int incl = warp_inclusive(v);
    if (b >= c && b < c + 32) *before = run + __shfl_sync(0xffffffffu, incl - v, b - c);
    run += __shfl_sync(0xffffffffu, incl, 31);
  }
  return run;
}

// The sequence that holds tile x < total, and the tiles before it.
template <int NT>
__device__ __forceinline__ int find_seq(const Params& p, int x, int* before) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int c = 0; c < p.batch; c += 32) {
    const int v = c + lane < p.batch ? load_seq<NT>(p, c + lane).total(p.nkv) : 0;
    const int incl = warp_inclusive(v);
    const unsigned past = __ballot_sync(0xffffffffu, x < run + incl);
    if (past) {
      const int l = __ffs(past) - 1;
      *before = run + __shfl_sync(0xffffffffu, incl - v, l);
      return c + l;
    }
    run += __shfl_sync(0xffffffffu, incl, 31);
  }
  *before = run;
  return p.batch;
}

// CTAs at work on a list of `total` tiles, and the first tile of CTA c.
__device__ __forceinline__ int active_ctas(int total, int ctas) {
  return max(1, min(ctas, (total + kMinTiles - 1) / kMinTiles));
}
__device__ __forceinline__ int first_tile(int total, int n, int c) {
  return static_cast<int>(static_cast<long long>(total) * c / n);
}
__device__ __forceinline__ int cta_of(int total, int n, int x) {
  return static_cast<int>(((x + 1ll) * n - 1) / total);
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {  // 128 + nibble, low and high half
  return (w & 0x000f000fu) | 0x43004300u;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

// One warp's state over a segment.
template <int NT>
struct Acc {
  float o[NT][4][2][4];  // [group][m16 tile]: dims 32g + 4 (lane / 4) + 2h, + 1; rows 2 (lane % 4), + 1
  float ps[NT][2][4];    // sums of the bf16 p scale: groups 2i (c0, c1) and 2i + 1 (c2, c3)
  float pm[NT][4][2];    // this lane's tokens' sum of p mid
  float l[NT][2], m[NT][2];
};

// One tile of 16 tokens for the segment's rows. MASKED: some row does not see some token.
template <int NT, bool MASKED>
__device__ __forceinline__ void tile_step(uint32_t base, const uint32_t (&qf)[NT][4][4],
                                          const float (&qs)[NT][4][2], Acc<NT>& A, float scale_log2,
                                          const int (&lim)[NT][2], int tok0, bool ok0, bool ok1) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float s[NT][4];
  {
    const uint4 k0 = lds128(base + 64 * g + 16 * t), k1 = lds128(base + kBlockBytes + 64 * g + 16 * t);
    const uint4 m0 = lds128(base + kOffKScale + 16 * g);
    const uint4 m1 = lds128(base + kBlockBytes + kOffKScale + 16 * g);
#pragma unroll
    for (int grp = 0; grp < 4; ++grp) {
      const uint32_t w0 = word(k0, grp), w1 = word(k1, grp);
      const uint32_t a0[4] = {codes_bf16(w0), codes_bf16(w1), codes_bf16(w0 >> 4), codes_bf16(w1 >> 4)};
      const uint32_t a1[4] = {codes_bf16(w0 >> 8), codes_bf16(w1 >> 8), codes_bf16(w0 >> 12),
                              codes_bf16(w1 >> 12)};
      const float s0 = lo_bf16(word(m0, grp)), d0 = hi_bf16(word(m0, grp));
      const float s1 = lo_bf16(word(m1, grp)), d1 = hi_bf16(word(m1, grp));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float q0 = qs[nt][grp][0], q1 = qs[nt][grp][1];
        float c[4] = {-kShift * q0, -kShift * q1, -kShift * q0, -kShift * q1};
        mma_bf16_16816(c, a0, qf[nt][grp][0], qf[nt][grp][1]);
        mma_bf16_16816(c, a1, qf[nt][grp][2], qf[nt][grp][3]);
        if (grp == 0) {
          s[nt][0] = s0 * c[0] + d0 * q0;
          s[nt][1] = s0 * c[1] + d0 * q1;
          s[nt][2] = s1 * c[2] + d1 * q0;
          s[nt][3] = s1 * c[3] + d1 * q1;
        } else {
          s[nt][0] += s0 * c[0] + d0 * q0;
          s[nt][1] += s0 * c[1] + d0 * q1;
          s[nt][2] += s1 * c[2] + d1 * q0;
          s[nt][3] += s1 * c[3] + d1 * q1;
        }
      }
    }
  }
  bool vis[NT][4];
  bool raise = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[nt][i] *= scale_log2;
      if (MASKED) {
        vis[nt][i] = (i < 2 ? ok0 && tok0 + g <= lim[nt][i & 1] : ok1 && tok0 + 8 + g <= lim[nt][i & 1]);
        if (!vis[nt][i]) s[nt][i] = -INFINITY;
      }
      raise |= s[nt][i] > A.m[nt][i & 1] + kLazy;
    }
  if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        mx = fmaxf(mx, A.m[nt][e]);
        const float f = A.m[nt][e] == -INFINITY ? 0.f : ex2(A.m[nt][e] - mx);
        A.m[nt][e] = mx;
        A.l[nt][e] *= f;
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) {
          A.pm[nt][grp][e] *= f;
          A.ps[nt][grp >> 1][(grp & 1) * 2 + e] *= f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            A.o[nt][grp][h][e] *= f;
            A.o[nt][grp][h][2 + e] *= f;
          }
        }
      }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = A.m[nt][i & 1];
      s[nt][i] = ex2(s[nt][i] - (MASKED && m == -INFINITY ? 0.f : m));
      A.l[nt][i & 1] += s[nt][i];
    }

  const uint32_t va = base + kOffV + 128 * t + 16 * (g ^ (2 * t));
  const uint4 v0 = lds128(va), v1 = lds128(va + kBlockBytes);
  const uint4 m0 = lds128(base + kOffVScale + 16 * g);
  const uint4 m1 = lds128(base + kBlockBytes + kOffVScale + 16 * g);
  constexpr uint32_t kOnes = 0x3f803f80u;
#pragma unroll
  for (int grp = 0; grp < 4; ++grp) {
    const float s0 = lo_bf16(word(m0, grp)), d0 = hi_bf16(word(m0, grp));
    const float s1 = lo_bf16(word(m1, grp)), d1 = hi_bf16(word(m1, grp));
    const uint32_t w0 = word(v0, grp), w1 = word(v1, grp);
    const uint32_t a0[4] = {codes_bf16(w0), codes_bf16(w0 >> 4), codes_bf16(w1), codes_bf16(w1 >> 4)};
    const uint32_t a1[4] = {codes_bf16(w0 >> 8), codes_bf16(w0 >> 12), codes_bf16(w1 >> 8),
                            codes_bf16(w1 >> 12)};
    const uint32_t ones[4] = {grp & 1 ? 0u : kOnes, grp & 1 ? kOnes : 0u, grp & 1 ? 0u : kOnes,
                              grp & 1 ? kOnes : 0u};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // A token that a row does not see adds nothing, whatever its scale and mid are.
        const float sc = i < 2 ? s0 : s1, md = i < 2 ? d0 : d1;
        x[i] = MASKED && !vis[nt][i] ? 0.f : s[nt][i] * sc;
        A.pm[nt][grp][i & 1] += MASKED && !vis[nt][i] ? 0.f : s[nt][i] * md;
      }
      const uint32_t b0 = transpose8x8(pack_bf16x2(x[0], x[1]));
      const uint32_t b1 = transpose8x8(pack_bf16x2(x[2], x[3]));
      mma_bf16_16816(A.o[nt][grp][0], a0, b0, b1);
      mma_bf16_16816(A.o[nt][grp][1], a1, b0, b1);
      mma_bf16_16816(A.ps[nt][grp >> 1], ones, b0, b1);
    }
  }
}

__device__ __forceinline__ void write_row4(const Params& p, int b, int kvh, int r, int c, float4 v) {
  const int i = r / p.group, h = kvh * p.group + r - i * p.group;
  uint2 pk;
  pk.x = pack_bf16x2(v.x, v.y);
  pk.y = pack_bf16x2(v.z, v.w);
  *reinterpret_cast<uint2*>(p.out + b * p.o_sb + i * p.o_st + h * p.o_sh + c) = pk;
}

template <int NT>
__global__ void __launch_bounds__(kThreads, Cfg<NT>::kCtasPerSm) decode_kernel(const Params p) {
  using C = Cfg<NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);
  float2* ml = reinterpret_cast<float2*>(smem + C::kOffMl);
  volatile int* failed = reinterpret_cast<volatile int*>(smem + C::kOffFlag);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::kOffBar) + warp * kDepth;
  const uint32_t ring = smem_u32(smem) + warp * kDepth * kTileBytes;

  pdl_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < kDepth; ++i) mbar_init(&bar[i], 1);
    fence_mbarrier_init();
  }
  if (tid == 0) *failed = 0;
  __syncthreads();
  const bool early = p.stable_prefix != 0;
  if (!early) pdl_wait();

  // This CTA's tiles [x0, x1) of the list, and the sequence of the first.
  int x0, x1, b, base;
  if (p.direct) {
    b = blockIdx.y;
    base = 0;
    const Seq s = load_seq<NT>(p, b);
    const int unit = blockIdx.x;
    if (unit >= s.units(p.nkv) || s.tiles == 0) {
      pdl_wait();
      const int kvh = s.rb ? unit / s.rb : 0, r0 = s.rb ? (unit % s.rb) * C::kRows : 0;
      if (unit < s.units(p.nkv))  // rows that see no key
        for (int i = tid; i < min(C::kRows, s.rows - r0) * (kHD / 4); i += kThreads)
          write_row4(p, b, kvh, r0 + i / (kHD / 4), (i % (kHD / 4)) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
      return;
    }
    x0 = unit * s.tiles;
    x1 = x0 + s.tiles;
  } else {
    int unused = 0;
    const int total = list_total<NT>(p, -1, &unused);
    const int n = active_ctas(total, p.ctas);
    if (total == 0 || static_cast<int>(blockIdx.x) >= n) {
      pdl_wait();
      return;
    }
    x0 = first_tile(total, n, blockIdx.x);
    x1 = first_tile(total, n, blockIdx.x + 1);
    b = find_seq<NT>(p, x0, &base);
  }

  // ---- the copies: lane i of the warp holds the addresses of the warp's tile 32 k + i ----
  const int mine = x1 - x0 > warp ? (x1 - x0 - warp + kWarps - 1) / kWarps : 0;  // tiles of this warp
  int ib = b, ibase = base;                        // sequence of this lane's tile
  const uint8_t *src0 = nullptr, *src1 = nullptr;  // its blocks; nullptr: none, or not in the arena
  bool stable = false;
  unsigned none0 = 0, none1 = 0;  // lanes whose first / second block is not there
  auto resolve = [&](int k) {     // tiles k .. k + 31
    src0 = src1 = nullptr;
    stable = false;
    const int x = x0 + warp + (k + lane) * kWarps;
    if (k + lane < mine) {
      Seq s = load_seq<NT>(p, ib);
      while (x >= ibase + s.total(p.nkv)) {
        ibase += s.total(p.nkv);
        s = load_seq<NT>(p, ++ib);
      }
      const int unit = (x - ibase) / s.tiles, tok = (x - ibase - unit * s.tiles) * kTile;
      const int head = unit / s.rb;
      const int32_t* bt = p.block_table + ib * p.bt_stride;
      const int pg0 = bt[tok >> p.page_shift];
      int pg1 = pg0;
      const bool two = s.kv_end - tok > kBlockTokens;
      if (two && p.page_size == kBlockTokens) pg1 = bt[(tok >> p.page_shift) + 1];
      const int row = tok & (p.page_size - 1);
      if (pg0 >= 0 && pg0 < p.num_pages)
        src0 = p.pages + block_offset(pg0, row, head, p.page_stride, p.head_stride);
      if (two && pg1 >= 0 && pg1 < p.num_pages)
        src1 = p.page_size == kBlockTokens
                   ? p.pages + block_offset(pg1, 0, head, p.page_stride, p.head_stride)
                   : src0 + kBlockBytes;
      if (!src0 || (two && !src1)) atomicOr(&g_int4_decode_status, kDevErrPage);
      stable = tok + kTile <= s.qpos;
    }
    none0 = __ballot_sync(0xffffffffu, src0 == nullptr);
    none1 = __ballot_sync(0xffffffffu, src1 == nullptr);
  };
  unsigned gone = 0;  // per ring slot: bit 2s block 0, bit 2s + 1 block 1 is not there
  auto issue = [&](int k) {  // the warp's tile k
    const int i = k & 31, slot = k % kDepth;
    if (i == 0 && k > 0) resolve(k);
    gone = (gone & ~(3u << (2 * slot))) | ((none0 >> i) & 1u) << (2 * slot) |
           ((none1 >> i) & 1u) << (2 * slot + 1);
    if (lane == i) {
      const uint32_t dst = ring + slot * kTileBytes, mb = smem_u32(&bar[slot]);
      mbar_arrive_expect_tx(&bar[slot], (src0 ? kBlockBytes : 0) + (src1 ? kBlockBytes : 0));
      if (src0 && src1 == src0 + kBlockBytes) {
        bulk_load(dst, src0, kTileBytes, mb);
      } else {
        if (src0) bulk_load(dst, src0, kBlockBytes, mb);
        if (src1) bulk_load(dst + kBlockBytes, src1, kBlockBytes, mb);
      }
    }
  };
  int issued = 0;
  resolve(0);
  if (early) {  // tiles that no earlier kernel on the stream still writes
    const unsigned steady = __ballot_sync(0xffffffffu, stable);
    while (issued < kDepth && issued < mine && (steady >> issued & 1u)) issue(issued++);
    pdl_wait();
  }
  while (issued < kDepth && issued < mine) issue(issued++);

  // ---- the segments: the parts of (sequence, head, row block) in [x0, x1) ----
  int done = 0;    // tiles of this warp consumed
  int stuck = -1;  // the tile whose copy did not come
  bool ok = true;
  Seq s = load_seq<NT>(p, b);
  int x = x0;
  while (x < x1) {
    while (x >= base + s.total(p.nkv)) {
      base += s.total(p.nkv);
      s = load_seq<NT>(p, ++b);
    }
    const int unit = (x - base) / s.tiles;
    const int u0 = base + unit * s.tiles, u1 = u0 + s.tiles;  // the unit's tiles
    const int seg_end = min(u1, x1);
    const int kvh = unit / s.rb, r0 = (unit - kvh * s.rb) * C::kRows;
    const int live = min(C::kRows, s.rows - r0);

    // Query fragments: column n = lane / 4 of each n8 tile; k pairs (j, j + 4) of dims 32 grp + 8t.
    uint32_t qf[NT][4][4];
    float qs[NT][4][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + nt * 8 + g;
      const int i = r / p.group;
      const bf16* src = p.q + b * p.q_sb + i * p.q_st + (kvh * p.group + r - i * p.group) * p.q_sh + 8 * t;
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < s.rows) v = *reinterpret_cast<const uint4*>(src + 32 * grp);
        qf[nt][grp][0] = __byte_perm(v.x, v.z, 0x5410);
        qf[nt][grp][1] = __byte_perm(v.x, v.z, 0x7632);
        qf[nt][grp][2] = __byte_perm(v.y, v.w, 0x5410);
        qf[nt][grp][3] = __byte_perm(v.y, v.w, 0x7632);
        float f[8];
        unpack8(v, f);
        float sum = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qs[nt][grp][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
        qs[nt][grp][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      }
    }
    Acc<NT> A;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) A.l[nt][e] = 0.f, A.m[nt][e] = -INFINITY;
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
        A.pm[nt][grp][0] = A.pm[nt][grp][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) A.o[nt][grp][0][i] = A.o[nt][grp][1][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) A.ps[nt][0][i] = A.ps[nt][1][i] = 0.f;
    }
    const long long first_lim = s.qpos + r0 / p.group;  // last key of the segment's first row
    bool any = false;
    for (; done < mine && x0 + warp + done * kWarps < seg_end; ++done) {
      const int slot = done % kDepth;
      const int tok = (x0 + warp + done * kWarps - u0) * kTile;
      if (ok) ok = mbar_wait(&bar[slot], (done / kDepth) & 1, &g_int4_decode_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok && stuck < 0) stuck = done;
      if (ok) {
        any = true;
        const uint32_t at = ring + slot * kTileBytes;
        const unsigned bad = gone >> (2 * slot) & 3u;
        if (bad || tok + kTile > s.kv_end || tok + kTile - 1 > first_lim) {
          int lim[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = r0 + nt * 8 + 2 * t + e;
              const long long last = min(s.qpos + r / p.group, static_cast<long long>(s.kv_end) - 1);
              lim[nt][e] = r < s.rows ? static_cast<int>(max(last, -1ll)) : -1;
            }
          tile_step<NT, true>(at, qf, qs, A, p.scale_log2, lim, tok, !(bad & 1u), !(bad & 2u));
        } else {
          const int lim[NT][2] = {};
          tile_step<NT, false>(at, qf, qs, A, p.scale_log2, lim, tok, true, true);
        }
        __syncwarp();
        if (issued < mine) issue(issued++);
      }
    }

    // ---- the warps' parts of the segment meet in shared memory ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = A.l[nt][e], pm[4];
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) pm[grp] = A.pm[nt][grp][e];
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) {
          l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
          for (int grp = 0; grp < 4; ++grp) pm[grp] += __shfl_xor_sync(0xffffffffu, pm[grp], o);
        }
        const int row = nt * 8 + 2 * t + e;
        if (g == 0) ml[warp * C::kRows + row] = make_float2(A.m[nt][e], l);
        if (any && row < live) {
#pragma unroll
          for (int grp = 0; grp < 4; ++grp) {
            const float add = pm[grp] - kShift * A.ps[nt][grp >> 1][(grp & 1) * 2 + e];
            const float4 v = make_float4(A.o[nt][grp][0][e] + add, A.o[nt][grp][0][2 + e] + add,
                                         A.o[nt][grp][1][e] + add, A.o[nt][grp][1][2 + e] + add);
            // float4 number 8 grp + g of the row, its place xored with the row pair: no bank conflict
            const int c4 = (8 * grp + g) ^ (2 * t);
            *reinterpret_cast<float4*>(red + (warp * C::kRows + row) * kHD + c4 * 4) = v;
          }
        }
      }
    }
    if (!ok && lane == 0) *failed = 1;
    __syncthreads();
    const bool whole = x <= u0 && seg_end == u1;
    const int part = 2 * blockIdx.x + (x == x0 ? 0 : 1);
    if (!*failed)
      for (int i = tid; i < live * (kHD / 4); i += kThreads) {
        const int row = i / (kHD / 4), c4 = i % (kHD / 4);
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w * C::kRows + row].x);
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 v = ml[w * C::kRows + row];
          if (v.y == 0.f) continue;  // nothing of this warp (a NaN goes on)
          const float f = ex2(v.x - M);
          L += f * v.y;
          const float4 u = *reinterpret_cast<const float4*>(
              red + (w * C::kRows + row) * kHD + (c4 ^ (row & 6)) * 4);
          o.x += f * u.x;
          o.y += f * u.y;
          o.z += f * u.z;
          o.w += f * u.w;
        }
        if (whole) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          write_row4(p, b, kvh, r0 + row, c4 * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
        } else {
          *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(part) * C::kRows + row) * kHD + c4 * 4) = o;
          if (c4 == 0) p.part_ml[part * C::kRows + row] = make_float2(M, L);
        }
      }
    x = seg_end;
    if (x < x1) __syncthreads();  // the next segment overwrites red and ml
  }
  // After a failed wait the copies still in flight must land before the shared memory goes.
  if (!ok)
    for (; stuck < issued; ++stuck) mbar_wait(&bar[stuck % kDepth], (stuck / kDepth) & 1, nullptr);
}

// The rows whose tiles were divided between CTAs: one CTA per output row, whose warps take the parts
// in turn. Rows that see no key are zeroed here too. Bound by its latency.
constexpr int kMergeWarps = 4;
template <int NT>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const Params p) {
  using C = Cfg<NT>;
  __shared__ float4 so[kMergeWarps][32];
  __shared__ float2 sm[kMergeWarps];
  pdl_launch_dependents();
  if (!p.stable_prefix) pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = blockIdx.x;
  const int h = R % p.nh, i = (R / p.nh) % p.q_len, b = R / (p.nh * p.q_len);
  int base = 0;
  const int total = list_total<NT>(p, b, &base);
  const Seq s = load_seq<NT>(p, b);
  if (p.stable_prefix) pdl_wait();
  const int kvh = h / p.group, r = i * p.group + h - kvh * p.group;
  if (r >= s.rows) return;
  if (s.tiles == 0) {
    if (warp == 0) write_row4(p, b, kvh, r, lane * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int n = active_ctas(total, p.ctas);
  const int u0 = base + (kvh * s.rb + r / C::kRows) * s.tiles;
  const int c0 = cta_of(total, n, u0), c1 = cta_of(total, n, u0 + s.tiles - 1);
  if (c0 == c1) return;  // written whole
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = c0 + warp; c <= c1; c += kMergeWarps) {
    const int part = 2 * c + (first_tile(total, n, c) >= u0 ? 0 : 1);
    const int64_t row = static_cast<int64_t>(part) * C::kRows + r % C::kRows;
    const float2 v = p.part_ml[row];
    const float4 u = *reinterpret_cast<const float4*>(p.part_o + row * kHD + lane * 4);
    if (v.y == 0.f) continue;  // the part sees no key of the row (a NaN goes on)
    const float m = fmaxf(M, v.x), f0 = L == 0.f ? 0.f : ex2(M - m), f1 = ex2(v.x - m);
    M = m;
    L = L * f0 + v.y * f1;
    o = make_float4(o.x * f0 + u.x * f1, o.y * f0 + u.y * f1, o.z * f0 + u.z * f1, o.w * f0 + u.w * f1);
  }
  so[warp][lane] = o;
  if (lane == 0) sm[warp] = make_float2(M, L);
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) M = fmaxf(M, sm[w].x);
  L = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) {
    if (sm[w].y == 0.f) continue;
    const float f = ex2(sm[w].x - M);
    const float4 u = so[w][lane];
    L += f * sm[w].y;
    o = make_float4(o.x + f * u.x, o.y + f * u.y, o.z + f * u.z, o.w + f * u.w);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  write_row4(p, b, kvh, r, lane * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

struct Plan {
  int nt = 1, ctas = 1, rb = 1;
  bool direct = false;
  size_t o_bytes = 0, ws_bytes = 0;
};

int make_plan(const SolortInt4DecodeArgs* a, Plan* pl) {
  if (!a) return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->head_dim != kHD) return SOLORT_ERR_UNSUPPORTED;
  if (a->batch <= 0 || a->q_len <= 0 || a->num_qo_heads <= 0 || a->num_kv_heads <= 0 ||
      a->max_kv_len <= 0 || a->num_ctas < 0)
    return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->num_qo_heads % a->num_kv_heads != 0) return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->batch > 65535) return SOLORT_ERR_UNSUPPORTED;
  // One n8 tile of rows where the rows fit it (two CTAs per SM), else blocks of 16 rows.
  const int64_t rows = static_cast<int64_t>(a->q_len) * (a->num_qo_heads / a->num_kv_heads);
  pl->nt = rows <= 8 ? 1 : 2;
  const int64_t rb = (rows + 8 * pl->nt - 1) / (8 * pl->nt);
  const int64_t tiles = (static_cast<int64_t>(a->max_kv_len) + kTile - 1) / kTile;
  const int64_t units = rb * a->num_kv_heads;
  const int64_t out_rows = static_cast<int64_t>(a->batch) * a->q_len * a->num_qo_heads;
  const int64_t limit = (1ll << 31) - 1;
  if (rows > limit || units > limit || out_rows > limit || tiles > limit / units ||
      tiles * units > limit / a->batch)
    return SOLORT_ERR_UNSUPPORTED;
  DeviceInfo di;
  int rc = current_device_info(&di);
  if (rc != SOLORT_OK) return rc;
  pl->rb = static_cast<int>(rb);
  pl->direct = tiles <= kDirectTiles && a->num_ctas == 0;
  if (pl->direct) return SOLORT_OK;
  const int64_t most = (tiles * units * a->batch + kMinTiles - 1) / kMinTiles;
  const int64_t wave = a->num_ctas > 0 ? a->num_ctas
                                       : static_cast<int64_t>(di.sm_count) *
                                             (pl->nt == 1 ? Cfg<1>::kCtasPerSm : Cfg<2>::kCtasPerSm);
  if (wave > (1 << 20)) return SOLORT_ERR_UNSUPPORTED;
  pl->ctas = static_cast<int>(most < wave ? most : wave);
  const size_t parts = static_cast<size_t>(2) * pl->ctas * 8 * pl->nt;
  pl->o_bytes = parts * kHD * 4;
  pl->ws_bytes = align_up(pl->o_bytes + parts * 8, 256);
  return SOLORT_OK;
}

inline cudaLaunchConfig_t pdl_config(dim3 grid, int threads, size_t smem, void* stream,
                                     cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

template <int NT>
int launch(const Params& prm, const Plan& pl, void* stream) {
  using C = Cfg<NT>;
  static std::atomic<unsigned> configured{0};  // one bit per device ordinal < 32
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SOLORT_ERR_CUDA;
  if (dev >= 32 || !(configured.load(std::memory_order_acquire) & (1u << dev))) {
    if (cudaFuncSetAttribute(decode_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
            cudaSuccess ||
        cudaFuncSetAttribute(decode_kernel<NT>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared) != cudaSuccess)
      return SOLORT_ERR_CUDA;
    if (dev < 32) configured.fetch_or(1u << dev, std::memory_order_release);
  }
  cudaLaunchAttribute attr[1];
  const dim3 grid = pl.direct ? dim3(prm.nkv * pl.rb, prm.batch) : dim3(pl.ctas);
  cudaLaunchConfig_t cfg = pdl_config(grid, kThreads, C::kSmem, stream, attr);
  if (cudaLaunchKernelEx(&cfg, decode_kernel<NT>, prm) != cudaSuccess) return SOLORT_ERR_CUDA;
  int rc = launch_status();
  if (rc != SOLORT_OK || pl.direct) return rc;
  cfg = pdl_config(dim3(prm.batch * prm.q_len * prm.nh), kMergeWarps * 32, 0, stream, attr);
  if (cudaLaunchKernelEx(&cfg, merge_kernel<NT>, prm) != cudaSuccess) return SOLORT_ERR_CUDA;
  return launch_status();
}

}  // namespace i4

int read_int4_decode_status(unsigned* flags) {
  unsigned v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_int4_decode_status, sizeof(v)) != cudaSuccess)
    return SOLORT_ERR_CUDA;
  if (v && cudaMemcpyToSymbol(g_int4_decode_status, &zero, sizeof(zero)) != cudaSuccess)
    return SOLORT_ERR_CUDA;
  *flags |= v;
  return SOLORT_OK;
}

}  // namespace solort

using namespace solort;

extern "C" int solort_attn_decode_int4_workspace_size(const SolortInt4DecodeArgs* a, size_t* bytes) {
  if (!bytes) return SOLORT_ERR_INVALID_ARGUMENT;
  i4::Plan pl;
  int rc = i4::make_plan(a, &pl);
  if (rc != SOLORT_OK) return rc;
  *bytes = pl.ws_bytes;
  return SOLORT_OK;
}

extern "C" int solort_attn_decode_int4(const SolortInt4DecodeArgs* a, void* stream) {
  if (!a) return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->head_dim != i4::kHD) return SOLORT_ERR_UNSUPPORTED;
  if (!a->q || !a->out || !a->kv_pages || !a->block_table || !a->q_pos)
    return SOLORT_ERR_INVALID_ARGUMENT;
  const int P = a->page_size;
  if (P < i4::kBlockTokens || (P & (P - 1)) != 0 || a->num_pages <= 0 || a->block_table_stride < 0)
    return SOLORT_ERR_INVALID_ARGUMENT;
  if (!aligned(a->q, 16) || ((a->q_stride_batch | a->q_stride_token | a->q_stride_head) & 7) ||
      !aligned(a->out, 8) || ((a->out_stride_batch | a->out_stride_token | a->out_stride_head) & 3) ||
      !aligned(a->kv_pages, 16) || ((a->kv_stride_page | a->kv_stride_head) & 15) ||
      a->kv_stride_page < 0 || a->kv_stride_head < 0 || !aligned(a->block_table, 4) ||
      !aligned(a->q_pos, 8) || !aligned(a->q_lens, 4))
    return SOLORT_ERR_INVALID_ARGUMENT;
  i4::Plan pl;
  int rc = i4::make_plan(a, &pl);
  if (rc != SOLORT_OK) return rc;
  if (pl.ws_bytes > 0 &&
      (!a->workspace || a->workspace_bytes < pl.ws_bytes || !aligned(a->workspace, 256)))
    return SOLORT_ERR_WORKSPACE;
  i4::Params p{};
  p.q = static_cast<const bf16*>(a->q);
  p.q_sb = a->q_stride_batch;
  p.q_st = a->q_stride_token;
  p.q_sh = a->q_stride_head;
  p.out = static_cast<bf16*>(a->out);
  p.o_sb = a->out_stride_batch;
  p.o_st = a->out_stride_token;
  p.o_sh = a->out_stride_head;
  p.pages = static_cast<const uint8_t*>(a->kv_pages);
  p.page_stride = a->kv_stride_page;
  p.head_stride = a->kv_stride_head;
  p.block_table = a->block_table;
  p.bt_stride = a->block_table_stride;
  p.page_size = P;
  while ((1 << p.page_shift) < P) ++p.page_shift;
  p.num_pages = a->num_pages;
  p.q_pos = a->q_pos;
  p.q_lens = a->q_lens;
  if (!pl.direct) {
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(a->workspace) + pl.o_bytes);
  }
  p.batch = a->batch;
  p.q_len = a->q_len;
  p.nh = a->num_qo_heads;
  p.nkv = a->num_kv_heads;
  p.group = a->num_qo_heads / a->num_kv_heads;
  p.max_kv_len = a->max_kv_len;
  p.direct = pl.direct ? 1 : 0;
  p.ctas = pl.ctas;
  p.stable_prefix = (a->flags & SOLORT_DECODE_STABLE_PREFIX) ? 1 : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  return pl.nt == 1 ? i4::launch<1>(p, pl, stream) : i4::launch<2>(p, pl, stream);
}
