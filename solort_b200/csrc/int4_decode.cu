// GQA decode / verify attention over the paged 4-bit KV cache (layout and formula: int4.cuh).
//
// With keys held as k = mid + scale (c - 7.5) and values likewise, per group g of 32 dims,
//   q . k       = sum_g scale_g sum_d q_d c_d + (mid_g - 7.5 scale_g) sum_d q_d
//   sum_t p v_d = sum_t (p scale_g) c_d + sum_t p (mid_g - 7.5 scale_g)
// so the tensor cores multiply the codes themselves and the scales are applied to their fp32 results
// (keys) or to the probabilities (values): the cache is never expanded.
//
// Keys: a nibble in a byte IS an e4m3 number. Bytes 0..15 are the subnormals and the first binade, the
// values c 2^-9 exactly, so eight codes become operands with a shift and two ands, and an e4m3 product
// takes a quarter of a bf16 one's time per multiply-add (measured: m16n8k32 e4m3 4.6 cycles a scheduler,
// m16n8k16 bf16 8.8). The query is split in two e4m3 numbers, hi and lo, four significant bits each, lo
// times 16; they are the two columns of one query row. A query row is scaled by a power of two to a
// maximum in [128, 256): hi + lo / 16 is then its bf16 values exactly down to 2^-13 of the row's maximum,
// and within 2^-22 of that maximum below. The mids' and -7.5 scales' share is one bf16 product more, of
// the held scales and mids with the query's group sums (themselves split in two bf16 numbers).
//
// Values: a nibble in a half is an f16 subnormal, c 2^-24 or 16 c 2^-24, which costs a shift and ands
// too and lets the other operand keep 11 bits: x = p scale sf, with p relative to the row's running maximum
// (at most 2^7 until that is raised) and sf a power of two for each row and group. sf follows the largest
// p scale as the maximum follows the scores, up and down: a token of large values and no weight takes no bits
// from the others. x is within 2^-11 of itself, and within 2^-25 below 2^-14, where the row's largest in the
// group is 2^5 at least. The codes are centred with the sum of the same numbers (a product with ones),
// O = sum x c - 7.5 sum x + sum p mid, so that their rounding weighs |v - mid| and not c. Tokens of a tile's
// second and fourth blocks enter as -x times 15 - c, which centres to the same x (c - 7.5): the tensor cores cut
// products off at a distance from the nominal exponent of the largest, and a subnormal's nominal exponent lies
// 6 to 10 bits above a nibble in the lowest bits, 2 to 6 above one in the next. With one sign that was a bias
// of 1e-5 of the values in every other dim, 0.05 % of the result at 131072 keys; with both it cancels (0.02 %,
// the f16 rounding), and the sums stay small. p, its sum, sum p mid and all accumulators are fp32.
//
// Both products are transposed, S^T = K Q^T and O^T = V^T P^T (tokens or dims as the 16 rows), so that
// four query rows fill an n8 tile of the first and a row pair a column pair of the second; P^T turns into
// its operand with movmatrix.
//
// Work split: the cache's 32-token tiles, over all sequences, KV heads and blocks of query rows, are one
// list, divided evenly over all warps of the GPU, so that sequences of any lengths load every SM alike. A
// unit (a sequence's KV head and row block) counts kUnitCost tiles more for its set-up: 48 sequences of
// 127 to 8111 keys take 35.5 us with 2, 35.4 with 4, 36.6 with 8. A warp has a ring of kDepth tiles of its
// own (5120 bytes a tile, in 16-byte asynchronous copies), so warps meet only when a unit that they share
// ends. A unit that lies within a CTA is added up there; parts of several CTAs meet in merge_kernel,
// through `span`. Lengths are read on the device. Short caches skip the division: a unit is a CTA, or a
// cluster of CTAs that add up their sums over shared memory (make_plan).
//
// Bound by memory for up to four rows: 32 query heads over 8 KV heads, 131072 keys 38.8 us (4.3 TB/s; 5.6
// TB/s for each key beyond 16384, of 6.57 measured for a copy). The rest is what every call pays, 6.5 us
// at 1000 keys: the way of the query rows into operands, a first tile that nothing hides, the sums of the
// parts and the cluster's barriers, or the merge's launch. Blocks of eight rows are bound by the
// instructions of a tile, 810 a warp (605 for four rows), 60 of them on the matrix pipe: 8 sequences of 5
// rows, 4099 keys 27.5 us. Probabilities are ex2.approx's, within 2^-22 of themselves.
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

constexpr int kTile = 32;                     // tokens of a tile: four blocks
constexpr int kTileBytes = 4 * kBlockBytes;   // 5120
constexpr int kUnitCost = 4;                  // tiles' worth of set-up of a unit
constexpr int kDirectSteps = 6;               // the most tiles a warp takes where the list is not divided
constexpr int kSplitSteps = 2;                // what the division and its merge cost more, in tiles
constexpr int kMostCluster = 8;               // CTAs of a cluster, the portable limit
constexpr int kApartTiles = 128;              // tiles of a warp from which eight rows' sums of a tile stay apart
constexpr int kMostKeys = 1 << 30;            // keys of a sequence
constexpr int kBareTiles = 16;                // up to this many tiles a unit may go without a workspace
// A row's running maximum is raised only when a score passes it by 2^kLazy, and its power of two for a group
// is set anew only when an x of a tile could pass 2^15, inside f16: it then brings the row's largest p scale
// into [2^kXBits, 2^(kXBits + 1)).
constexpr float kLazy = 7.f;
constexpr int kXBits = 6;
constexpr float kMostX = 32768.f;
constexpr int kMostSf = 127 + 119;         // exponent field of the greatest power of two: p sf stays finite
constexpr float kCodeUnit = 512.f;         // a key code's e4m3 value is c / 512
constexpr float kValueUnit = 16777216.f;   // a value code's f16 value is c 2^-24, or 16 c 2^-24

// NT n8 tiles of four query rows each; two CTAs of six warps share an SM, 168 registers a thread. A third
// tile in the ring, which fits for four rows, takes longer (131072 keys 40.2 us, 38.8 without). Eight rows
// spill a little (192 bytes of stores and 80 of loads a thread, 220 and 108 with kApart), and on 8 sequences
// of 5 rows, 4099 keys, eight warps of 255 registers without spills are no faster; ten warps load the four
// schedulers unevenly (14 % slower); sixteen rows in one warp want 255 registers and spill (24 % slower).
template <int NT>
struct Cfg {
  static constexpr int kWarps = 6;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtasPerSm = 2;
  static constexpr int kDepth = 2;  // tiles of a warp in shared memory
  static constexpr int kRows = 4 * NT;
  static constexpr int kRing = kWarps * kDepth * kTileBytes;
  static constexpr int kRed = kWarps * kRows * kHD * 4;
  static_assert(kRows * kHD * 4 <= kDepth * kTileBytes, "a part fits a ring");
  static constexpr int kOffRed = kRing;
  static constexpr int kOffMl = kOffRed + kRed;
  static constexpr int kOffEdge = kOffMl + 2 * kWarps * kRows * 8;
  static constexpr int kOffRange = kOffEdge + 2 * kWarps * 24;
  static constexpr int kOffPlaces = (kOffRange + (kWarps + 1) * 12 + 15) / 16 * 16;  // [warp][32 tiles][4]
  static constexpr int kOffUnit = kOffPlaces + kWarps * 32 * 32;  // a CTA's sums for its cluster: [row][128]
  static constexpr int kOffUnitMl = kOffUnit + kRows * kHD * 4;   // and [row]
  static constexpr int kSmem = kOffUnitMl + kRows * 8;
};
static_assert(Cfg<1>::kSmem <= 115712 && Cfg<2>::kSmem <= 115712, "two CTAs per SM");

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
  float2* part_ml;  // [2 * ctas][rows] reference (log2 domain) and sum
  int2* span;       // [batch][nkv][row block] its first part, and the CTA of its last
  int rb;           // row blocks of q_len tokens
  int batch, q_len, nh, nkv, group, max_kv_len;
  uint32_t group_mul;  // n / group = umulhi(n, group_mul) >> group_shift for 0 <= n < 2^31, group > 1
  int group_shift;
  int direct;   // grid (head and row block, sequence): no parts
  int cluster;  // then the CTAs of a unit, a cluster
  int ctas;
  int stable_prefix;
  float scale_log2;
};

__device__ __forceinline__ int by_group(const Params& p, int n) {
  return p.group == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), p.group_mul) >> p.group_shift);
}

struct Seq {  // one sequence's share of the list
  long long qpos;
  int kv_end, rows, rb, tiles;
  __device__ __forceinline__ int units(int nkv) const { return nkv * rb; }
  __device__ __forceinline__ int total(int nkv) const { return nkv * rb * tiles; }
  __device__ __forceinline__ int cost(int nkv) const { return tiles ? nkv * rb * (tiles + kUnitCost) : 0; }
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

// Prefix sums over the sequences, 32 at a time: lane i has sequence first + i.
struct Prefix {
  int cost, tiles, unit_tiles;  // of this lane's sequence: in all, and of one unit
  int cost_incl, tiles_incl;    // sums from `first` on
  int cost_run, tiles_run;      // before `first`
};
template <int NT>
__device__ __forceinline__ void load_prefix(const Params& p, Prefix& f, int first) {
  const int lane = threadIdx.x & 31;
  f.cost_run = first ? f.cost_run + __shfl_sync(0xffffffffu, f.cost_incl, 31) : 0;
  f.tiles_run = first ? f.tiles_run + __shfl_sync(0xffffffffu, f.tiles_incl, 31) : 0;
  f.cost = f.tiles = f.unit_tiles = 0;
  if (first + lane < p.batch) {
    const Seq s = load_seq<NT>(p, first + lane);
    f.cost = s.cost(p.nkv);
    f.tiles = s.total(p.nkv);
    f.unit_tiles = s.tiles;
  }
  f.cost_incl = f.cost;
  f.tiles_incl = f.tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, f.cost_incl, o), v = __shfl_up_sync(0xffffffffu, f.tiles_incl, o);
    if (lane >= o) f.cost_incl += u, f.tiles_incl += v;
  }
}

// CTAs at work on a list of that cost, and its division between workers: the first cost % n of n have
// one position more than the others.
struct Division {
  int n, each, more;
  __device__ __forceinline__ Division(int cost, int ctas, int warps) {
    n = max(1, min(ctas, (cost + warps - 1) / warps)) * warps;
    each = cost / n;
    more = cost - each * n;
  }
  __device__ __forceinline__ int first(int w) const { return w * each + min(w, more); }
};

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// Shared memory of the cluster's CTA `rank`, at this CTA's address `addr`.
__device__ __forceinline__ uint32_t in_cluster(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 cluster_lds128(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 cluster_lds64(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
constexpr uint32_t kNibbles = 0x0f0f0f0fu;
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
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {  // all but the last N groups of this thread have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// d = a b + c, m16n8k32 e4m3.
__device__ __forceinline__ void mma_e4m3(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         float c0, float c1, float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// d = a b, and d += a b, m16n8k16 f16.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void add4(float (&d)[4], const float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float2 r = both(add2(pair(d[i], d[i + 1]), pair(v[i], v[i + 1])));
    d[i] = r.x, d[i + 1] = r.y;
  }
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// One warp's state over a segment. This lane's query row of n8 tile nt is row 4 nt + lane % 4.
template <int NT>
struct Acc {
  static constexpr int kCols = NT > 1 ? NT / 2 : 1;  // n8 tiles of the second product
  // [tile][group][m16 tile h]: c0, c1 dim 32 g + 4 (lane / 4) + 2 h, c2, c3 the dim after. The columns
  // are two rows (nt = 2 tile, 2 tile + 1), or with one row a lane that row for the two groups of a
  // pair, of which the group's own is kept.
  static constexpr int kKept = NT > 1 ? 4 : 2;
  float o[kCols][4][2][kKept];
  // Sums of +-x: [tile][group pair], columns of the even group in c0, c1 and of the odd in c2, c3; with
  // one row a lane [0][0], of the pair 0 and 1.
  float xs[kCols][NT > 1 ? 2 : 1][4];
  f2 pm[NT][2];   // this lane's tokens' sum of p mid, a group pair each
  float l[NT];    // and of p
  float off[NT];  // p = 2^(score - off)
  float top[NT];  // scores above it raise the maximum
  f2 sf[NT][2];   // per row and group pair
};

// One tile of 32 tokens for the segment's rows; this lane's tokens are tok0 + 8 i + lane / 4 of block
// i. `masked`: some row does not see some token; `there` has a bit for each block that was loaded.
template <int NT, bool kApart>
__device__ __forceinline__ void tile_step(uint32_t base, const uint32_t (&qf)[NT][4][2],
                                          const uint32_t (&qm)[NT][2], Acc<NT>& A, const float (&fr)[NT],
                                          bool masked, const int (&lim)[NT], int tok0, unsigned there) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float s[NT][4];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
    const uint32_t b0 = base + 2 * mt * kBlockBytes, b1 = b0 + kBlockBytes;
    const uint4 k0 = lds128(b0 + 64 * g + 16 * t), k1 = lds128(b1 + 64 * g + 16 * t);
    const uint4 m0 = lds128(b0 + kOffKScale + 16 * g), m1 = lds128(b1 + kOffKScale + 16 * g);
    f2 acc[NT];
    {
      // sum_g (mid_g - 7.5 scale_g) sum_d q_d, a product itself: k = mids, mids, scales, scales of the four
      // groups against the sums of q, their low parts, and both times -7.5.
      const uint32_t at = kOffKScale + 16 * g + 8 * (t & 1);
      const uint2 n0 = lds64(b0 + at), n1 = lds64(b1 + at);
      const uint32_t a[4] = {__byte_perm(n0.x, n0.y, 0x7632), __byte_perm(n1.x, n1.y, 0x7632),
                             __byte_perm(n0.x, n0.y, 0x5410), __byte_perm(n1.x, n1.y, 0x5410)};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        mma_bf16_16816(c, a, qm[nt][0], qm[nt][1]);
        acc[nt] = pair(c[0], c[2]);
      }
    }
#pragma unroll
    for (int grp = 0; grp < 4; ++grp) {
      const uint32_t w0 = word(k0, grp), w1 = word(k1, grp);
      const uint32_t a[4] = {w0 & kNibbles, w1 & kNibbles, (w0 >> 4) & kNibbles, (w1 >> 4) & kNibbles};
      const f2 sc = pair(lo_bf16(word(m0, grp)), lo_bf16(word(m1, grp)));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c[4];
        mma_e4m3(c, a, qf[nt][grp][0], qf[nt][grp][1], 0.f, 0.f, 0.f, 0.f);
        acc[nt] = fma2(sc, pair(fmaf(c[1], 0.0625f, c[0]), fmaf(c[3], 0.0625f, c[2])), acc[nt]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 x = both(mul2(acc[nt], dup(fr[nt])));
      s[nt][2 * mt] = x.x, s[nt][2 * mt + 1] = x.y;
    }
  }
  uint4 meta[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) meta[i] = lds128(base + i * kBlockBytes + kOffVScale + 16 * g);
  if (__builtin_expect(masked, 0)) {
    // A token that a row does not see adds nothing, whatever its scale and mid are: they count as 0
    // where no row of the lane sees it, and where some do, a NaN goes into those rows' scores.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bool any = false, all = true;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bool vis = (there >> i & 1u) && tok0 + 8 * i + g <= lim[nt];
        if (!vis) s[nt][i] = -INFINITY;
        any |= vis;
        all &= vis;
      }
      bool drop = !any;
      if (NT > 1 && any && !all) {
#pragma unroll
        for (int grp = 0; grp < 4; ++grp)
          drop |= isnan(lo_bf16(word(meta[i], grp))) || isnan(hi_bf16(word(meta[i], grp)));
        if (drop)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (tok0 + 8 * i + g <= lim[nt]) s[nt][i] = NAN;
      }
      if (drop) meta[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  bool raise = false;
  {
    f2 wide[2];  // the largest scales of this lane's tokens (not negative: as integers; with a NaN the group is NaN)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w = __vmaxu2(w, __byte_perm(word(meta[i], 2 * q), word(meta[i], 2 * q + 1), 0x5410));
      wide[q] = pair(lo_bf16(w), hi_bf16(w));
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mx = fmaxf(fmaxf(s[nt][0], s[nt][1]), fmaxf(s[nt][2], s[nt][3]));
      const float2 a = both(mul2(wide[0], A.sf[nt][0])), c = both(mul2(wide[1], A.sf[nt][1]));
      const float most = fmaxf(fmaxf(a.x, a.y), fmaxf(c.x, c.y)) * ex2(mx - A.off[nt]);
      raise |= mx > A.top[nt] || !(most <= kMostX);
    }
  }
  if (__builtin_expect(__any_sync(0xffffffffu, raise), 0)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = nt / 2, e = nt & 1;
      float mx = fmaxf(fmaxf(s[nt][0], s[nt][1]), fmaxf(s[nt][2], s[nt][3]));
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      int up = 0;  // what is summed up has lost so many bits of weight
      if (mx > A.top[nt]) {
        const bool first = A.top[nt] == -INFINITY;
        const float f = first ? 0.f : ex2(A.off[nt] - mx);
        up = first ? 255 : static_cast<int>(fminf(mx - A.off[nt], 255.f));
        A.off[nt] = mx;
        A.top[nt] = mx + kLazy;
        A.l[nt] *= f;
        A.pm[nt][0] = mul2(A.pm[nt][0], dup(f));
        A.pm[nt][1] = mul2(A.pm[nt][1], dup(f));
#pragma unroll
        for (int grp = 0; grp < 4; ++grp)
#pragma unroll
          for (int i = 0; i < Acc<NT>::kKept; ++i)
            if (NT == 1 || (i & 1) == e) A.o[c][grp][0][i] *= f, A.o[c][grp][1][i] *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (NT == 1)
            A.xs[0][0][i] *= f;
          else if ((i & 1) == e)
            A.xs[c][0][i] *= f, A.xs[c][NT > 1][i] *= f;
      }
      // The exponents of the groups' largest p scale, a byte each; a NaN does not count, it makes the sums of
      // the rows that see it NaN by itself.
      uint32_t top = 0;
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
        float w = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) w = fmaxf(w, ex2(s[nt][i] - A.off[nt]) * lo_bf16(word(meta[i], grp)));
        top |= (__float_as_uint(w) >> 23) << (8 * grp);
      }
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) top = __vmaxu4(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float2 was = both(A.sf[nt][q]);
        float sf[2];
#pragma unroll
        for (int g2 = 0; g2 < 2; ++g2) {
          const int grp = 2 * q + g2, old = static_cast<int>(__float_as_uint(g2 ? was.y : was.x) >> 23);
          const int now = min(min(old + up, kMostSf), 254 + kXBits - static_cast<int>(top >> (8 * grp) & 255u));
          sf[g2] = __uint_as_float(static_cast<uint32_t>(now) << 23);
          const int by = min(127 + now - old, 254);
          const float f = by < 1 ? 0.f : __uint_as_float(static_cast<uint32_t>(by) << 23);  // sf / old
#pragma unroll
          for (int i = 0; i < Acc<NT>::kKept; ++i)
            if (NT == 1 || (i & 1) == e) A.o[c][grp][0][i] *= f, A.o[c][grp][1][i] *= f;
          if (NT > 1)
            A.xs[c][q & (NT > 1)][2 * g2 + e] *= f;
          else
            A.xs[0][0][grp] *= f;
        }
        A.sf[nt][q] = pair(sf[0], sf[1]);
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[nt][i] = ex2(s[nt][i] - A.off[nt]);
      A.l[nt] += s[nt][i];
    }

  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = lds128(base + i * kBlockBytes + kOffV + 128 * t + 16 * (g ^ (2 * t)));
  constexpr uint32_t kOnes = 0x3c003c00u, kLow = 0x000f000fu, kHigh = 0x00f000f0u;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    f2 x[NT][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f2 mid = pair(hi_bf16(word(meta[i], 2 * q)), hi_bf16(word(meta[i], 2 * q + 1)));
      const f2 scale = pair(lo_bf16(word(meta[i], 2 * q)), lo_bf16(word(meta[i], 2 * q + 1)));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        x[nt][i] = mul2(mul2(dup(i & 1 ? -s[nt][i] : s[nt][i]), A.sf[nt][q]), scale);
        A.pm[nt][q] = fma2(dup(s[nt][i]), mid, A.pm[nt][q]);
      }
    }
    uint32_t bb[2][Acc<NT>::kCols][4];  // [group of the pair][tile][block]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (NT == 1) {
        const float2 x0 = both(x[0][i]);
        bb[0][0][i] = bb[1][0][i] = transpose8x8(pack_f16x2(x0.x, x0.y));
      } else {
#pragma unroll
        for (int c = 0; c < Acc<NT>::kCols; ++c) {
          const float2 x0 = both(x[2 * c][i]), x1 = both(x[2 * c + (NT > 1)][i]);
          bb[0][c][i] = transpose8x8(pack_f16x2(x0.x, x1.x));
          bb[1][c][i] = transpose8x8(pack_f16x2(x0.y, x1.y));
        }
      }
    }
    // Sums of +-x and of their products with c or 15 - c over the tile: into the running ones, or apart and then
    // added to them.
    float sum[2][Acc<NT>::kCols][2][4], ones_sum[Acc<NT>::kCols][4];
    auto product = [&](float(&part)[4], auto& all, const uint32_t(&a4)[4], uint32_t b0, uint32_t b1, bool first) {
      if constexpr (!kApart)
        mma_f16(all, a4, b0, b1);
      else if (first)
        mma_f16_first(part, a4, b0, b1);
      else
        mma_f16(part, a4, b0, b1);
    };
#pragma unroll
    for (int c = 0; c < Acc<NT>::kCols; ++c)
#pragma unroll
      for (int e = 0; e < (NT > 1 ? 2 : 1); ++e) {
        // rows 0..7 of ones add up the first of two groups, or pairs, and rows 8..15 the second
        const bool second = NT > 1 ? e : q;
        const uint32_t lo_rows = second ? 0u : kOnes, hi_rows = second ? kOnes : 0u;
        const uint32_t ones[4] = {lo_rows, hi_rows, lo_rows, hi_rows};
#pragma unroll
        for (int k = 0; k < 4; k += 2)
          product(ones_sum[c], A.xs[c][q & (NT > 1)], ones, bb[e][c][k], bb[e][c][k + 1], e + k == 0);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int grp = 2 * q + e;
#pragma unroll
      for (int k = 0; k < 4; k += 2) {  // tokens of blocks k, k + 1
        const uint32_t w0 = word(v[k], grp), w1 = word(v[k + 1], grp), y0 = w0 >> 8, y1 = w1 >> 8;
        const uint32_t a0[4] = {w0 & kLow, w0 & kHigh, ~w1 & kLow, ~w1 & kHigh};
        const uint32_t a1[4] = {y0 & kLow, y0 & kHigh, ~y1 & kLow, ~y1 & kHigh};
#pragma unroll
        for (int c = 0; c < Acc<NT>::kCols; ++c) {
          product(sum[e][c][0], A.o[c][grp][0], a0, bb[e][c][k], bb[e][c][k + 1], k == 0);
          product(sum[e][c][1], A.o[c][grp][1], a1, bb[e][c][k], bb[e][c][k + 1], k == 0);
        }
      }
    }
    if constexpr (kApart) {
#pragma unroll
      for (int c = 0; c < Acc<NT>::kCols; ++c) {
        add4(A.xs[c][q & (NT > 1)], ones_sum[c]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float(&o)[Acc<NT>::kKept] = A.o[c][2 * q + e][h];
            if constexpr (NT > 1)
              add4(o, sum[e][c][h]);
            else
              o[0] += sum[e][c][h][e], o[1] += sum[e][c][h][2 + e];
          }
      }
    }
  }
}

__device__ __forceinline__ void write_row4(const Params& p, int b, int kvh, int r, int c, float4 v) {
  const int i = by_group(p, r), h = kvh * p.group + r - i * p.group;
  uint2 pk;
  pk.x = pack_bf16x2(v.x, v.y);
  pk.y = pack_bf16x2(v.z, v.w);
  *reinterpret_cast<uint2*>(p.out + b * p.o_sb + i * p.o_st + h * p.o_sh + c) = pk;
}

// This lane's chunk of its row of n8 tile nt: dims 32 grp + 4 (lane / 4) .. + 3.
template <int NT>
__device__ __forceinline__ float4 chunk_of(const Acc<NT>& A, int nt, int grp, float pm) {
  const float2 sf = both(A.sf[nt][grp >> 1]);
  // 1 / sf, a power of two
  const float inv = __uint_as_float((254u << 23) - __float_as_uint(grp & 1 ? sf.y : sf.x));
  const int c = nt / 2, e = NT > 1 ? nt & 1 : grp & 1;
  const float sum = NT > 1 ? A.xs[c][(grp >> 1) & (NT > 1)][(grp & 1) * 2 + e] : A.xs[0][0][grp];
  // sum x (c - 7.5) first: 2^24 / sf would pass fp32's range for scales from 2^103 on
  const float centre = -7.5f * sum;
  constexpr int kKept = Acc<NT>::kKept;
  const float(&a0)[kKept] = A.o[c][grp][0];
  const float(&a1)[kKept] = A.o[c][grp][1];
  const int i0 = NT > 1 ? e : 0, i1 = NT > 1 ? 2 + e : 1;
  auto value = [&](float unit, float a) { return fmaf(inv, fmaf(unit, a, centre), pm); };
  return make_float4(value(kValueUnit, a0[i0]), value(kValueUnit * 0.0625f, a0[i1]), value(kValueUnit, a1[i0]),
                     value(kValueUnit * 0.0625f, a1[i1]));
}

// A warp's tiles of the list: from x0 on, the sequence of the first and the tiles before that. Entry
// kWarps is the end of the CTA's.
struct Range {
  int x0, seq, base;
};
// A unit of which a warp holds a part: its tiles [u0, u1) of the list, and where its rows belong.
struct Edge {
  int u0, u1, seq, head, row0, live;
};

// kApart: the tensor cores add up the products of a tile, and the tiles' sums are added here, in fp32 with
// rounding to nearest. A tensor core's own running sum is cut off, for codes always downwards: of 131072 keys
// with 8 KV heads in one CTA's warps (5461 tiles each) that was 1.13 % of the result, and 0.06 % so (0.02 %
// with both signs); at 125 tiles a warp the two are alike. Four rows keep half of the sums and gain registers;
// eight rows pay 9 % of a tile (8 sequences of 5 rows, 4099 keys: 29.0 us, 27.5 without), and have it only
// where a warp's tiles may be more than kApartTiles.
template <int NT, bool kApart>
__global__ void __launch_bounds__(Cfg<NT>::kThreads, Cfg<NT>::kCtasPerSm) decode_kernel(const Params p) {
  using C = Cfg<NT>;
  constexpr int kWarps = C::kWarps, kDepth = C::kDepth;
  extern __shared__ __align__(128) uint8_t smem[];
  // What a warp leaves of a unit that it shares with other warps: its first unit's (begun before the
  // warp's range) in `red`, and its last's (begun in it, going on behind it) where its ring was.
  float2* ml = reinterpret_cast<float2*>(smem + C::kOffMl);   // [2 warp + which][row]
  Edge* edge = reinterpret_cast<Edge*>(smem + C::kOffEdge);   // [2 warp + which]; u0 -1: none
  Range* range = reinterpret_cast<Range*>(smem + C::kOffRange);
  auto part_row = [&](int which, int row) {
    return reinterpret_cast<float*>(smem + (which & 1 ? (which >> 1) * kDepth * kTileBytes
                                                      : C::kOffRed + (which >> 1) * C::kRows * kHD * 4)) + row * kHD;
  };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * kDepth * kTileBytes;
  // Where the blocks of the warp's next tiles are: an address each, with its count of blocks in the
  // low bits. Pages of 16 tokens and more: two of two blocks per tile; of 8: four.
  const uint32_t places = smem_u32(smem) + C::kOffPlaces + warp * 32 * 32;

  if (lane == 0) edge[2 * warp].u0 = edge[2 * warp + 1].u0 = -1;
  float2* unit_ml = reinterpret_cast<float2*>(smem + C::kOffUnitMl);
  if (tid < C::kRows) unit_ml[tid] = make_float2(-INFINITY, 0.f);
  const bool early = p.stable_prefix != 0;
  if (!early) pdl_wait();
  if (warp == 0) {
    Range r = {0, 0, 0};
    if (p.direct) {
      const Seq s = load_seq<NT>(p, blockIdx.y);
      r.seq = blockIdx.y;
      const int unit = blockIdx.x / p.cluster, at = (blockIdx.x - unit * p.cluster) * kWarps + min(lane, kWarps);
      if (unit < s.units(p.nkv)) r.x0 = unit * s.tiles + s.tiles * at / (p.cluster * kWarps);
    } else {
      Prefix f;
      for (int c = 0; c < p.batch; c += 32) load_prefix<NT>(p, f, c);
      const int cost = f.cost_run + __shfl_sync(0xffffffffu, f.cost_incl, 31);
      const Division d(cost, p.ctas, kWarps);
      const int X = d.first(min(static_cast<int>(blockIdx.x) * kWarps + min(lane, kWarps), d.n));
      r.x0 = f.tiles_run + __shfl_sync(0xffffffffu, f.tiles_incl, 31);  // the end of the list
      r.seq = p.batch;
      bool found = false;
      for (int c = 0; c < p.batch; c += 32) {
        if (p.batch > 32) load_prefix<NT>(p, f, c);
        const int y = X - f.cost_run;
        int l = 0;  // the first sequence of the 32 that ends behind X
#pragma unroll
        for (int step = 16; step > 0; step >>= 1)
          if (y >= __shfl_sync(0xffffffffu, f.cost_incl, l + step - 1)) l += step;
        const int end = __shfl_sync(0xffffffffu, f.cost_incl, l);
        const int in_seq = y - end + __shfl_sync(0xffffffffu, f.cost, l);
        const int before = f.tiles_run + __shfl_sync(0xffffffffu, f.tiles_incl - f.tiles, l);
        const int tiles = __shfl_sync(0xffffffffu, f.unit_tiles, l);
        if (!found && y < end) {
          found = true;
          const int unit = in_seq / (tiles + kUnitCost);
          r.seq = c + l;
          r.base = before;
          r.x0 = before + unit * tiles + max(0, in_seq - unit * (tiles + kUnitCost) - kUnitCost);
        }
      }
    }
    if (lane <= kWarps) range[lane] = r;
  }
  __syncthreads();
  const int x0 = range[warp].x0, x1 = range[warp + 1].x0;
  int b = range[warp].seq, base = range[warp].base;

  // ---- the copies ----
  const bool by_block = p.page_size == kBlockTokens;
  int ib = b, ibase = base;  // sequence of this lane's tile of the batch
  unsigned absent = 0;       // tiles of the batch of which a block should be there and is not
  unsigned moving = 0;       // tiles of the batch that a kernel before this one may still be writing
  unsigned gone = 0;         // four bits per ring slot: blocks that should be there and are not
  auto resolve = [&](int first) {  // the places of tiles first .. first + 31, a lane each
    bool lost = false, change = false;
    const int y = first + lane;
    unsigned long long at[4] = {0, 0, 0, 0};
    if (y < x1) {
      Seq is = load_seq<NT>(p, ib);
      while (y >= ibase + is.total(p.nkv)) {
        ibase += is.total(p.nkv);
        is = load_seq<NT>(p, ++ib);
      }
      const int unit = (y - ibase) / is.tiles, head = unit / is.rb;
      const int tok0 = (y - ibase - unit * is.tiles) * kTile;
      const int step = by_block ? kBlockTokens : 2 * kBlockTokens;
      change = tok0 + kTile > is.qpos;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = tok0 + j * step;
        if (tok >= is.kv_end || tok >= tok0 + kTile) continue;
        const int page = p.block_table[ib * p.bt_stride + (tok >> p.page_shift)];
        if (page < 0 || page >= p.num_pages) {
          at[j] = 8;
          lost = true;
        } else {
          at[j] = reinterpret_cast<unsigned long long>(
                      p.pages + block_offset(page, tok & (p.page_size - 1), head, p.page_stride, p.head_stride)) +
                  min(step, is.kv_end - tok + kBlockTokens - 1) / kBlockTokens;
        }
      }
      if (lost) atomicOr(&g_int4_decode_status, kDevErrPage);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; j += 2)
      asm volatile("st.shared.v2.u64 [%0], {%1, %2};" ::"r"(places + lane * 32 + j * 8), "l"(at[j]), "l"(at[j + 1])
                   : "memory");
    __syncwarp();
    absent = __ballot_sync(0xffffffffu, lost);
    moving = __ballot_sync(0xffffffffu, change);
  };
  auto issue = [&](int y) {  // tile y, or nothing behind the last; always one group
    if (y < x1) {
      const int i = (y - x0) & 31, slot = (y - x0) % kDepth;
      const uint32_t to = ring + slot * kTileBytes + lane * 16;
      const uint4 e = lds128(places + i * 32);
      if (__builtin_expect((absent | gone) != 0, 0)) {
        const uint4 f = lds128(places + i * 32 + 16);
        const unsigned b0 = e.x >> 3 & 1u, b1 = e.z >> 3 & 1u, b2 = f.x >> 3 & 1u, b3 = f.z >> 3 & 1u;
        const unsigned blocks = by_block ? b0 | b1 << 1 | b2 << 2 | b3 << 3 : b0 * 3u | b1 * 12u;
        gone = (gone & ~(15u << (4 * slot))) | blocks << (4 * slot);
      }
      auto source = [&](uint32_t lo, uint32_t hi) {
        return reinterpret_cast<const char*>(static_cast<unsigned long long>(hi) << 32 | (lo & ~15u)) + lane * 16;
      };
      auto copy = [&](uint32_t lo, uint32_t hi, uint32_t dst) {
        const char* from = source(lo, hi);
        const int size = static_cast<int>(lo & 3u) * kBlockBytes - lane * 16;
#pragma unroll
        for (int u = 0; u < 2 * kBlockBytes; u += 512)
          if (u < size) copy16(dst + u, from + u);
      };
      if ((((e.x ^ 2u) | (e.z ^ 2u)) & 15u) == 0) {  // two runs of two blocks, as most tiles are
        const char *f0 = source(e.x, e.y), *f1 = source(e.z, e.w);
#pragma unroll
        for (int u = 0; u < 2 * kBlockBytes; u += 512) {
          copy16(to + u, f0 + u);
          copy16(to + 2 * kBlockBytes + u, f1 + u);
        }
      } else if (by_block) {
        const uint4 f = lds128(places + i * 32 + 16);
        copy(e.x, e.y, to);
        copy(e.z, e.w, to + kBlockBytes);
        copy(f.x, f.y, to + 2 * kBlockBytes);
        copy(f.z, f.w, to + 3 * kBlockBytes);
      } else {
        copy(e.x, e.y, to);
        copy(e.z, e.w, to + 2 * kBlockBytes);
      }
    }
    commit_copies();
  };
  // The unit of tile x: its sequence, its place in the list, KV head and first row, the last token that
  // every row sees, and this lane's query rows.
  Seq s;
  int unit = 0, u0 = 0, seg_end = 0, kvh = 0, r0 = 0, all_see = 0;
  const bf16* rows[NT];
  auto enter = [&](int x) {
    s = load_seq<NT>(p, b);
    while (x >= base + s.total(p.nkv)) {
      base += s.total(p.nkv);
      s = load_seq<NT>(p, ++b);
    }
    unit = (x - base) / s.tiles;
    u0 = base + unit * s.tiles;
    seg_end = min(u0 + s.tiles, x1);
    kvh = unit / s.rb;
    r0 = (unit - kvh * s.rb) * C::kRows;
    all_see = static_cast<int>(min(max(s.qpos + by_group(p, r0), -1ll), s.kv_end - 1ll));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + nt * 4 + (g >> 1), i = by_group(p, r);
      rows[nt] = r < s.rows ? p.q + b * p.q_sb + i * p.q_st + (kvh * p.group + r - i * p.group) * p.q_sh + 8 * t
                            : nullptr;
    }
  };
  int issued = x0;
  resolve(x0);
  if (early) {  // tiles that no earlier kernel on the stream still writes
    for (; issued < x0 + kDepth - 1 && !(moving >> (issued - x0) & 1u); ++issued) issue(issued);
  }
  if (x0 < x1) enter(x0);
  if (early) pdl_wait();
  for (; issued < x0 + kDepth - 1; ++issued) issue(issued);

  // ---- the warp's segments: its parts of the units (sequence, head, row block) in [x0, x1) ----
  for (int x = x0; x < x1;) {
    uint32_t qf[NT][4][2], qm[NT][2];
    float fr[NT];
    Acc<NT> A;
    // Query fragments: column lane / 4 of an n8 tile is the hi (even) or lo part of row lane / 8, its k
    // bytes the dims 32 grp + 8t + {0, 2, 4, 6} and + {1, 3, 5, 7}; scores come out times 2^-9 2^e.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint4 v[4];
      uint32_t big = 0;
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
        v[grp] = rows[nt] ? *reinterpret_cast<const uint4*>(rows[nt] + 32 * grp) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int d = 0; d < 4; ++d) big = __vmaxu2(big, word(v[grp], d) & 0x7fff7fffu);
      }
      big = max(big >> 16, big & 0xffffu);  // magnitudes of bf16 numbers compare as integers
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // 2^up with the row's maximum times 2^up in [128, 256); for a row of zeros any power will do
      const int up = min(134 - static_cast<int>(big >> 7), 100);
      const float f = __uint_as_float(static_cast<uint32_t>(127 + up + (g & 1) * 4) << 23);
      float qs[4];
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
        uint32_t two[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {  // dims 2d (low half) and 2d + 1
          // hi: the upper four significant bits; lo: the other four, both exact in bf16
          const uint32_t w = word(v[grp], d), hi = w & 0xfff0fff0u;
          const __nv_bfloat162 lo = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&w),
                                            *reinterpret_cast<const __nv_bfloat162*>(&hi));
          const uint32_t e = g & 1 ? *reinterpret_cast<const uint32_t*>(&lo) : hi;
          const float2 ef = both(mul2(pair(lo_bf16(e), hi_bf16(e)), dup(f)));
          two[d] = e4m3x2(ef.x, ef.y);
        }
        const uint32_t w0 = __byte_perm(two[0], two[1], 0x5410), w1 = __byte_perm(two[2], two[3], 0x5410);
        const uint32_t k[2] = {__byte_perm(w0, w1, 0x6420), __byte_perm(w0, w1, 0x7531)};
        qf[nt][grp][0] = k[0];
        qf[nt][grp][1] = k[1];
        // The sum of the row's dims in the group, as held: a product with ones gives columns 2t, 2t + 1.
        constexpr uint32_t kOnes = 0x38383838u;
        const uint32_t ones[4] = {kOnes, kOnes, kOnes, kOnes};
        float c[4];
        mma_e4m3(c, ones, k[0], k[1], 0.f, 0.f, 0.f, 0.f);
        qs[grp] = fmaf(c[1], 0.0625f, c[0]) * (1.f / kCodeUnit);
      }
      // Column g of the product with mids and scales: the row's sums if g is even, else zeros; k bytes as
      // in tile_step.
      float z[4];
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) z[grp] = __shfl_sync(0xffffffffu, qs[grp], g >> 1);
      float z0 = t & 1 ? z[2] : z[0], z1 = t & 1 ? z[3] : z[1], y0 = -7.5f * z0, y1 = -7.5f * z1;
      if (t & 2) {
        z0 -= __bfloat162float(__float2bfloat16_rn(z0)), z1 -= __bfloat162float(__float2bfloat16_rn(z1));
        y0 -= __bfloat162float(__float2bfloat16_rn(y0)), y1 -= __bfloat162float(__float2bfloat16_rn(y1));
      }
      qm[nt][0] = g & 1 ? 0u : pack_bf16x2(z0, z1);
      qm[nt][1] = g & 1 ? 0u : pack_bf16x2(y0, y1);
      const int row_up = __shfl_sync(0xffffffffu, up, 8 * t);
      fr[nt] = p.scale_log2 * kCodeUnit * __uint_as_float(static_cast<uint32_t>(127 - row_up) << 23);
      A.l[nt] = 0.f, A.off[nt] = 0.f, A.top[nt] = -INFINITY;
      A.pm[nt][0] = A.pm[nt][1] = 0;
      A.sf[nt][0] = A.sf[nt][1] = dup(__uint_as_float(static_cast<uint32_t>(kMostSf) << 23));  // the first tile sets it
    }
#pragma unroll
    for (int c = 0; c < Acc<NT>::kCols; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int grp = 0; grp < 4; ++grp)
          if (j < Acc<NT>::kKept) A.o[c][grp][0][j] = A.o[c][grp][1][j] = 0.f;
        A.xs[c][0][j] = A.xs[c][NT > 1][j] = 0.f;
      }
    // ---- its tiles ----
    for (; x < seg_end; ++x) {
      if (__builtin_expect((issued - x0 & 31) == 0, 0)) resolve(issued);
      issue(issued++);
      wait_copies<kDepth - 1>();
      __syncwarp();
      const int slot = (x - x0) % kDepth;
      const int tok = (x - u0) * kTile;
      const unsigned there = ~gone >> (4 * slot) & 15u;
      const bool masked = there != 15u || tok + kTile - 1 > all_see;
      int lim[NT];
      if (__builtin_expect(masked, 0)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int r = r0 + nt * 4 + t;
          const long long last = min(s.qpos + by_group(p, r), static_cast<long long>(s.kv_end) - 1);
          lim[nt] = r < s.rows ? static_cast<int>(max(last, -1ll)) : -1;
        }
      }
      tile_step<NT, kApart>(ring + slot * kTileBytes, qf, qm, A, fr, masked, lim, tok, there);
      __syncwarp();
    }

    const bool from_before = x0 > u0, goes_on = seg_end < u0 + s.tiles;
    if (!p.direct && lane == 0) {
      int2* span = p.span + (b * p.nkv + kvh) * p.rb + (unit - kvh * s.rb);
      if (!from_before) span->x = 2 * blockIdx.x + (range[0].x0 >= u0 ? 0 : 1);
      if (!goes_on) span->y = blockIdx.x;
    }
    const int which = 2 * warp + (from_before ? 0 : 1);
    const int live = min(C::kRows, s.rows - r0);
    const bool mine = !from_before && !goes_on && p.cluster == 1;
    if (!mine && lane == 0) edge[which] = {u0, u0 + s.tiles, b, kvh, r0, live};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 pm0 = both(A.pm[nt][0]), pm1 = both(A.pm[nt][1]);
      float l = A.l[nt], pm[4] = {pm0.x, pm0.y, pm1.x, pm1.y};
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) pm[grp] += __shfl_xor_sync(0xffffffffu, pm[grp], o);
      }
      const int row = nt * 4 + t;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (!mine && g == 0) ml[which * C::kRows + row] = make_float2(A.off[nt], l);
      const int i = by_group(p, r0 + row), h = kvh * p.group + r0 + row - i * p.group;
      bf16* to = p.out + b * p.o_sb + i * p.o_st + h * p.o_sh + 4 * g;
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
        const float4 v = chunk_of<NT>(A, nt, grp, pm[grp]);
        if (!mine) {
          // float4 number 8 grp + g of the row, its place xored with the row: no bank conflict
          *reinterpret_cast<float4*>(part_row(which, row) + ((8 * grp + g) ^ (2 * t)) * 4) = v;
        } else if (row < live) {
          *reinterpret_cast<uint2*>(to + 32 * grp) =
              make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
        }
      }
    }
    if (x < x1) enter(x);
  }
  __syncthreads();

  // ---- units that the CTA's warps share, added up row by row by warps in turn ----
  const int e = lane < 2 * kWarps ? edge[lane].u0 : -1;
  const int cta0 = range[0].x0, cta1 = range[kWarps].x0;
  if (p.direct && p.cluster == 1 && cta0 == cta1) {  // rows that see no key
    const Seq z = load_seq<NT>(p, blockIdx.y);
    if (static_cast<int>(blockIdx.x) >= z.units(p.nkv)) return;
    const int head = blockIdx.x / z.rb, row0 = (blockIdx.x - head * z.rb) * C::kRows;
    for (int row = warp; row < min(C::kRows, z.rows - row0); row += kWarps)
      write_row4(p, blockIdx.y, head, row0 + row, lane * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  unsigned todo = __ballot_sync(0xffffffffu, e >= 0);
  for (int turn = 0; todo; ) {
    const int first = __ffs(todo) - 1, unit0 = __shfl_sync(0xffffffffu, e, first);
    const unsigned parts = __ballot_sync(0xffffffffu, e == unit0);
    todo &= ~parts;
    const Edge u = edge[first];
    const bool whole = cta0 <= u.u0 && u.u1 <= cta1 && p.cluster == 1;
    const int part = 2 * blockIdx.x + (cta0 >= u.u0 ? 0 : 1);
    for (int row = 0; row < u.live; ++row, ++turn) {
      if (turn % kWarps != warp) continue;
      float2 v[kWarps];
      float4 x[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {  // a warp has one part of a unit at most, as its first or its last
        const unsigned has = parts >> (2 * w) & 3u;
        const int at = 2 * w + static_cast<int>(has >> 1);
        v[w] = has ? ml[at * C::kRows + row] : make_float2(-INFINITY, 0.f);
        x[w] = has ? *reinterpret_cast<const float4*>(part_row(at, row) + (lane ^ (2 * (row & 3))) * 4)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float M = -INFINITY, L = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        if (v[w].y != 0.f) M = fmaxf(M, v[w].x);  // a part that sees no key of the row does not count
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = v[w].y == 0.f ? 0.f : ex2(v[w].x - M);
        L += f * v[w].y;
        o = make_float4(o.x + f * x[w].x, o.y + f * x[w].y, o.z + f * x[w].z, o.w + f * x[w].w);
      }
      if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        write_row4(p, u.seq, u.head, u.row0 + row, lane * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      } else if (p.cluster > 1) {
        *reinterpret_cast<float4*>(smem + C::kOffUnit + (row * kHD + lane * 4) * 4) = o;
        if (lane == 0) unit_ml[row] = make_float2(M, L);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(part) * C::kRows + row) * kHD + lane * 4) = o;
        if (lane == 0) p.part_ml[part * C::kRows + row] = make_float2(M, L);
      }
    }
  }
  if (p.cluster == 1) return;

  // ---- the cluster's unit, its rows added up by the CTAs and their warps in turn ----
  cluster_sync();
  const Seq z = load_seq<NT>(p, blockIdx.y);
  const int cu = blockIdx.x / p.cluster, rank = blockIdx.x - cu * p.cluster;
  if (cu < z.units(p.nkv)) {
    const int head = cu / z.rb, row0 = (cu - head * z.rb) * C::kRows;
    for (int row = rank + warp * p.cluster; row < min(C::kRows, z.rows - row0); row += kWarps * p.cluster) {
      const uint32_t at = smem_u32(smem) + C::kOffUnit + (row * kHD + lane * 4) * 4;
      const uint32_t at_ml = smem_u32(smem) + C::kOffUnitMl + row * 8;
      float2 v[kMostCluster];
      float4 x[kMostCluster];
#pragma unroll
      for (int c = 0; c < kMostCluster; ++c) {
        v[c] = make_float2(-INFINITY, 0.f);
        x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < p.cluster) {
          v[c] = cluster_lds64(in_cluster(at_ml, c));
          if (v[c].y != 0.f) x[c] = cluster_lds128(in_cluster(at, c));
        }
      }
      float M = -INFINITY, L = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kMostCluster; ++c)
        if (v[c].y != 0.f) M = fmaxf(M, v[c].x);
#pragma unroll
      for (int c = 0; c < kMostCluster; ++c) {
        const float f = v[c].y == 0.f ? 0.f : ex2(v[c].x - M);
        L += f * v[c].y;
        o = make_float4(o.x + f * x[c].x, o.y + f * x[c].y, o.z + f * x[c].z, o.w + f * x[c].w);
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      write_row4(p, blockIdx.y, head, row0 + row, lane * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
  }
  cluster_sync();  // no CTA leaves while its sums are read
}

// The rows whose tiles were divided between CTAs: one CTA per output row, whose warps take the parts
// in turn. Rows that see no key are zeroed here too. Bound by its latency: two round trips to L2, and
// what the many rows of a large batch, mostly written whole already, take to leave.
constexpr int kMergeWarps = 8;
constexpr int kMergeLoads = 5;  // parts of a warp whose loads are in flight together: 40 parts a round trip
template <int NT>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const Params p) {
  using C = Cfg<NT>;
  __shared__ float4 so[kMergeWarps][32];
  __shared__ float2 sm[kMergeWarps];
  if (!p.stable_prefix) pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  const int R = blockIdx.x;
  const int h = R % p.nh, i = (R / p.nh) % p.q_len, b = R / (p.nh * p.q_len);
  const int kvh = h / p.group, r = i * p.group + h - kvh * p.group;
  const Seq s = load_seq<NT>(p, b);
  if (p.stable_prefix) pdl_wait();
  const int2 span = p.span[(b * p.nkv + kvh) * p.rb + r / C::kRows];
  if (r >= s.rows) return;
  if (s.tiles == 0) {
    if (warp == 0) write_row4(p, b, kvh, r, lane * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int c0 = span.x >> 1, c1 = span.y;
  if (c0 == c1) return;  // written whole
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = c0 + warp; c <= c1; c += warps * kMergeLoads) {
    float2 v[kMergeLoads];
    float4 u[kMergeLoads];
#pragma unroll
    for (int j = 0; j < kMergeLoads; ++j) {
      const int cj = c + j * warps;
      v[j] = make_float2(-INFINITY, 0.f);
      u[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (cj <= c1) {
        const int part = cj == c0 ? span.x : 2 * cj;  // behind its first CTA a unit is the CTA's first
        const int64_t row = static_cast<int64_t>(part) * C::kRows + r % C::kRows;
        v[j] = p.part_ml[row];
        u[j] = *reinterpret_cast<const float4*>(p.part_o + row * kHD + lane * 4);
      }
    }
    float m = M;  // a part that sees no key of the row (sum 0) does not count; a NaN goes on
#pragma unroll
    for (int j = 0; j < kMergeLoads; ++j) m = v[j].y == 0.f ? m : fmaxf(m, v[j].x);
    const float f0 = L == 0.f ? 0.f : ex2(M - m);
    M = m;
    L *= f0;
    o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
#pragma unroll
    for (int j = 0; j < kMergeLoads; ++j) {
      const float f = v[j].y == 0.f ? 0.f : ex2(v[j].x - m);
      L += f * v[j].y;
      o = make_float4(o.x + f * u[j].x, o.y + f * u[j].y, o.z + f * u[j].z, o.w + f * u[j].w);
    }
  }
  so[warp][lane] = o;
  if (lane == 0) sm[warp] = make_float2(M, L);
  __syncthreads();
  if (warp) return;
  for (int w = 0; w < warps; ++w) M = sm[w].y == 0.f ? M : fmaxf(M, sm[w].x);
  L = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < warps; ++w) {
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
  int nt = 1, ctas = 1, rb = 1, cluster = 1;
  bool direct = false, apart = false;
  size_t o_bytes = 0, ml_bytes = 0, ws_bytes = 0;
};

int make_plan(const SolortInt4DecodeArgs* a, Plan* pl) {
  if (!a) return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->head_dim != kHD) return SOLORT_ERR_UNSUPPORTED;
  if (a->batch <= 0 || a->q_len <= 0 || a->num_qo_heads <= 0 || a->num_kv_heads <= 0 ||
      a->max_kv_len <= 0 || a->num_ctas < 0)
    return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->num_qo_heads % a->num_kv_heads != 0) return SOLORT_ERR_INVALID_ARGUMENT;
  if (a->batch > 65535) return SOLORT_ERR_UNSUPPORTED;
  // Four rows a block where they fit one, else eight: a tile of eight takes 1.4 of four's time (1392 and
  // 979 cycles a scheduler, 1519 with kApart), which two blocks of four would take twice.
  const int64_t rows = static_cast<int64_t>(a->q_len) * (a->num_qo_heads / a->num_kv_heads);
  pl->nt = rows <= 4 ? 1 : 2;
  const int warps = pl->nt == 1 ? Cfg<1>::kWarps : Cfg<2>::kWarps;
  const int64_t rb = (rows + 4 * pl->nt - 1) / (4 * pl->nt);
  const int64_t tiles = (static_cast<int64_t>(a->max_kv_len) + kTile - 1) / kTile + kUnitCost;
  const int64_t units = rb * a->num_kv_heads;
  const int64_t out_rows = static_cast<int64_t>(a->batch) * a->q_len * a->num_qo_heads;
  // Tokens, and places in the list, stay inside an int with a tile, or a CTA's warps, added to them.
  const int64_t limit = (1ll << 31) - 1, most_listed = 1ll << 30;
  if (rows > limit || units > limit || out_rows > limit || a->max_kv_len > kMostKeys ||
      tiles > most_listed / units || tiles * units > most_listed / a->batch)
    return SOLORT_ERR_UNSUPPORTED;
  DeviceInfo di;
  int rc = current_device_info(&di);
  if (rc != SOLORT_OK) return rc;
  pl->rb = static_cast<int>(rb);
  const int64_t most = (tiles * units * a->batch + warps - 1) / warps;
  const int64_t wave = a->num_ctas > 0 ? a->num_ctas
                                       : static_cast<int64_t>(di.sm_count) *
                                             (pl->nt == 1 ? Cfg<1>::kCtasPerSm : Cfg<2>::kCtasPerSm);
  if (wave > (1 << 20)) return SOLORT_ERR_UNSUPPORTED;
  // Short caches are not divided: a unit is a cluster of k CTAs with 6 k warps, where all clusters are
  // resident at once, a warp's tiles are few, and no more than its share of the divided list and what the
  // division costs. k is what a warp's tiles and the cluster cost least with, in quarters of a tile; two
  // CTAs on an SM cost one more. 32 heads over 8, us with clusters of 1, 2, 4, 8 | divided:
  //   1 x 256 keys   4.9  5.5  5.8  6.6 | 7.5      8 x 1024    9.9  8.7  9.2    - | 10.6
  //   1 x 768        7.7  6.8  5.9  6.5 | 7.7      8 x 4096   28.6 18.2 15.9    - | 17.5
  //   1 x 1536      12.4  9.2  7.2  6.6 | 7.8     16 x 1024   10.3 10.7    -    - | 12.6
  //   1 x 4096      27.8 17.2 11.4  9.1 | 9.0     64 x 256       -    -    -    - | 16.5
  constexpr int kClusterCost[] = {0, 4, 5, 8};
  int64_t least = 0, steps = 0;
  for (int i = 0; (1 << i) <= kMostCluster && (units * a->batch << i) <= wave; ++i) {
    const int64_t of = (tiles - kUnitCost + (warps << i) - 1) / (warps << i);
    const int64_t cost = 4 * of + kClusterCost[i] + (i && (units * a->batch << i) > di.sm_count ? 4 : 0);
    if (i == 0 || cost < least) least = cost, steps = of, pl->cluster = 1 << i;
  }
  const bool bare = tiles - kUnitCost <= kBareTiles;
  pl->direct = a->num_ctas == 0 && units * a->batch <= wave &&
               (bare || (steps <= kDirectSteps && (steps - kSplitSteps) * wave <= most));
  if (!pl->direct) pl->cluster = 1;
  // The workspace never shrinks as a size grows: one for the largest call serves the smaller ones.
  if (pl->direct && bare) return SOLORT_OK;
  pl->ctas = static_cast<int>(most < wave ? most : wave);
  pl->apart = !pl->direct && tiles * units * a->batch > static_cast<int64_t>(kApartTiles) * pl->ctas * warps;
  const size_t parts = static_cast<size_t>(2) * pl->ctas * 4 * pl->nt;
  pl->o_bytes = parts * kHD * 4;
  pl->ml_bytes = parts * 8;
  pl->ws_bytes = align_up(pl->o_bytes + pl->ml_bytes + static_cast<size_t>(units) * a->batch * 8, 256);
  return SOLORT_OK;
}

inline cudaLaunchConfig_t pdl_config(dim3 grid, int threads, size_t smem, void* stream,
                                     int cluster, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cfg;
}

template <int NT, bool kApart>
int launch(const Params& prm, const Plan& pl, void* stream) {
  using C = Cfg<NT>;
  static std::atomic<unsigned> configured{0};  // one bit per device ordinal < 32
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SOLORT_ERR_CUDA;
  if (dev >= 32 || !(configured.load(std::memory_order_acquire) & (1u << dev))) {
    if (cudaFuncSetAttribute(decode_kernel<NT, kApart>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
            cudaSuccess ||
        cudaFuncSetAttribute(decode_kernel<NT, kApart>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared) != cudaSuccess)
      return SOLORT_ERR_CUDA;
    if (dev < 32) configured.fetch_or(1u << dev, std::memory_order_release);
  }
  cudaLaunchAttribute attr[2];
  const dim3 grid = pl.direct ? dim3(prm.nkv * pl.rb * pl.cluster, prm.batch) : dim3(pl.ctas);
  cudaLaunchConfig_t cfg = pdl_config(grid, C::kThreads, C::kSmem, stream, pl.cluster, attr);
  if (cudaLaunchKernelEx(&cfg, decode_kernel<NT, kApart>, prm) != cudaSuccess) return SOLORT_ERR_CUDA;
  int rc = launch_status();
  if (rc != SOLORT_OK || pl.direct) return rc;
  // Few rows have many parts each and want many warps (131072 keys, 32 rows: 8 warps 38.8 us, 2 warps
  // 41.1); of many rows most are written already and want to leave (48 sequences, 1536 rows: 38.1 and 35.4).
  const int rows = prm.batch * prm.q_len * prm.nh;
  cfg = pdl_config(dim3(rows), (rows <= pl.ctas ? kMergeWarps : 2) * 32, 0, stream, 1, attr);
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
    p.span = reinterpret_cast<int2*>(static_cast<uint8_t*>(a->workspace) + pl.o_bytes + pl.ml_bytes);
  }
  p.batch = a->batch;
  p.q_len = a->q_len;
  p.nh = a->num_qo_heads;
  p.nkv = a->num_kv_heads;
  p.group = a->num_qo_heads / a->num_kv_heads;
  int log = 0;  // ceil(log2(group))
  while ((1ll << log) < p.group) ++log;
  p.group_mul = static_cast<uint32_t>(((1ull << (31 + log)) + p.group - 1) / p.group);
  p.group_shift = log - 1;
  p.max_kv_len = a->max_kv_len;
  p.direct = pl.direct ? 1 : 0;
  p.cluster = pl.cluster;
  p.ctas = pl.ctas;
  p.rb = pl.rb;
  p.stable_prefix = (a->flags & SOLORT_DECODE_STABLE_PREFIX) ? 1 : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  return pl.nt == 1 ? i4::launch<1, true>(p, pl, stream)
         : pl.apart ? i4::launch<2, true>(p, pl, stream)
                    : i4::launch<2, false>(p, pl, stream);
}
