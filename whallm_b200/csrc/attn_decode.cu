// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale q.k_j,  lse = log sum_j exp(s_j),  out = sum_j exp(s_j - lse) v_j
//
// for the G = Hq / Hkv query heads of each key-value head at once.  The call is
// HBM bound: every cached row is read once for each 16 of these heads, 4 D bytes (bf16)
// per entry and head against 4 D G operations.
//
// Work split.  The entries of all (sequence, head) pairs form one line of units
// of 64 keys; every CTA takes a share of the line (struct Line), found from the
// lengths on the device (no host copy, so a captured call follows the lengths).
// A CTA that meets the end of a pair writes its part (running maximum, sum and
// unnormalised output) and goes on with the next pair; a second kernel joins
// the parts of each pair with weights 2^(m_part - m).  Ragged batches are
// balanced to one unit, and one long sequence fills the GPU.
//
// A warp owns 16 keys of each unit.  It streams their rows through its own ring
// of cp.async stages, so the main loop has no block-wide barrier; rows behind
// the length are filled with zeros and never read.  Scores are computed as
// K Q^T with the keys on the M side of m16n8k16 (8 query heads cost one N = 8
// tile; padding heads to M = 16 would double the arithmetic of small groups),
// and O^T = V^T P^T likewise: the score fragment, rounded to bf16, turns into
// the B operand by one 8x8 transpose in registers.  Maximum, sum and output are
// 32-bit; P is rounded to bf16 once, the type of V, an error of at most 2^-8 of
// each weight that the sum over keys averages out.
//
// e4m3 rows are widened to f16, which holds every e4m3 value, in one instruction
// per pair, and multiplied there (widening to bf16 takes four; at D = 256 that
// arithmetic, not the memory, set the time).  The query goes to f16 with a power
// of two per head that puts its largest magnitude into [2^14, 2^15): exact for
// values within 2^-28 of it, off by less than 2^-39 of it below.  A key's block
// scales multiply its partial scores.  A value's block scales multiply its weight
// before the rounding, times a power of two for the block's dimensions that keeps
// the product at most 2^15.  It starts at 2^115 and falls when a scale of the warp's
// values needs it, then to 2^13 so that this happens once or twice per part (O is
// rescaled as for the maximum): the weights are rounded to 11 bits down to 2^-26 of
// the largest of their block, and no dequantized row is ever rounded.
//
// Measured (CUDA graphs, three input sets in turn): 64 sequences of 90 to 8190
// entries, 32/8 heads of 128, bf16: 166 us, 6.7 TB/s (a plain copy: 6.5); two of
// 130,000 entries, 16/2 heads of 256, e4m3: 53 to 56 us, the rows at 5.7 TB/s; one of
// 4095 entries, 32/8 heads of 128: 9.4 us, a chain of latencies.
#include <cooperative_groups.h>

#include <algorithm>

#include "wm_paged.cuh"
#include "wm_stream.cuh"
#include "wm_tc.cuh"

namespace cg = cooperative_groups;
using wm_paged::Pool;

namespace {

constexpr int kWarps = 4;
constexpr int kTile = 16;               // keys of a warp's tile
constexpr int kUnit = kWarps * kTile;   // keys of a unit of work
constexpr int kMaxCluster = 8;
constexpr int kClusterKeys = 1024;      // capacity per CTA up to which a cluster joins a pair
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTopWeight = 32768.0f;  // of a weight in f16
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();

struct DecodeArgs {
  Pool pool;
  const wm_bf16 *q;
  int64_t q_stride;                     // between sequences; heads are dense
  const int32_t *lengths;
  int B, Hq, G, NC;                     // query heads, heads per kv head, chunks of query heads per kv head
  float scale2;                         // scale * log2(e)
  wm_bf16 *out;                         // [B, Hq, D]
  float *lse;                           // [B, Hq] or null
  float *mass;                          // [B, Hkv, capacity] or null
  float *part_o, *part_m, *part_l;      // parts: [slots][heads of a chunk][D] and [slots][heads of a chunk]
  float *scores;                        // [pairs][capacity][score_heads], with mass only
  int score_heads;                      // a chunk's query heads, rounded up to 2
  int n_cta, rounds;                    // CTAs of a round over the line; rounds that a full cache would have
  int cluster;                          // CTAs per pair, or 0 for the line
};

// x / y for x >= 0, y > 0: 64-bit divisions are subroutines of about 0.4 us on the
// critical path, and nearly every position on the line fits 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return x / y;
}

__device__ __forceinline__ int64_t units_of(const DecodeArgs &a, int b) {
  const int64_t len = a.lengths[b], cap = static_cast<int64_t>(a.pool.max_pages) * a.pool.page_size;
  return len <= 0 ? 0 : ((len < cap ? len : cap) + kUnit - 1) / kUnit;
}

// Units before sequence `upto` (all of them for upto = B), summed by one warp.
__device__ __forceinline__ int64_t warp_units(const DecodeArgs &a, int upto) {
  int64_t s = 0;
  for (int b = threadIdx.x & 31; b < upto; b += 32) s += units_of(a, b);
#pragma unroll
  for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
  return s;
}

// The line of units cut among the CTAs.  Equal shares end at different times, as
// SMs do not get equal bandwidth (130 to 180 us for 114 units a CTA), so a long line
// has three rounds of up to a.n_cta CTAs, as many as fit on the GPU at once: the
// first round gets 12 / 16 of it, the later ones, whose CTAs start wherever one has
// ended, 3 / 16 and 1 / 16 in shares of at least kLeastUnits.  64 sequences of 90 to
// 8190 entries, 32/8 heads of 128: 182 -> 165 us.  At 27 units a CTA the later CTAs'
// starts cost more than they even out (two of 130,000 entries, e4m3 of 256 values:
// 53 -> 61 us), so shorter lines have one round.  Every CTA that takes part has at
// least one unit and their numbers follow one another along the line, so every part
// between a pair's first and last is written.
constexpr int kTiers = 3;
__device__ constexpr int kShare[kTiers] = {12, 3, 1};
constexpr int kTierUnits = 64;          // units per CTA from which there are several rounds
constexpr int kLeastUnits = 16;

struct Line {
  int64_t from[kTiers + 1];             // the rounds' ends on the line
  int n;                                // CTAs of a round
  __device__ __forceinline__ Line(const DecodeArgs &a, int64_t total) : n(a.n_cta) {
    const bool several = total >= static_cast<int64_t>(kTierUnits) * a.n_cta;
    from[0] = 0;
    int done = 0;
#pragma unroll
    for (int k = 0; k < kTiers; ++k) {
      done += kShare[k];
      from[k + 1] = several ? total * done / 16 : total;
    }
  }
  // CTAs of round k that have units, and the units of CTA i: [start(i), start(i + 1))
  __device__ __forceinline__ int64_t count(int k) const {
    const int64_t l = from[k + 1] - from[k];
    return min(k ? (l + kLeastUnits - 1) / kLeastUnits : l, static_cast<int64_t>(n));
  }
  __device__ __forceinline__ int64_t start(int i) const {
    int64_t x = from[kTiers];
#pragma unroll
    for (int k = kTiers - 1; k >= 0; --k) {
      const int64_t r = i - base(k), c = count(k);
      if (r >= 0 && r < c) x = from[k] + quotient((from[k + 1] - from[k]) * r, c);
    }
    return x;
  }
  __device__ __forceinline__ int64_t base(int k) const {           // CTAs of the rounds before
    int64_t b = 0;
#pragma unroll
    for (int y = 0; y < kTiers; ++y) b += y < k ? count(y) : 0;
    return b;
  }
  // the CTA that holds unit x
  __device__ __forceinline__ int64_t cta(int64_t x) const {
    int64_t i = 0;
#pragma unroll
    for (int k = 0; k < kTiers; ++k)
      if (x >= from[k] && x < from[k + 1]) i = base(k) + quotient((x - from[k] + 1) * count(k) - 1, from[k + 1] - from[k]);
    return i;
  }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// cached rows pass through L2 once: evict-first, so that the scores and parts that the join reads stay there
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Scales of one row as floats.
template <int FMT, int N>
__device__ __forceinline__ void load_scales(const uint8_t *p, float (&f)[N]) {
  if constexpr (FMT == WKV_FP8_F32_B64) {
    if constexpr (N == 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p);
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else if constexpr (N == 2) {
      const float2 v = *reinterpret_cast<const float2 *>(p);
      f[0] = v.x; f[1] = v.y;
    } else {
      f[0] = *reinterpret_cast<const float *>(p);
    }
  } else if constexpr (FMT == WKV_MXFP8_B32) {
    uint32_t w[(N + 3) / 4];
    if constexpr (N == 8) {
      const uint2 v = *reinterpret_cast<const uint2 *>(p);
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (N == 4) {
      w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = wm_e8m0((w[i >> 2] >> (8 * (i & 3))) & 255u);
  }
}

template <int D, int FMT, int NH>
struct Shape {
  static constexpr int kRow = wm_paged::row_bytes(FMT, D);        // bytes of a row
  static constexpr int kChunks = kRow / 16;
  static constexpr int kScale = wm_paged::scale_bytes(FMT, D);    // bytes of a row's scales
  static constexpr int kBlocks = FMT == WKV_BF16 ? 1 : (FMT == WKV_FP8_F32_B64 ? D / 64 : D / 32);
  // 16 heads of 256 fill the registers: the blocks' factors are held in shared memory (87 -> 79 us for two of 130,000
  // MXFP8 entries, 32/2 heads; smaller shapes lose 1 %)
  static constexpr bool kFar = D == 256 && NH == 2 && FMT != WKV_BF16;
  static constexpr int kStage = 2 * kTile * (kRow + kScale);      // keys, values and their scales
  static constexpr int kStages = D == 64 && FMT != WKV_BF16 ? 4 : 3;
  static constexpr int kHeads = 8 * NH;
  static constexpr int kMerge = kWarps * kHeads * D * 4;          // the warps' outputs when a part ends
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

// 16-byte piece c of row r: an XOR of the piece with the row (pairs of rows for
// 64-byte rows) spreads the eight rows of an 8x8 block over all banks.
template <int kRow>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  if constexpr (kRow >= 128) return static_cast<uint32_t>(r * kRow + ((c ^ (r & 7)) << 4));
  const uint32_t a = static_cast<uint32_t>(r * kRow + (c << 4));
  return a ^ ((a >> 3) & 0x70u);
}

// Factor of a part with maximum m under the pair's maximum: a part without a
// finite score keeps its sum (zero, or NaN).
__device__ __forceinline__ float part_factor(float m, float top) { return m == kNegInf ? 1.0f : ex2(m - top); }

// 1 / x for a power of two in [2^-126, 2^126]
__device__ __forceinline__ float inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// CL: a cluster of CTAs per pair instead of a share of the line (see launch()).
template <int D, int FMT, int NH, bool CL>
__global__ void __launch_bounds__(kWarps * 32) k_attn_decode(DecodeArgs a) {
  using S = Shape<D, FMT, NH>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_m[kWarps][S::kHeads], sm_l[kWarps][S::kHeads];
  __shared__ float2 sm_part[S::kHeads];               // the CTA's maximum and sum
  __shared__ __align__(16) float sm_factor[kWarps][S::kFar ? S::kBlocks : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, i2 = (lane & 3) * 2;
  uint8_t *ring = smem + warp * (S::kStages * S::kStage);
  const uint32_t ring_u = wm_tc::smem_u32(ring);
  const uint64_t policy = wm_tc::l2_evict_first_policy();
  WM_PDL_WAIT();
  WM_PDL_LAUNCH();                                    // the join may be placed; it waits for this kernel's end

  const int PH = a.pool.Hkv * a.NC;
  const int64_t cap = static_cast<int64_t>(a.pool.max_pages) * a.pool.page_size;

  // units [unit0, unit1) of the pair (sequence b, hc = kv head and chunk of its query heads)
  auto segment = [&](const int b, const int hc, const int64_t unit0, const int64_t unit1) {
    const int h = hc / a.NC, c = hc - h * a.NC;
    const int64_t pair = static_cast<int64_t>(b) * PH + hc;
    const int len = static_cast<int>(a.lengths[b] < cap ? max(a.lengths[b], 0) : cap);
    const int32_t *table = a.pool.table + static_cast<int64_t>(b) * a.pool.max_pages;

    // tiles of this warp: 16 keys at (unit * 4 + warp) * 16
    const int t0 = static_cast<int>(unit0) * kWarps + warp;
    int n = static_cast<int>(unit1 - unit0);
    if (n > 0 && (static_cast<int64_t>(t0) + static_cast<int64_t>(n - 1) * kWarps) * kTile >= len) --n;
    bool bad = false;

    // query fragments (the B operand: k = dimension, n = head), zero for heads past the group
    constexpr int KS = D / 16;
    uint32_t qf[NH][KS][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      const int hg = c * S::kHeads + nh * 8 + g;
      const wm_bf16 *qp = a.q + b * a.q_stride + static_cast<int64_t>(h * a.G + hg) * D;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // e4m3 fragments hold four neighbouring values where bf16 ones hold two pairs eight apart
        const int d0 = FMT == WKV_BF16 ? 16 * ks + i2 : 16 * ks + 2 * i2;
        const int d1 = FMT == WKV_BF16 ? d0 + 8 : d0 + 2;
        qf[nh][ks][0] = hg < a.G ? *reinterpret_cast<const uint32_t *>(qp + d0) : 0u;
        qf[nh][ks][1] = hg < a.G ? *reinterpret_cast<const uint32_t *>(qp + d1) : 0u;
      }
    }

    // scores in units of log2: factor of this thread's two heads
    float sc2[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      sc2[nh][0] = sc2[nh][1] = a.scale2;
      if constexpr (FMT != WKV_BF16) {
        uint32_t top = 0u;                            // largest magnitude of head g, as bf16 bits
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) top = __vmaxu2(top, __vmaxu2(qf[nh][ks][0] & 0x7fff7fffu, qf[nh][ks][1] & 0x7fff7fffu));
        top = max(top & 0xffffu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max(static_cast<int>(top >> 7) - 141, -100);
        const float down = wm_stream::pow2f(-e), up = wm_stream::pow2f(e) * a.scale2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            qf[nh][ks][x] = wm_stream::f32x2_to_f16x2(wm_bf16lo(qf[nh][ks][x]) * down, wm_bf16hi(qf[nh][ks][x]) * down);
        sc2[nh][0] = __shfl_sync(0xffffffffu, up, i2 * 4);
        sc2[nh][1] = __shfl_sync(0xffffffffu, up, i2 * 4 + 4);
      }
    }

    float o[D / 16][NH][4];
    float m[NH][2], l[NH][2];
    float factor[S::kBlocks];                         // e4m3: of the weights and O of a block's dimensions, a power of two
#pragma unroll
    for (int blk = 0; blk < S::kBlocks; ++blk) factor[blk] = 0x1p115f;
    auto keep_factors = [&] {                         // where registers are short: in shared memory between their uses
      if constexpr (S::kFar) {
        __syncwarp();
        if (lane == 0)
#pragma unroll
          for (int blk = 0; blk < S::kBlocks; ++blk) sm_factor[warp][blk] = factor[blk];
        __syncwarp();
      }
    };
    auto fetch_factors = [&] {
      if constexpr (S::kFar) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int blk = 0; blk < S::kBlocks; ++blk) factor[blk] = sm_factor[warp][blk];
      }
    };
    keep_factors();
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
      for (int nh = 0; nh < NH; ++nh)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[mt][nh][j] = 0.0f;
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      m[nh][0] = m[nh][1] = kNegInf;
      l[nh][0] = l[nh][1] = 0.0f;
    }

    const uint32_t lane_swz = swz<S::kRow>(lane / S::kChunks, lane % S::kChunks);
    int pages = 0, slots = 0;                         // lane i: page and slot of the first key of tile 32 * block + i
    auto issue = [&](int i) {
      if (i < n) {
        if ((i & 31) == 0) {
          if (i + lane < n) {
            const int first = (t0 + (i + lane) * kWarps) * kTile, pi = first / a.pool.page_size;
            pages = table[pi];
            slots = first - pi * a.pool.page_size;
          }
        }
        const int page = __shfl_sync(0xffffffffu, pages, i & 31), slot = __shfl_sync(0xffffffffu, slots, i & 31);
        const int key = (t0 + i * kWarps) * kTile;
        const int rows = min(kTile, len - key);
        const bool ok = page >= 0 && page < a.pool.n_pages;
        bad |= !ok;
        const int64_t row = ok ? (static_cast<int64_t>(page) * a.pool.Hkv + h) * a.pool.page_size + slot : 0;
        const uint32_t st = ring_u + (i % S::kStages) * S::kStage;
        const uint8_t *kp = static_cast<const uint8_t *>(a.pool.k) + row * S::kRow;
        const uint8_t *vp = static_cast<const uint8_t *>(a.pool.v) + row * S::kRow;
        // a tile is one run of bytes; step x of the warp copies 512 of them, whose swizzle differs from step 0's by
        // a constant
        if (ok && rows == kTile) {
#pragma unroll
          for (int x = 0; x < kTile * S::kChunks / 32; ++x) {
            constexpr int kStep = S::kRow >= 128 ? 512 / S::kRow : 4;     // swizzle units of 512 bytes
            const uint32_t dst = st + x * 512 + (lane_swz ^ (((x * kStep) & 7) << 4));
            cp16(dst, kp + lane * 16 + x * 512, policy);
            cp16(dst + kTile * S::kRow, vp + lane * 16 + x * 512, policy);
          }
        } else {
#pragma unroll 1
          for (int x = 0; x < kTile * S::kChunks / 32; ++x) {
            const int r = (x * 32 + lane) / S::kChunks, cc = (x * 32 + lane) % S::kChunks;
            const int take = ok && r < rows ? 16 : 0;
            const int64_t off = take ? (x * 32 + lane) * 16 : 0;
            cp16(st + swz<S::kRow>(r, cc), kp + off, take);
            cp16(st + kTile * S::kRow + swz<S::kRow>(r, cc), vp + off, take);
          }
        }
        if constexpr (S::kScale > 0) {
          constexpr int per = kTile * S::kScale / 16; // 16-byte pieces of a tile's scales
          const int which = lane / per, cc = lane % per;
          if (which < 2) {
            const int take = ok ? max(0, min(16, rows * S::kScale - cc * 16)) : 0;
            const uint8_t *sp = static_cast<const uint8_t *>(which ? a.pool.vs : a.pool.ks) + row * S::kScale + (take ? cc * 16 : 0);
            cp16(st + 2 * kTile * S::kRow + which * (kTile * S::kScale) + cc * 16, sp, take);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) issue(i);
    for (int i = 0; i < n; ++i) {
      issue(i + S::kStages - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
      __syncwarp();
      const uint32_t kt = ring_u + (i % S::kStages) * S::kStage, vt = kt + kTile * S::kRow;
      const uint8_t *sc = ring + (i % S::kStages) * S::kStage + 2 * kTile * S::kRow;
      float ka[S::kBlocks], kb[S::kBlocks], va[S::kBlocks], vb[S::kBlocks];     // scales of keys and values g and g + 8
      if constexpr (FMT != WKV_BF16) {
        load_scales<FMT>(sc + g * S::kScale, ka);
        load_scales<FMT>(sc + (g + 8) * S::kScale, kb);
      }

      // scores: rows are keys (g, g + 8), columns heads (i2, i2 + 1)
      float s[NH][4];
#pragma unroll
      for (int nh = 0; nh < NH; ++nh)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[nh][j] = 0.0f;
      const int lr = lane & 15, lc = lane >> 4;
      if constexpr (FMT == WKV_BF16) {
        float s2[NH][4] = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t f[4];
          ldsm4(f, kt + swz<S::kRow>(lr, 2 * ks + lc));
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) mma((ks & 1) ? s2[nh] : s[nh], f, qf[nh][ks][0], qf[nh][ks][1]);
        }
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[nh][j] += s2[nh][j];
      } else {
        constexpr int per = D / 16 / S::kBlocks;      // 16-value pieces of a scale block: 4 or 2
#pragma unroll
        for (int blk = 0; blk < S::kBlocks; ++blk) {
          float t[NH][4] = {};
#pragma unroll
          for (int x = 0; x < per; x += 2) {
            const int ks = blk * per + x;
            uint32_t f[4];
            ldsm4(f, kt + swz<S::kRow>(lr, ks + lc));
            // f[0], f[1]: rows g, g + 8 of piece ks; f[2], f[3]: of piece ks + 1
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t h0[2], h1[2];
              wm_stream::e4m3x4_to_f16x2(f[2 * y], h0);
              wm_stream::e4m3x4_to_f16x2(f[2 * y + 1], h1);
              const uint32_t fa[4] = {h0[0], h1[0], h0[1], h1[1]};
#pragma unroll
              for (int nh = 0; nh < NH; ++nh) mma_f16(t[nh], fa, qf[nh][ks + y][0], qf[nh][ks + y][1]);
            }
          }
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) {
            s[nh][0] = fmaf(t[nh][0], ka[blk], s[nh][0]);
            s[nh][1] = fmaf(t[nh][1], ka[blk], s[nh][1]);
            s[nh][2] = fmaf(t[nh][2], kb[blk], s[nh][2]);
            s[nh][3] = fmaf(t[nh][3], kb[blk], s[nh][3]);
          }
        }
      }
      if constexpr (FMT != WKV_BF16) {
        load_scales<FMT>(sc + (kTile + g) * S::kScale, va);
        load_scales<FMT>(sc + (kTile + g + 8) * S::kScale, vb);
      }
      const int key = (t0 + i * kWarps) * kTile;
      const int rows = min(kTile, len - key);
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) {
        s[nh][0] = g < rows ? s[nh][0] * sc2[nh][0] : kNegInf;
        s[nh][1] = g < rows ? s[nh][1] * sc2[nh][1] : kNegInf;
        s[nh][2] = g + 8 < rows ? s[nh][2] * sc2[nh][0] : kNegInf;
        s[nh][3] = g + 8 < rows ? s[nh][3] * sc2[nh][1] : kNegInf;
      }
      if (a.scores) {
        const int sh = a.score_heads;
        float *sp = a.scores + (pair * cap + key) * sh + i2;
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
          if (nh * 8 + i2 >= sh) continue;
          if (g < rows) *reinterpret_cast<float2 *>(sp + g * sh + nh * 8) = make_float2(s[nh][0], s[nh][1]);
          if (g + 8 < rows) *reinterpret_cast<float2 *>(sp + (g + 8) * sh + nh * 8) = make_float2(s[nh][2], s[nh][3]);
        }
      }

      // running maximum; the output is rescaled only when some head's maximum grew
      float mx[NH][2];
      bool grew = false;
#pragma unroll
      for (int nh = 0; nh < NH; ++nh)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = fmaxf(s[nh][j], s[nh][j + 2]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          mx[nh][j] = fmaxf(x, m[nh][j]);
          grew |= mx[nh][j] > m[nh][j];
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float f = mx[nh][j] > m[nh][j] ? ex2(m[nh][j] - mx[nh][j]) : 1.0f;
            l[nh][j] *= f;
            m[nh][j] = mx[nh][j];
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
              o[mt][nh][j] *= f;
              o[mt][nh][j + 2] *= f;
            }
          }
      }
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) {
        // while every score so far is -inf the weights are 2^-inf, not 2^(-inf + inf)
        const float m0 = m[nh][0] == kNegInf ? 0.0f : m[nh][0], m1 = m[nh][1] == kNegInf ? 0.0f : m[nh][1];
        s[nh][0] = ex2(s[nh][0] - m0);
        s[nh][1] = ex2(s[nh][1] - m1);
        s[nh][2] = ex2(s[nh][2] - m0);
        s[nh][3] = ex2(s[nh][3] - m1);
        l[nh][0] += s[nh][0] + s[nh][2];
        l[nh][1] += s[nh][1] + s[nh][3];
      }

      // output: rows are value dimensions, columns heads
      if constexpr (FMT == WKV_BF16) {
        uint32_t p[NH][2];
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
          p[nh][0] = transpose8(bf16x2(s[nh][0], s[nh][1]));
          p[nh][1] = transpose8(bf16x2(s[nh][2], s[nh][3]));
        }
        const int vr = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          uint32_t f[4];
          ldsm4t(f, vt + swz<S::kRow>(vr, 2 * mt + vc));
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) mma(o[mt][nh], f, p[nh][0], p[nh][1]);
        }
      } else {
        float s0[S::kBlocks], s1[S::kBlocks], big = 0.0f;
        fetch_factors();
#pragma unroll
        for (int blk = 0; blk < S::kBlocks; ++blk) {
          s0[blk] = va[blk] * factor[blk];
          s1[blk] = vb[blk] * factor[blk];
          big = fmaxf(big, fmaxf(s0[blk], s1[blk]));
        }
        if (__any_sync(0xffffffffu, big > kTopWeight)) {
          asm volatile("" ::: "memory");              // all read again: none is held in a register for this
          fetch_factors();
          load_scales<FMT>(sc + (kTile + g) * S::kScale, va);
          load_scales<FMT>(sc + (kTile + g + 8) * S::kScale, vb);
#pragma unroll
          for (int blk = 0; blk < S::kBlocks; ++blk) {
            float x = fmaxf(va[blk], vb[blk]);        // the largest scale of the block's values
#pragma unroll
            for (int y = 16; y; y >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, y));
            // to less than 2^13: a scale has to grow four times before the next change
            const bool low = x * factor[blk] > kTopWeight;
            const float next = low ? wm_stream::pow2f(139 - static_cast<int>(__float_as_uint(x) >> 23)) : factor[blk];
            const float f = low ? next * inverse(factor[blk]) : 1.0f;
            factor[blk] = next;
            s0[blk] = va[blk] * next;
            s1[blk] = vb[blk] * next;
#pragma unroll
            for (int y = 0; y < D / 16 / S::kBlocks; ++y)
#pragma unroll
              for (int nh = 0; nh < NH; ++nh)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[blk * (D / 16 / S::kBlocks) + y][nh][j] *= f;
          }
          keep_factors();
        }
        constexpr int per = D / 16 / S::kBlocks;
        const int vr = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;
#pragma unroll
        for (int blk = 0; blk < S::kBlocks; ++blk) {
          uint32_t p[NH][2];
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) {
            p[nh][0] = transpose8(wm_stream::f32x2_to_f16x2(s[nh][0] * s0[blk], s[nh][1] * s0[blk]));
            p[nh][1] = transpose8(wm_stream::f32x2_to_f16x2(s[nh][2] * s1[blk], s[nh][3] * s1[blk]));
          }
#pragma unroll
          for (int x = 0; x < per; x += 2) {
            const int mt = blk * per + x;
            uint32_t f[4];
            ldsm4t(f, vt + swz<S::kRow>(vr, mt + vc));
            // f[0], f[2]: piece mt, keys 0-7 and 8-15; f[1], f[3]: piece mt + 1.  A register holds
            // dimensions 2g, 2g + 1 of two keys: row g of the tile is dimension 2g, row g + 8 is 2g + 1
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t h0[2], h1[2];
              wm_stream::e4m3x4_to_f16x2(__byte_perm(f[y], 0u, 0x3120), h0);
              wm_stream::e4m3x4_to_f16x2(__byte_perm(f[y + 2], 0u, 0x3120), h1);
              const uint32_t fa[4] = {h0[0], h0[1], h1[0], h1[1]};
#pragma unroll
              for (int nh = 0; nh < NH; ++nh) mma_f16(o[mt + y][nh], fa, p[nh][0], p[nh][1]);
            }
          }
        }
      }
      __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // the part of this CTA: merge the four warps
#pragma unroll
    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[nh][j];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        l[nh][j] = x;
      }
    if (bad)                                          // a page out of range: the sequence's outputs are NaN
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) l[nh][0] = l[nh][1] = __uint_as_float(0x7fc00000u);
    if (g == 0)
#pragma unroll
      for (int nh = 0; nh < NH; ++nh)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sm_m[warp][nh * 8 + i2 + j] = m[nh][j];
          sm_l[warp][nh * 8 + i2 + j] = l[nh][j];
        }
    __syncthreads();                                  // all rings are drained
    float *mg = reinterpret_cast<float *>(smem);      // [warp][head][D]
    fetch_factors();
#pragma unroll
    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int hd = nh * 8 + i2 + j;
        const float top = fmaxf(fmaxf(sm_m[0][hd], sm_m[1][hd]), fmaxf(sm_m[2][hd], sm_m[3][hd]));
        const float f = m[nh][j] == kNegInf ? (n > 0 ? 1.0f : 0.0f) : ex2(m[nh][j] - top);
        float *row = mg + (warp * S::kHeads + hd) * D;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          const int d0 = FMT == WKV_BF16 ? 16 * mt + g : 16 * mt + 2 * g, d1 = FMT == WKV_BF16 ? d0 + 8 : d0 + 1;
          const float to = FMT == WKV_BF16 ? f : f * inverse(factor[mt / (D / 16 / S::kBlocks)]);
          row[d0] = o[mt][nh][j] * to;
          row[d1] = o[mt][nh][j + 2] * to;
        }
      }
    __syncthreads();
    auto merged = [&](int x) {                        // four values of the CTA's output
      const float4 *p = reinterpret_cast<const float4 *>(mg) + x;
      float4 r = p[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 y = p[w * (S::kHeads * D / 4)];
        r.x += y.x; r.y += y.y; r.z += y.z; r.w += y.w;
      }
      return r;
    };
    auto stats = [&](int hd, float &top, float &sum) {
      top = fmaxf(fmaxf(sm_m[0][hd], sm_m[1][hd]), fmaxf(sm_m[2][hd], sm_m[3][hd]));
      sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += sm_m[w][hd] == kNegInf ? sm_l[w][hd] : sm_l[w][hd] * ex2(sm_m[w][hd] - top);
    };
    if constexpr (!CL) {
      const int64_t slot = blockIdx.x + pair;
      for (int x = threadIdx.x; x < S::kHeads * D / 4; x += kWarps * 32)
        reinterpret_cast<float4 *>(a.part_o + slot * (S::kHeads * D))[x] = merged(x);
      if (threadIdx.x < S::kHeads) {
        float top, sum;
        stats(threadIdx.x, top, sum);
        a.part_m[slot * S::kHeads + threadIdx.x] = top;
        a.part_l[slot * S::kHeads + threadIdx.x] = sum;
      }
      __syncthreads();
    } else {
      // join over distributed shared memory: the CTA's output replaces its warp 0's, every CTA of the cluster
      // then adds up a share of the columns
      cg::cluster_group cluster = cg::this_cluster();
      const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
      for (int x = threadIdx.x; x < S::kHeads * D / 4; x += kWarps * 32) reinterpret_cast<float4 *>(mg)[x] = merged(x);
      if (threadIdx.x < S::kHeads) {
        float top, sum;
        stats(threadIdx.x, top, sum);
        sm_part[threadIdx.x] = make_float2(top, sum);
      }
      cluster.sync();
      const int live = min(S::kHeads, a.G - c * S::kHeads);
      const bool bad_len = a.lengths[b] < 0 || a.lengths[b] > cap;
      const float nan = __uint_as_float(0x7fc00000u);
      for (int x = rank * (kWarps * 32) + threadIdx.x; x < live * (D / 4); x += C * (kWarps * 32)) {
        const int hd = x / (D / 4);
        float top = kNegInf, sum = 0.0f;
        float2 st[kMaxCluster];
        float4 v[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < C) {
            st[r] = cluster.map_shared_rank(sm_part, r)[hd];
            v[r] = reinterpret_cast<const float4 *>(cluster.map_shared_rank(mg, r))[x];
            top = fmaxf(top, st[r].x);
          }
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < C) {
            const float f = part_factor(st[r].x, top);
            sum = fmaf(st[r].y, f, sum);
            o.x = fmaf(v[r].x, f, o.x);
            o.y = fmaf(v[r].y, f, o.y);
            o.z = fmaf(v[r].z, f, o.z);
            o.w = fmaf(v[r].w, f, o.w);
          }
        const int64_t head = static_cast<int64_t>(b) * a.Hq + h * a.G + c * S::kHeads + hd;
        const float inv = bad_len ? nan : (len > 0 ? 1.0f / sum : 0.0f);
        reinterpret_cast<uint2 *>(a.out + head * D)[x % (D / 4)] = make_uint2(bf16x2(o.x * inv, o.y * inv), bf16x2(o.z * inv, o.w * inv));
        if (a.lse && x % (D / 4) == 0) a.lse[head] = bad_len ? nan : (len > 0 ? (top + log2f(sum)) * kLn2 : kNegInf);
      }
      cluster.sync();                                 // no CTA leaves while its shared memory is read
    }
  };

  if constexpr (CL) {
    cg::cluster_group cluster = cg::this_cluster();
    const int64_t C = cluster.num_blocks(), rank = cluster.block_rank(), pair = blockIdx.x / static_cast<unsigned>(C);
    const int b = static_cast<int>(quotient(pair, PH));
    const int64_t nu = units_of(a, b);
    segment(b, static_cast<int>(pair - static_cast<int64_t>(b) * PH), quotient(nu * rank, C), quotient(nu * (rank + 1), C));
  } else {
    // this CTA's share [u, u_end) of the line of units
    const int64_t total = warp_units(a, a.B) * PH;
    const Line line(a, total);
    int64_t u = line.start(blockIdx.x);
    const int64_t u_end = line.start(blockIdx.x + 1);
    if (u >= u_end) return;
    int b = 0;
    int64_t base = 0;                                 // line position of sequence b
    for (int b0 = 0;; b0 += 32) {                     // the sequence that holds unit u
      const int64_t mine = b0 + lane < a.B ? units_of(a, b0 + lane) * PH : 0;
      int64_t s = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += o;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + s > u);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = b0 + l;
        base += __shfl_sync(0xffffffffu, s - mine, l);
        break;
      }
      base += __shfl_sync(0xffffffffu, s, 31);
    }
    while (u < u_end) {
      const int64_t nu = units_of(a, b);
      if (nu == 0 || u >= base + nu * PH) {           // next sequence
        base += nu * PH;
        ++b;
        continue;
      }
      const int hc = static_cast<int>(quotient(u - base, nu));
      const int64_t unit0 = (u - base) - hc * nu;
      const int64_t unit1 = unit0 + (u_end - u) < nu ? unit0 + (u_end - u) : nu;
      u += unit1 - unit0;
      segment(b, hc, unit0, unit1);
    }
  }
}

// Joins the parts of a pair.  Blocks (pair, group of heads) give the output; with
// a mass array blocks (pair, groups + x) add the weights of a run of keys.  A pair
// has up to one part per CTA: their factors go to shared memory first, so that the
// loads of the parts' outputs are independent of one another (a first form that
// walked the parts one by one took 9.8 us for 37 parts of 128 values).  Two forms:
// for few parts per pair 128 threads take kHpb heads, four values each; for many
// 512 threads take one head and share the parts (74 parts of 8 x 256 values took
// 8 us on 128 threads).
constexpr int kManyParts = 8;          // parts per pair from which a block takes a single head
constexpr int kKeysPerThread = 4;      // of a mass block

template <int D, int NH, int TJ, int HPB>
__global__ void __launch_bounds__(TJ) k_attn_join(DecodeArgs a, int groups) {
  constexpr int kHeads = 8 * NH, kJW = TJ / 32;
  constexpr int kCols = HPB * D / 4, kGroups = TJ / kCols;     // a thread sums 4 values over every kGroups-th part
  constexpr int kPer = TJ / HPB;                               // parts whose factors are held at once
  static_assert(kGroups >= 1 && 32 % HPB == 0, "join shape");
  __shared__ float s_f[TJ], s_top[kJW][HPB], s_sum[kJW][HPB];
  __shared__ float4 s_o[TJ];
  __shared__ float2 s_st[kJW][kHeads];
  __shared__ float s_lse2[kHeads];
  const int PH = a.pool.Hkv * a.NC;
  const int64_t pair = blockIdx.x;
  const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(PH)), hc = static_cast<int>(pair - static_cast<int64_t>(b) * PH);
  const int h = hc / a.NC, c = hc - h * a.NC;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool output = static_cast<int>(blockIdx.y) < groups;
  if (output ? c * kHeads + static_cast<int>(blockIdx.y) * HPB >= a.G : c != 0) return;
  WM_PDL_WAIT();
  const int64_t cap = static_cast<int64_t>(a.pool.max_pages) * a.pool.page_size;
  int64_t total = 0, first = 0;                       // units of all sequences, and of those before b
  for (int x = lane; x < a.B; x += 32) {
    const int64_t n = units_of(a, x);
    total += n;
    first += x < b ? n : 0;
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, m);
    first += __shfl_xor_sync(0xffffffffu, first, m);
  }
  const int64_t nu = units_of(a, b);
  total *= PH;
  first = first * PH + hc * nu;
  const int len = a.lengths[b];
  const bool bad = len < 0 || len > cap;
  const float nan = __uint_as_float(0x7fc00000u);
  const Line line(a, total);
  // CTAs that hold the nu units from `at`
  auto part0 = [&](int64_t at) { return nu ? line.cta(at) : 0; };
  auto parts = [&](int64_t at, int64_t p0) { return nu ? static_cast<int>(line.cta(at + nu - 1) - p0) + 1 : 0; };

  if (output) {
    const int64_t p00 = part0(first), slot0 = p00 + pair;
    const int hd0 = blockIdx.y * HPB, np = parts(first, p00);
    const int col = tid % kCols, grp = tid / kCols, ch = col / (D / 4);       // column: head ch, values 4 (col % (D / 4))
    const float4 *po = reinterpret_cast<const float4 *>(a.part_o + (slot0 * kHeads + hd0) * D) + col;
    constexpr int64_t kNext = kHeads * D / 4;                                  // from part to part
    // the first parts' outputs load while their factors are found
    constexpr int kAhead = 8;
    float4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int y = grp + k * kGroups;
      v[k] = y < np ? po[y * kNext] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    // thread t: head hd0 + t % HPB, part t / HPB
    const int th = tid % HPB, tp = tid / HPB;
    const float *pm = a.part_m + slot0 * kHeads + hd0 + th, *pl = a.part_l + slot0 * kHeads + hd0 + th;
    float m0 = kNegInf, l0 = 0.0f;
    if (tp < np) {
      m0 = pm[tp * kHeads];
      l0 = pl[tp * kHeads];
    }
    float top = m0;
    for (int i = tp + kPer; i < np; i += kPer) top = fmaxf(top, pm[i * kHeads]);
#pragma unroll
    for (int x = 16; x >= HPB; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if (lane < HPB) s_top[warp][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJW; ++w) top = fmaxf(top, s_top[w][th]);

    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float4 &x, float f) {
      o.x = fmaf(x.x, f, o.x);
      o.y = fmaf(x.y, f, o.y);
      o.z = fmaf(x.z, f, o.z);
      o.w = fmaf(x.w, f, o.w);
    };
    for (int p0 = 0; p0 < np; p0 += kPer) {
      const int i = p0 + tp, m = min(kPer, np - p0);
      float f = 0.0f;
      if (i < np) {
        f = part_factor(p0 ? pm[i * kHeads] : m0, top);
        sum += f * (p0 ? pl[i * kHeads] : l0);
      }
      if (p0) __syncthreads();
      s_f[tid] = f;
      __syncthreads();
      int y = grp;
      if (p0 == 0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k, y += kGroups)
          if (y < m) add(v[k], s_f[y * HPB + ch]);
      }
#pragma unroll 4
      for (; y < m; y += kGroups) add(po[(p0 + y) * kNext], s_f[y * HPB + ch]);
    }
#pragma unroll
    for (int x = 16; x >= HPB; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane < HPB) s_sum[warp][lane] = sum;
    if constexpr (kGroups > 1) s_o[tid] = o;
    __syncthreads();
    if (tid < kCols && c * kHeads + hd0 + ch < a.G) {
      sum = 0.0f;
      top = kNegInf;
#pragma unroll
      for (int w = 0; w < kJW; ++w) {
        sum += s_sum[w][ch];
        top = fmaxf(top, s_top[w][ch]);
      }
#pragma unroll
      for (int y = 1; y < kGroups; ++y) {
        const float4 v = s_o[y * kCols + tid];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
      }
      const int64_t head = static_cast<int64_t>(b) * a.Hq + h * a.G + c * kHeads + hd0 + ch;
      const int x = col % (D / 4);
      const float inv = bad ? nan : (np > 0 ? 1.0f / sum : 0.0f);
      reinterpret_cast<uint2 *>(a.out + head * D)[x] = make_uint2(bf16x2(o.x * inv, o.y * inv), bf16x2(o.z * inv, o.w * inv));
      if (a.lse && x == 0) a.lse[head] = bad ? nan : (np > 0 ? (top + log2f(sum)) * kLn2 : kNegInf);
    }
    return;
  }

  // mass: the weights of keys [k0, k1), summed over the query heads of all chunks
  constexpr int kRun = TJ * kKeysPerThread;
  const int64_t k0 = static_cast<int64_t>(blockIdx.y - groups) * kRun;
  if (bad || k0 >= len) return;
  const int64_t k1 = k0 + kRun < len ? k0 + kRun : len;
  float *mass = a.mass + (static_cast<int64_t>(b) * a.pool.Hkv + h) * cap;
  float acc[kKeysPerThread];
#pragma unroll
  for (int x = 0; x < kKeysPerThread; ++x) {
    const int64_t key = k0 + x * TJ + tid;
    acc[x] = key < k1 ? mass[key] : 0.0f;
  }
  for (int cc = 0; cc < a.NC; ++cc) {
    const int64_t at = first + cc * nu, p00 = part0(at), slot0 = p00 + pair + cc;
    const int n = parts(at, p00) * kHeads;
    const float *qm = a.part_m + slot0 * kHeads, *ql = a.part_l + slot0 * kHeads;
    // the scores load while the heads' normalisers are found
    const int live = min(kHeads, a.G - cc * kHeads);
    const float *sc = a.scores + (pair + cc) * cap * a.score_heads;
    float2 v[kKeysPerThread][kHeads / 2];
#pragma unroll
    for (int x = 0; x < kKeysPerThread; ++x) {
      const int64_t key = k0 + x * TJ + tid;
      const float2 *sp = reinterpret_cast<const float2 *>(sc + key * a.score_heads);
#pragma unroll
      for (int y = 0; y < kHeads / 2; ++y) v[x][y] = key < k1 && 2 * y < live ? sp[y] : make_float2(0.0f, 0.0f);
    }
    // thread t joins every (TJ / kHeads)-th part of head t % kHeads
    float top = kNegInf, sum = 0.0f;
#pragma unroll 4
    for (int i = tid; i < n; i += TJ) {
      const float mi = qm[i], li = ql[i], t = fmaxf(top, mi);
      sum = sum * part_factor(top, t) + li * part_factor(mi, t);
      top = t;
    }
#pragma unroll
    for (int x = 16; x >= kHeads; x >>= 1) {
      const float mi = __shfl_xor_sync(0xffffffffu, top, x), li = __shfl_xor_sync(0xffffffffu, sum, x), t = fmaxf(top, mi);
      sum = sum * part_factor(top, t) + li * part_factor(mi, t);
      top = t;
    }
    if (lane < kHeads) s_st[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (tid < kHeads) {
#pragma unroll
      for (int w = 0; w < kJW; ++w) top = fmaxf(top, s_st[w][tid].x);
      sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kJW; ++w) sum += s_st[w][tid].y * part_factor(s_st[w][tid].x, top);
      s_lse2[tid] = top + log2f(sum);
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kKeysPerThread; ++x) {
      float w = 0.0f;
#pragma unroll
      for (int y = 0; y < kHeads / 2; ++y) {
        if (2 * y < live) w += ex2(v[x][y].x - s_lse2[2 * y]);
        if (2 * y + 1 < live) w += ex2(v[x][y].y - s_lse2[2 * y + 1]);
      }
      acc[x] += w;
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < kKeysPerThread; ++x) {
    const int64_t key = k0 + x * TJ + tid;
    if (key < k1) mass[key] = acc[x];
  }
}

template <int D, int NH, int TJ, int HPB>
cudaError_t launch_join(const DecodeArgs &a, cudaStream_t stream) {
  const int64_t cap = static_cast<int64_t>(a.pool.max_pages) * a.pool.page_size;
  const int groups = (std::min(8 * NH, a.G) + HPB - 1) / HPB;
  const unsigned runs = a.mass ? static_cast<unsigned>((cap + TJ * kKeysPerThread - 1) / (TJ * kKeysPerThread)) : 0u;
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.B) * a.pool.Hkv * a.NC), groups + runs);
  return wm::launch_pdl(k_attn_join<D, NH, TJ, HPB>, grid, dim3(TJ), 0, stream, a, groups);
}

int chunk_heads(int G) { return G <= 8 ? 8 : 16; }

// CTAs the line of units is split over: what fits on the GPU at once, and no
// more than there are units when every sequence is at capacity.
template <int D, int FMT, int NH>
int grid_of(int64_t most_units) {
  using S = Shape<D, FMT, NH>;
  const int per_sm = std::max(1, std::min(4, (225 * 1024) / (S::kSmem + 1024 + 8 * S::kHeads * kWarps)));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most_units, static_cast<int64_t>(per_sm) * wm::sm_count())));
}

template <int D, int FMT, int NH>
int launch(DecodeArgs &a, cudaStream_t stream) {
  using S = Shape<D, FMT, NH>;
  if (a.cluster) {
    cudaError_t e = wm::allow_smem<k_attn_decode<D, FMT, NH, true>>(S::kSmem);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.n_cta));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(a.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, k_attn_decode<D, FMT, NH, true>, a);
    if (e != cudaSuccess) return wm::fail(WM_ERR_CUDA, std::string("wattn_decode: ") + cudaGetErrorString(e));
    return wm::check_launch("wattn_decode");
  }
  cudaError_t e = wm::allow_smem<k_attn_decode<D, FMT, NH, false>>(S::kSmem);
  if (e == cudaSuccess) e = wm::launch_pdl(k_attn_decode<D, FMT, NH, false>, dim3(a.rounds * a.n_cta), dim3(kWarps * 32), S::kSmem, stream, a);
  if (e != cudaSuccess) return wm::fail(WM_ERR_CUDA, std::string("wattn_decode: ") + cudaGetErrorString(e));
  const int64_t pairs = static_cast<int64_t>(a.B) * a.pool.Hkv * a.NC;
  const bool many = a.n_cta >= kManyParts * pairs;
  if (!many) e = launch_join<D, NH, 128, 512 / D>(a, stream);
  else if (!a.mass) e = launch_join<D, NH, 512, 1>(a, stream);
  else e = launch_join<D, NH, 128, 1>(a, stream);     // the mass blocks' registers: four 128-thread blocks per SM, one of 512
  if (e != cudaSuccess) return wm::fail(WM_ERR_CUDA, std::string("wattn_decode: ") + cudaGetErrorString(e));
  return wm::check_launch("wattn_decode");
}

// Runs f.template operator()<D, FMT, NH>() for the call's shape.
template <typename F>
auto dispatch(int D, int fmt, int G, F &&f) {
#define WM_ATTN_NH(d, x) return G <= 8 ? f.template operator()<d, x, 1>() : f.template operator()<d, x, 2>()
#define WM_ATTN_FMT(d)                                          \
  if (fmt == WKV_BF16) WM_ATTN_NH(d, WKV_BF16);                 \
  if (fmt == WKV_FP8_F32_B64) WM_ATTN_NH(d, WKV_FP8_F32_B64);   \
  WM_ATTN_NH(d, WKV_MXFP8_B32)
  if (D == 64) { WM_ATTN_FMT(64); }
  if (D == 128) { WM_ATTN_FMT(128); }
  WM_ATTN_FMT(256);
#undef WM_ATTN_FMT
#undef WM_ATTN_NH
}

struct GridOf {
  int64_t most;
  template <int D, int FMT, int NH>
  int operator()() const { return grid_of<D, FMT, NH>(most); }
};
struct Launch {
  DecodeArgs &a;
  cudaStream_t stream;
  template <int D, int FMT, int NH>
  int operator()() const { return launch<D, FMT, NH>(a, stream); }
};

struct Plan {
  int NC, heads, score_heads, n_cta, rounds, cluster;
  int64_t pairs, slots, cap;
  size_t off_m, off_l, off_s, bytes;
};

Plan plan_of(int B, int Hq, int Hkv, int D, int fmt, int page_size, int max_pages, bool with_mass) {
  Plan p{};
  const int G = Hq / Hkv;
  p.heads = chunk_heads(G);
  p.NC = (G + p.heads - 1) / p.heads;
  p.score_heads = std::min(p.heads, (G + 1) & ~1);
  p.pairs = static_cast<int64_t>(B) * Hkv * p.NC;
  p.cap = static_cast<int64_t>(max_pages) * page_size;
  // Short caches: a cluster of CTAs per pair that joins over shared memory, in one launch and without a workspace.
  // Its split is by pairs, not by the line, so it is taken while a CTA has at most kClusterKeys keys.
  p.cluster = kMaxCluster;
  while (p.cluster > 1 && p.pairs * p.cluster > 2 * wm::sm_count()) p.cluster /= 2;
  if (with_mass || p.cap > static_cast<int64_t>(kClusterKeys) * p.cluster || p.pairs * p.cluster > INT32_MAX) p.cluster = 0;
  if (p.cluster) {
    p.n_cta = static_cast<int>(p.pairs * p.cluster);
    return p;
  }
  const int64_t most = p.pairs * ((p.cap + kUnit - 1) / kUnit);
  p.n_cta = dispatch(D, fmt, G, GridOf{most});
  p.rounds = most >= static_cast<int64_t>(kTierUnits) * p.n_cta ? kTiers : 1;
  p.slots = static_cast<int64_t>(p.rounds) * p.n_cta + p.pairs;
  auto up = [](size_t x) { return (x + 255) & ~size_t{255}; };
  p.off_m = up(static_cast<size_t>(p.slots) * p.heads * D * 4);
  p.off_l = p.off_m + up(static_cast<size_t>(p.slots) * p.heads * 4);
  p.off_s = p.off_l + up(static_cast<size_t>(p.slots) * p.heads * 4);
  p.bytes = p.off_s + (with_mass ? static_cast<size_t>(p.pairs) * p.cap * p.score_heads * 4 : 0);
  return p;
}

bool shape_ok(int B, int Hq, int Hkv, int D, int fmt, int page_size, int max_pages) {
  return B > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && (D == 64 || D == 128 || D == 256) && wm_paged::is_paged_fmt(fmt) &&
         page_size > 0 && max_pages >= 0;
}

}  // namespace

extern "C" {

size_t wattn_decode_workspace_size(int B, int Hq, int Hkv, int D, int fmt, int page_size, int max_pages, int with_mass) {
  if (!shape_ok(B, Hq, Hkv, D, fmt, page_size, max_pages)) return 0;
  return plan_of(B, Hq, Hkv, D, fmt, page_size, max_pages, with_mass != 0).bytes;
}

int wattn_decode(const wm_bf16 *q, int64_t q_stride, int B, int Hq, int Hkv, int D, const void *k_cache, const void *v_cache,
                 const void *k_scales, const void *v_scales, int fmt, int n_pages, int page_size, const int32_t *page_table,
                 int max_pages, const int32_t *lengths, float scale, wm_bf16 *out, float *lse, float *mass, void *workspace,
                 size_t ws_bytes, wm_stream_t stream) {
  wm::clear_error();
  Pool pool{const_cast<void *>(k_cache), const_cast<void *>(v_cache), const_cast<void *>(k_scales),
            const_cast<void *>(v_scales), page_table, n_pages, page_size, max_pages, Hkv};
  if (int rc = wm_paged::check_pool(pool, B, D, fmt)) return rc;
  WM_REQUIRE(Hq > 0 && Hq % Hkv == 0, "decode attention: the query heads must be a multiple of the key-value heads");
  WM_REQUIRE(scale > 0.0f && scale * kLog2e <= 3.4028234663852886e38f, "decode attention: the scale must be positive and finite");
  if (B == 0) return WM_OK;
  WM_REQUIRE(q && lengths && out, "decode attention: missing input or output");
  WM_REQUIRE(q_stride >= static_cast<int64_t>(Hq) * D && q_stride % 2 == 0 && wm::aligned(q, 4) && wm::aligned(out, 8),
             "decode attention: query rows must be 4-byte aligned and hold Hq * D values, the output 8-byte aligned");
  const Plan p = plan_of(B, Hq, Hkv, D, fmt, page_size, max_pages, mass != nullptr);
  // the join's grid has a row per 512 entries of the capacity
  WM_REQUIRE(p.pairs <= INT32_MAX && (mass == nullptr || p.cap <= 512ll * 65000), "decode attention: batch or capacity too large");
  if (ws_bytes < p.bytes) return wm::fail(WM_ERR_WORKSPACE, "decode attention: workspace too small");
  WM_REQUIRE(p.bytes == 0 || (workspace && wm::aligned(workspace, 256)), "decode attention: the workspace must be 256-byte aligned");
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  DecodeArgs a{pool, q, q_stride, lengths, B, Hq, Hq / Hkv, p.NC, scale * kLog2e, out, lse, mass,
               reinterpret_cast<float *>(ws), reinterpret_cast<float *>(ws + p.off_m), reinterpret_cast<float *>(ws + p.off_l),
               mass ? reinterpret_cast<float *>(ws + p.off_s) : nullptr, p.score_heads, p.n_cta, p.rounds, p.cluster};
  return dispatch(D, fmt, a.G, Launch{a, stream});
}

}  // extern "C"
