// Paged key-value cache: append (bf16 or quantized rows) and eviction by
// accumulated attention weight.  Compiled with -fmad=false, as formats.cu: the
// quantized rows are the bytes of wkv_quantize.
#include <cooperative_groups.h>

#include <algorithm>

#include "wm_kvfp8.cuh"
#include "wm_paged.cuh"

namespace cg = cooperative_groups;
using wm_paged::Pool;

namespace {

// ------------------------------------------------------------------ append --
//
// A warp takes kFly x 32 neighbouring pieces of 16 values (two 16-byte loads per
// lane and piece, all issued first).  Its lanes then find, one token each, where
// the tokens it touches go: binary search in cu_seqlens (held in shared memory),
// length, page.  The pieces get their token's row by shuffle; a quantized row's
// scale blocks are 2 or 4 adjacent lanes, as in k_kv_fp8_quantize.  Bound by the
// waves of CTAs (2.8 of them below) and, for e4m3 rows, the quantizer's arithmetic:
// with a search per piece it took 475 instructions per 16 values, 59 % of the issue
// slots.  16,784 tokens of 2 x 256 values: bf16 rows 14.1 us (4.9 TB/s read and
// written), e4m3 with float32 scales 15.1, MXFP8 15.0, each 0.7 to 0.9 more with weights
// and positions (e4m3 22.5 with one piece per lane and a search each); 64 tokens of 8 x
// 128: 2.5 us.  Five CTAs per SM cap the registers at 48, at which the float32-scale form
// with two pieces spills 76 bytes.

constexpr int kSeqSmem = 512;          // sequences searched in shared memory

template <int FMT, int kFly>
__global__ void __launch_bounds__(256, 5) k_paged_append(const wm_bf16 *__restrict__ k, const wm_bf16 *__restrict__ v,
                                                      int64_t k_stride, int64_t v_stride, unsigned n16, unsigned per_tok,
                                                      unsigned tok_magic, int row_log2, const int32_t *__restrict__ cu, int T,
                                                      int B, const int32_t *__restrict__ lengths, Pool pool,
                                                      float *__restrict__ mass, int32_t *__restrict__ positions,
                                                      const int32_t *__restrict__ seen) {
  const bool is_v = blockIdx.y != 0;
  const wm_bf16 *src = is_v ? v : k;
  const int64_t stride = is_v ? v_stride : k_stride;
  uint8_t *cache = static_cast<uint8_t *>(is_v ? pool.v : pool.k);
  void *scales = is_v ? pool.vs : pool.ks;
  const int lane = threadIdx.x & 31;
  constexpr int G = FMT == WKV_BF16 ? 1 : wm_kv::Fp8Fmt<FMT == WKV_BF16 ? WKV_MXFP8_B32 : FMT>::kG / 2;
  const unsigned gmask = ((1u << G) - 1u) << (lane & ~(G - 1));
  const int64_t cap = static_cast<int64_t>(pool.max_pages) * pool.page_size;
  __shared__ int32_t s_cu[kSeqSmem + 1], s_len[kSeqSmem];
  const bool held = B <= kSeqSmem;
  WM_PDL_WAIT();
  WM_PDL_LAUNCH();
  if (held) {
    for (int i = threadIdx.x; i <= B; i += 256) {
      s_cu[i] = __ldg(cu + i);
      if (i < B) s_len[i] = __ldg(lengths + i);
    }
    __syncthreads();
  }
  auto cu_at = [&](int i) { return held ? s_cu[i] : __ldg(cu + i); };
  constexpr unsigned kSpan = 32u * kFly;
  const unsigned warps = gridDim.x * 8u;
  for (unsigned base = (blockIdx.x * 8u + (threadIdx.x >> 5)) * kSpan; base < n16; base += warps * kSpan) {
    const unsigned t0 = base / per_tok, off = base - t0 * per_tok;
    uint4 u[kFly][2];
#pragma unroll
    for (int x = 0; x < kFly; ++x) {
      const unsigned y = off + x * 32u + lane, t = __umulhi(y, tok_magic), c = y - t * per_tok;
      if (base + x * 32u + lane < n16) {
        const uint4 *p = reinterpret_cast<const uint4 *>(src + (t0 + t) * stride) + 2 * c;
        u[x][0] = __ldcs(p);
        u[x][1] = __ldcs(p + 1);
      }
    }
    // lane l: token t0 + l; its row for head 0, or -1
    int64_t row0 = -1;
    const int tok = static_cast<int>(t0) + lane;
    if (tok < T && __umulhi(off + kSpan - 1u, tok_magic) >= static_cast<unsigned>(lane)) {
      int lo = 0, hi = B;                              // the last b with cu[b] <= tok
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu_at(mid) <= tok) lo = mid; else hi = mid;
      }
      const int b = lo, end = cu_at(b + 1);
      const int64_t e = static_cast<int64_t>(held ? s_len[b] : __ldg(lengths + b)) - (end - tok);
      if (tok >= cu_at(b) && tok < end && e >= 0 && e < cap) {     // else behind the last sequence: not a token
        const int pi = static_cast<int>(e) / pool.page_size, slot = static_cast<int>(e) - pi * pool.page_size;
        const int page = __ldg(pool.table + static_cast<int64_t>(b) * pool.max_pages + pi);
        if (page >= 0 && page < pool.n_pages) {
          row0 = static_cast<int64_t>(page) * pool.Hkv * pool.page_size + slot;
          // by the key warp that has the token's first piece
          if (!is_v && (lane > 0 || off == 0) && (mass || positions)) {
            const int position = positions ? __ldg(seen + b) - (end - tok) : 0;
            for (int h = 0; h < pool.Hkv; ++h) {
              const int64_t at = (static_cast<int64_t>(b) * pool.Hkv + h) * cap + e;
              if (mass) mass[at] = 0.0f;
              if (positions) positions[at] = position;
            }
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kFly; ++x) {
      const unsigned y = off + x * 32u + lane, t = __umulhi(y, tok_magic), c = y - t * per_tok;
      const int64_t row = __shfl_sync(0xffffffffu, row0, t);
      if (base + x * 32u + lane >= n16 || row < 0) continue;       // the lanes of a scale block together
      const unsigned h = c >> row_log2, cr = c - (h << row_log2);
      const int64_t chunk = ((row + static_cast<int64_t>(h) * pool.page_size) << row_log2) + cr;
      if constexpr (FMT == WKV_BF16) {
        uint4 *d = reinterpret_cast<uint4 *>(cache) + 2 * chunk;
        d[0] = u[x][0];
        d[1] = u[x][1];
      } else {
        wm_kv::kv_fp8_quant<FMT, 16>(u[x], chunk, gmask, lane, cache, scales);
      }
    }
  }
}

// ------------------------------------------------------------------- evict --
//
// One CTA, or for more than 4096 entries one cluster of CTAs, per (sequence,
// head).  Every entry gets a 32-bit key whose unsigned order is (protected,
// weight); the budget-th largest key is found by a radix select of four 8-bit
// digits, its ties go to the lowest entries, and the r-th kept entry behind the
// budget moves into the r-th hole before it.  Attention does not depend on the
// order of its keys, so nothing that stays is copied, sources and destinations
// never overlap, and no move waits for another.
//
// The CTAs of a cluster hold a slice of the keys each in shared memory and add
// their digit counts over distributed shared memory: weights and positions are
// read from memory once.  256 bins rather than 2048 (three passes) because every
// CTA reads the bins of all: 8 x 8 KB took 6000 cycles a pass.  The first digit
// of positive weights falls into a few bins, so lanes with equal digits add once.
// A single CTA moves its rows itself; behind a cluster a second kernel does, over
// the whole GPU.  Bound by the latency of the selection's steps (about 15
// dependent phases) for short caches and by the moved rows for long ones: 64 heads
// of 2049 entries 10.5 us, 8 heads of 20,000 to 32,768 entries down to 4096 31 us
// (67 us when the clusters' own CTAs moved the rows one load at a time).

constexpr int kET = 512;           // threads
constexpr int kBins = 256;         // bins of a digit
constexpr int kKeySmem = 40960;    // keys held per CTA (160 KB); longer slices read them again
constexpr int kTableSmem = 2048;   // page numbers held per CTA
constexpr int kMoveCtas = 4;       // CTAs per SM of the move kernel
constexpr int kBatch = 4;          // loads in flight per thread
constexpr int kMostCtas = 8;       // CTAs of a cluster
constexpr int kPastEnd = 8192;     // an index runs less than this past the last entry
static_assert(kMostCtas * kET <= kPastEnd && 2 * kBatch * kET <= kPastEnd, "evict: indexes past the end");

struct EvictArgs {
  Pool pool;
  const int32_t *lengths, *seen;
  const float *mass;
  const int32_t *positions;
  float *mass_out;
  int32_t *positions_out, *lengths_out;
  int64_t *rows;                   // [B * Hkv][2][budget]: cache rows of the holes, then of the tails
  int32_t *lists;                  // the same for the entries' numbers
  int32_t *moves;                  // [B * Hkv]
  int budget, recent, sinks, row16_log2, scale_bytes, key_cap;
};

__device__ __forceinline__ uint32_t evict_key(float m, int32_t pos, int32_t from, int32_t sinks) {
  if (pos >= from || pos < sinks) return 0xffffffffu;
  if (m != m) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(m + 0.0f);        // -0 becomes +0
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive sum over the block's threads; *total gets the whole sum.
__device__ __forceinline__ int block_scan(int x, int *warp_sums, int *total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == 31) warp_sums[w] = s;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int j = 0; j < kET / 32; ++j) {
    const int v = warp_sums[j];
    if (j < w) base += v;
    all += v;
  }
  *total = all;
  return base + s - x;
}

// Copies rows of one scale array, `T` bytes each.
template <typename T>
__device__ __forceinline__ void move_scales(void *base, const int64_t *to, const int64_t *from, int moves, int at, int step) {
  T *p = static_cast<T *>(base);
#pragma unroll 4
  for (int r = at; r < moves; r += step) {
    const T v = p[from[r]];
    p[to[r]] = v;
  }
}

// Thread ct of CT carries out the moves of one (sequence, head).
__device__ __forceinline__ void carry_out(const EvictArgs &a, int64_t bh, int moves, int ct, int CT) {
  const int n = a.budget;
  const int64_t cap = static_cast<int64_t>(a.pool.max_pages) * a.pool.page_size;
  const int32_t *hl = a.lists + bh * 2 * n, *tl = hl + n;
  const int64_t *to = a.rows + bh * 2 * n, *from = to + n;
  for (int r = ct; r < moves; r += CT) {
    const int d = hl[r], s = tl[r];
    const float m = a.mass[bh * cap + s];
    const int32_t p = a.positions[bh * cap + s];
    a.mass_out[bh * cap + d] = m;
    a.positions_out[bh * cap + d] = p;
  }
  // 16-byte pieces of the moved rows, the key rows' then the value rows'; several loads in flight per thread
  constexpr int kFly = 8;
  const int lg = a.row16_log2;
  const int64_t items = static_cast<int64_t>(moves) << (lg + 1);
  for (int64_t j0 = ct; j0 < items; j0 += static_cast<int64_t>(kFly) * CT) {
    uint4 v[kFly];
    uint4 *dst[kFly];
#pragma unroll
    for (int x = 0; x < kFly; ++x) {
      const int64_t j = j0 + static_cast<int64_t>(x) * CT;
      dst[x] = nullptr;
      if (j < items) {
        const int r = static_cast<int>(j >> (lg + 1)), c = static_cast<int>(j) & ((2 << lg) - 1);
        uint4 *base = static_cast<uint4 *>(c >> lg ? a.pool.v : a.pool.k) + (c & ((1 << lg) - 1));
        v[x] = base[from[r] << lg];
        dst[x] = base + (to[r] << lg);
      }
    }
#pragma unroll
    for (int x = 0; x < kFly; ++x)
      if (dst[x]) *dst[x] = v[x];
  }
  if (a.scale_bytes)
    for (int x = 0; x < 2; ++x) {
      void *base = x ? a.pool.vs : a.pool.ks;
      const int at = x ? CT - 1 - ct : ct;             // the two arrays begin at different threads
      if (a.scale_bytes == 2) move_scales<uint16_t>(base, to, from, moves, at, CT);
      else if (a.scale_bytes == 4) move_scales<uint32_t>(base, to, from, moves, at, CT);
      else if (a.scale_bytes == 8) move_scales<uint2>(base, to, from, moves, at, CT);
      else move_scales<uint4>(base, to, from, moves, at, CT);
    }
}

__global__ void __launch_bounds__(256) k_paged_move(EvictArgs a) {
  WM_PDL_WAIT();
  const int moves = a.moves[blockIdx.x];
  carry_out(a, blockIdx.x, moves, static_cast<int>(blockIdx.y * blockDim.x + threadIdx.x), static_cast<int>(gridDim.y * blockDim.x));
}

__global__ void __launch_bounds__(kET) k_paged_evict(EvictArgs a) {
  extern __shared__ uint32_t sk[];                     // [key_cap] keys of this CTA's slice
  __shared__ uint32_t hist[2][kBins];
  __shared__ int32_t stab[kTableSmem];
  __shared__ int warp_sums[kET / 32];
  __shared__ int counts[3];                            // this CTA's ties, holes, tails
  __shared__ int pick[2];                              // chosen digit, keys above it
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), C = static_cast<int>(cluster.num_blocks());
  auto sync_all = [&] {
    if (C > 1) cluster.sync();
    else __syncthreads();
  };
  const int bh = static_cast<int>(blockIdx.x) / C, b = bh / a.pool.Hkv, h = bh - b * a.pool.Hkv;
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t cap = static_cast<int64_t>(a.pool.max_pages) * a.pool.page_size;
  WM_PDL_WAIT();
  WM_PDL_LAUNCH();
  const int len = a.lengths[b];
  const int n = a.budget;
  const int32_t *table = a.pool.table + static_cast<int64_t>(b) * a.pool.max_pages;
  const float *mass = a.mass + bh * cap;
  const int32_t *pos = a.positions + bh * cap;
  float *mass_out = a.mass_out + bh * cap;
  int32_t *pos_out = a.positions_out + bh * cap;

  // a length or a page out of range leaves the sequence as it is
  bool bad = len < 0 || len > cap;
  const int np = bad ? 0 : (len + a.pool.page_size - 1) / a.pool.page_size;
#pragma unroll 4
  for (int i = tid; i < np; i += kET) {
    const int p = table[i];
    bad |= p < 0 || p >= a.pool.n_pages;
    if (i < kTableSmem) stab[i] = p;
  }
  bad = __syncthreads_or(bad);
  const int live = bad ? (len < 0 ? 0 : static_cast<int>(len < cap ? len : cap)) : len;
  const bool copy = mass_out != mass;
  if (bad || len <= n) {
    if (copy)
      for (int i = rank * kET + tid; i < live; i += C * kET) {
        mass_out[i] = mass[i];
        pos_out[i] = pos[i];
      }
    if (h == 0 && rank == 0 && tid == 0) a.lengths_out[b] = len;
    if (rank == 0 && tid == 0) a.moves[bh] = 0;
    return;                                            // every CTA of the cluster returns here together
  }
  if (h == 0 && rank == 0 && tid == 0) a.lengths_out[b] = n;

  // this CTA's slice of the entries
  const int S = ((len + C - 1) / C + 3) & ~3;
  const int s0 = min(rank * S, len), s1 = min(s0 + S, len);
  const int32_t from = a.seen[b] - a.recent;
  const bool held = S <= a.key_cap;
  auto key_at = [&](int i) { return held ? sk[i - s0] : evict_key(mass[i], pos[i], from, a.sinks); };
  if (tid < kBins) hist[0][tid] = 0u;
  __syncthreads();
  for (int i0 = s0; i0 < s1; i0 += kBatch * kET) {
    float m[kBatch];
    int32_t p[kBatch];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int i = i0 + x * kET + tid;
      m[x] = i < s1 ? mass[i] : 0.0f;
      p[x] = i < s1 ? pos[i] : 0;
    }
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int i = i0 + x * kET + tid;
      const uint32_t key = evict_key(m[x], p[x], from, a.sinks);
      const unsigned in = __ballot_sync(0xffffffffu, i < s1);
      if (i < s1) {
        if (held) sk[i - s0] = key;
        if (copy && i < n) {                           // a hole's copy is replaced after the last barrier
          mass_out[i] = m[x];
          pos_out[i] = p[x];
        }
        const unsigned same = __match_any_sync(in, key >> 24);
        if (lane == __ffs(same) - 1) atomicAdd(&hist[0][key >> 24], static_cast<uint32_t>(__popc(same)));
      }
    }
  }

  // radix select of the n-th largest key
  uint32_t prefix = 0u, mask = 0u;
  int need = n;
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    uint32_t *hc = hist[pass & 1];
    if (pass > 0)
      for (int i = s0 + tid; i < s1; i += kET) {
        const uint32_t key = key_at(i);
        if ((key & mask) == prefix) atomicAdd(&hc[(key >> shift) & 255u], 1u);
      }
    sync_all();
    if (pass < 3 && tid < kBins) hist[(pass + 1) & 1][tid] = 0u;     // last read two barriers ago
    int count = 0;                                     // thread t < 256: bin 255 - t, over the cluster
    if (tid < kBins) {
#pragma unroll 8
      for (int r = 0; r < C; ++r) count += static_cast<int>(cluster.map_shared_rank(hc, r)[kBins - 1 - tid]);
    }
    int total;
    const int before = block_scan(count, warp_sums, &total);
    if (before < need && need <= before + count) {
      pick[0] = kBins - 1 - tid;
      pick[1] = before;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(pick[0]) << shift;
    mask |= 255u << shift;
    need -= pick[1];
  }
  // keys above prefix stay, and the first `need` entries whose key is prefix

  // Sums of counts[which] over the CTAs before this one and over all, by every warp.
  auto across = [&](int which, int &before, int &all) {
    const int v = lane < C ? *cluster.map_shared_rank(&counts[which], lane) : 0;
    int x = lane < rank ? v : 0, y = v;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      x += __shfl_xor_sync(0xffffffffu, x, d);
      y += __shfl_xor_sync(0xffffffffu, y, d);
    }
    before = x;
    all = y;
  };
  // ranks: each thread walks a run of consecutive entries
  const int E = (s1 - s0 + kET - 1) / kET;
  const int r0 = min(s0 + tid * E, s1), r1 = r0 + min(E, s1 - r0);
  int ties = 0;
  for (int i = r0; i < r1; ++i) ties += key_at(i) == prefix;
  int total, before, all, tie0 = block_scan(ties, warp_sums, &total);
  if (tid == 0) counts[0] = total;
  sync_all();
  across(0, before, all);
  tie0 += before;
  int holes = 0, tails = 0, tr = tie0;
  for (int i = r0; i < r1; ++i) {
    const uint32_t key = key_at(i);
    const bool keep = key > prefix || (key == prefix && tr++ < need);
    holes += i < n && !keep;
    tails += i >= n && keep;
  }
  int hole0 = block_scan(holes, warp_sums, &total);
  if (tid == 0) counts[1] = total;
  int tail0 = block_scan(tails, warp_sums, &total);
  if (tid == 0) counts[2] = total;
  sync_all();
  int moves;
  across(1, before, moves);
  hole0 += before;
  across(2, before, all);
  tail0 += before;
  int32_t *hl = a.lists + static_cast<int64_t>(bh) * 2 * n, *tl = hl + n;
  int64_t *hole_rows = a.rows + static_cast<int64_t>(bh) * 2 * n, *tail_rows = hole_rows + n;
  auto row_of = [&](int e) {
    const int pi = e / a.pool.page_size;
    return (static_cast<int64_t>(pi < kTableSmem ? stab[pi] : table[pi]) * a.pool.Hkv + h) * a.pool.page_size + (e - pi * a.pool.page_size);
  };
  tr = tie0;
  for (int i = r0; i < r1; ++i) {
    const uint32_t key = key_at(i);
    const bool keep = key > prefix || (key == prefix && tr++ < need);
    if (i < n && !keep) {
      hl[hole0] = i;
      hole_rows[hole0++] = row_of(i);
    }
    if (i >= n && keep) {
      tl[tail0] = i;
      tail_rows[tail0++] = row_of(i);
    }
  }
  if (rank == 0 && tid == 0) a.moves[bh] = moves;
  sync_all();                                          // also: no CTA leaves while its counts are read
  if (C == 1) carry_out(a, bh, moves, tid, kET);
}

}  // namespace

extern "C" {

int wkv_paged_append(const wm_bf16 *k, const wm_bf16 *v, int64_t k_stride, int64_t v_stride, const int32_t *cu_seqlens,
                     int T, int B, int Hkv, int D, void *k_cache, void *v_cache, void *k_scales, void *v_scales, int fmt,
                     int n_pages, int page_size, const int32_t *page_table, int max_pages, const int32_t *lengths,
                     float *mass, int32_t *positions, const int32_t *seen, wm_stream_t stream) {
  wm::clear_error();
  const Pool pool{k_cache, v_cache, k_scales, v_scales, page_table, n_pages, page_size, max_pages, Hkv};
  if (int rc = wm_paged::check_pool(pool, B, D, fmt)) return rc;
  WM_REQUIRE(T >= 0, "paged append: negative token count");
  if (T == 0 || B == 0) return WM_OK;
  WM_REQUIRE(k && v && cu_seqlens && lengths, "paged append: missing input");
  WM_REQUIRE(k_stride >= static_cast<int64_t>(Hkv) * D && v_stride >= static_cast<int64_t>(Hkv) * D && k_stride % 8 == 0 &&
                 v_stride % 8 == 0 && wm::aligned(k, 16) && wm::aligned(v, 16),
             "paged append: token rows must be 16-byte aligned and hold Hkv * D values");
  WM_REQUIRE(!positions || seen, "paged append: positions need the sequences' token counts");
  const int row_log2 = D == 64 ? 2 : (D == 128 ? 3 : 4);           // pieces of a row
  WM_REQUIRE(Hkv <= 4096, "paged append: at most 4096 heads");
  const unsigned per_tok = static_cast<unsigned>(Hkv) << row_log2;
  // x / per_tok = umulhi(x, magic) for x * per_tok < 2^32; the kernel divides numbers below per_tok + 128
  const unsigned magic = static_cast<unsigned>((1ull << 32) / per_tok + 1);
  const int64_t pieces = static_cast<int64_t>(T) * per_tok;
  WM_REQUIRE(pieces <= INT32_MAX, "paged append: too many values in one call");
  const unsigned n16 = static_cast<unsigned>(pieces);
  // several pieces per lane once that leaves every SM with work; a small call spreads over the SMs instead
  const bool many = pieces >= 2ll * 256 * wm::sm_count();
  const int64_t want = (pieces + (many ? 511 : 255)) / (many ? 512 : 256);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(want, static_cast<int64_t>(wm::sm_count()) * 16)), 2);
  cudaError_t err = cudaSuccess;
#define WM_APPEND(F)                                                                                                    \
  err = wm::launch_pdl(many ? k_paged_append<F, 2> : k_paged_append<F, 1>, grid, dim3(256), 0, stream, k, v, k_stride,  \
                       v_stride, n16, per_tok, magic, row_log2, cu_seqlens, T, B, lengths, pool, mass, positions, seen)
  if (fmt == WKV_BF16) WM_APPEND(WKV_BF16);
  else if (fmt == WKV_FP8_F32_B64) WM_APPEND(WKV_FP8_F32_B64);
  else WM_APPEND(WKV_MXFP8_B32);
#undef WM_APPEND
  if (err != cudaSuccess) return wm::fail(WM_ERR_CUDA, std::string("wkv_paged_append: ") + cudaGetErrorString(err));
  return wm::check_launch("wkv_paged_append");
}

size_t wkv_evict_workspace_size(int B, int Hkv, int budget) {
  if (B <= 0 || Hkv <= 0 || budget <= 0) return 0;
  return static_cast<size_t>(B) * Hkv * (2 * static_cast<size_t>(budget) * (sizeof(int64_t) + sizeof(int32_t)) + sizeof(int32_t));
}

int wkv_paged_evict(int B, int Hkv, int D, void *k_cache, void *v_cache, void *k_scales, void *v_scales, int fmt, int n_pages,
                    int page_size, const int32_t *page_table, int max_pages, const int32_t *lengths, const int32_t *seen,
                    const float *mass, const int32_t *positions, int budget, int recent, int sinks, float *mass_out,
                    int32_t *positions_out, int32_t *lengths_out, void *workspace, size_t ws_bytes, wm_stream_t stream) {
  wm::clear_error();
  const Pool pool{k_cache, v_cache, k_scales, v_scales, page_table, n_pages, page_size, max_pages, Hkv};
  if (int rc = wm_paged::check_pool(pool, B, D, fmt)) return rc;
  WM_REQUIRE(budget > 0 && recent >= 0 && sinks >= 0 && static_cast<int64_t>(recent) + sinks <= budget,
             "evict: the budget must be positive and hold the recent and the first positions");
  const int64_t cap = static_cast<int64_t>(max_pages) * page_size;
  // the kernel counts entries in 32 bits: its indexes run up to a round of all threads' loads, or a page, past the last one
  WM_REQUIRE(cap + page_size + kPastEnd <= INT32_MAX, "evict: the capacity and a page must stay 8192 entries below 2^31");
  if (B == 0) return WM_OK;
  WM_REQUIRE(lengths && seen && mass && positions && mass_out && positions_out && lengths_out, "evict: missing array");
  WM_REQUIRE(lengths_out != lengths, "evict: the new lengths need an array of their own");
  WM_REQUIRE((mass_out == mass) == (positions_out == positions), "evict: weights and positions are both in place or both not");
  const int n = static_cast<int>(std::min<int64_t>(budget, std::max<int64_t>(cap, 1)));
  if (ws_bytes < wkv_evict_workspace_size(B, Hkv, n)) return wm::fail(WM_ERR_WORKSPACE, "evict: workspace too small");
  WM_REQUIRE(workspace && wm::aligned(workspace, 8), "evict: the workspace must be 8-byte aligned");
  const int64_t heads = static_cast<int64_t>(B) * Hkv;
  // CTAs per (sequence, head): enough to fill the GPU, at least 2048 entries each, at most a portable cluster; up
  // to 4096 entries one CTA, whose barriers are cheaper than a cluster's and which needs no second launch
  int C = 1;
  while (cap > 4096 && C < kMostCtas && heads * C * 2 <= 2 * wm::sm_count() && cap > 2048 * C) C *= 2;
  const int64_t slice = ((cap + C - 1) / C + 3) & ~int64_t{3};
  const int key_cap = static_cast<int>(std::min<int64_t>(slice, kKeySmem));
  const size_t smem = static_cast<size_t>(key_cap) * 4;
  WM_REQUIRE(heads * C <= INT32_MAX, "evict: too many sequences");
  cudaError_t e = wm::allow_smem<k_paged_evict>(kKeySmem * 4);
  if (e != cudaSuccess) return wm::fail(WM_ERR_CUDA, std::string("wkv_paged_evict: ") + cudaGetErrorString(e));
  int64_t *rows = static_cast<int64_t *>(workspace);
  int lg = 0;
  while ((16 << lg) < wm_paged::row_bytes(fmt, D)) ++lg;
  const EvictArgs args{pool, lengths, seen, mass, positions, mass_out, positions_out, lengths_out, rows,
                       reinterpret_cast<int32_t *>(rows + heads * 2 * n), reinterpret_cast<int32_t *>(rows + heads * 3 * n), n,
                       recent, sinks, lg, wm_paged::scale_bytes(fmt, D), key_cap};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(heads * C));
  cfg.blockDim = dim3(kET);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(C);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, k_paged_evict, args);
  if (e == cudaSuccess && C > 1) {
    const int64_t per = std::max<int64_t>(1, std::min<int64_t>(kMoveCtas * wm::sm_count() / heads, (static_cast<int64_t>(n) << (lg + 1)) / 256));
    e = wm::launch_pdl(k_paged_move, dim3(static_cast<unsigned>(heads), static_cast<unsigned>(per)), dim3(256), 0, stream, args);
  }
  if (e != cudaSuccess) return wm::fail(WM_ERR_CUDA, std::string("wkv_paged_evict: ") + cudaGetErrorString(e));
  return wm::check_launch("wkv_paged_evict");
}

}  // extern "C"
