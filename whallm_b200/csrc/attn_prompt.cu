// Attention of packed prompts: grouped heads, causal (aligned at the end, so new
// tokens may continue a longer history) or full, on the 5th-generation tensor
// cores.
//
//   row i of a sequence with nq rows and nk keys sees the keys j <= i + nk - nq
//   (causal) or all nk;  s_j = scale q.k_j,  lse = log sum_j exp(s_j),
//   out = sum_j exp(s_j - lse) v_j;  a row that sees no key: out 0, lse -inf.
//
// Rows.  The query heads of one key-value head are packed with the tokens: packed
// row R is token R / G, head R % G of the group.  A work item is kRows packed
// rows of one (sequence, key-value head): with G = 8 a block of 256 rows is 32
// tokens, so short prompts fill whole tiles, K and V are read once for all query
// heads, and the two tiles of a block end at (almost) the same key.
//
// One pass over the keys with a running maximum and sum per row (32 bits).  Step
// s of an item is: S = Q K^T (tcgen05, both operands from shared memory) into one
// of two TMEM buffers; a softmax warpgroup, one thread per row, reads its row,
// writes P = exp2(S scale log2e - m) as bf16 over S; O += P V with P from TMEM.
// Up to D = 128 the block has two tiles of 128 rows and step s works on tile
// s & 1 (two softmax warpgroups in turn, each with its own O).  At D = 256, where
// TMEM holds one O of 256 columns, and for sequences of few rows the block has one
// tile, step s takes the s-th key tile and the two warpgroups hand the running
// maximum to each other.
// The MMA warp issues PV(s), S(s + 2), PV(s + 1), ...: instructions of one thread
// execute in order, so S(s + 2) may overwrite the buffer that PV(s) read.
//
// The reference point m of a row moves only when its maximum grows by more than
// 2^8 (P then stays below 2^8, harmless in bf16 and in 32-bit sums): O is rescaled
// in TMEM a few times per item instead of once per step, by the softmax threads
// themselves.  P is rounded to bf16 once, the type of V; the sum adds the
// unrounded values.
//
// Keys and values come by TMA in the 128-byte swizzle, K with D along the rows
// (K-major), V with the keys along the rows (its MN-major operand form, no
// transpose anywhere).  Tiles with keys that some row of the block does not see
// are special in V only: a hidden key has P = 0, but 0 times a value that is not
// finite is NaN.  Two helper warps therefore clear, in those tiles, the rows
// behind the sequence's end (another sequence's values) and every value that is
// not finite; such values (there are none in a healthy model) are added to the
// rows that do see them at the end.  The check hides under the step's softmax.
//
// Few rows on many keys.  Where the blocks do not fill the GPU their keys are split
// into parts (find_item), each of which leaves its reference point, sum and
// unnormalised output in a workspace; a second kernel joins them.
//
// Measured (events, back to back): 8192 tokens without a mask, 32/8 heads, D = 64
// 730 us (750 TF/s), D = 128 845 us (1300 TF/s), 16/2 heads, D = 256 795 us (1380
// TF/s; cuBLAS sustains 1406 on the same GPU); causal 16384 tokens 1450, 1715 and
// 1635 us.  D = 128 and 256 are bound by the tensor pipe and the power limit, D = 64
// by the exp2 unit (16 per cycle and SM: 2048 of the 3200 cycles of two steps) and
// the issue of its short MMAs; many short sequences by the 4 us between a block's
// last product and the next block's (1 PV, 1.5 output, the rest the first S and
// its softmax).
#include <algorithm>
#include <type_traits>

#include "wm_giveup.cuh"
#include "wm_tc.cuh"

namespace {

using wm_tc::elect_one;
using wm_tc::mbar_arrive;
using wm_tc::mbar_expect_tx;
using wm_tc::mbar_init;
using wm_tc::smem_u32;
using wm_tc::tc_commit;
using wm_tc::tc_fence_after;
using wm_tc::tc_fence_before;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kSlack = 8.0f;          // growth of a row's maximum (log2) before it is rescaled
constexpr int kThreads = 384;           // two softmax warpgroups, one warpgroup of TMA, MMA and two helper warps
constexpr int kHelpers = 64;

struct PromptArgs {
  const wm_bf16 *q, *v;
  int64_t q_stride, v_stride;
  const int32_t *cu_q, *cu_k;
  int B, Tq, Tk, Hq, Hkv, G, causal;
  int q_tma;                // G divides 128: a tile of packed rows is one box of q
  float scale2;
  wm_bf16 *out;
  float *lse;
  // few blocks on long histories: their keys are split, item x leaves its sums in slot x
  int slots, sms;           // work items at most, 0: no block is split; SMs
  float *part_o;            // [slots, kRows, D]
  float2 *part_ml;          // [slots, kRows]: reference point (log2) and sum
};

constexpr int kLeastTiles = 2;          // key tiles of a part
constexpr int kSplitKeys = 2048;        // fewer keys in all, or half of it per sequence, are not split

// ONE: one tile of 128 rows, which the warpgroups share, in place of two
template <int D, bool ONE>
struct Cfg {
  static constexpr bool kChain = ONE;
  static constexpr int kTiles = kChain ? 1 : 2;       // 128-row tiles of a block
  static constexpr int kRows = 128 * kTiles;
  static constexpr int kN = 128;                      // keys of a tile
  static constexpr int kQBytes = kRows * D * 2;
  // K and V tiles come in pieces of one slot: at D = 256 two, half of the dimensions of K or half of the keys of V
  static constexpr int kParts = D == 256 ? 2 : 1;
  static constexpr int kSlot = kN * D * 2 / kParts;
  static constexpr int kSlots = D == 64 ? 8 : 5;
  static constexpr int kKDims = D / kParts, kVKeys = kN / kParts;
  static constexpr int kKPanel = kN * 128, kVPanel = kVKeys * 128;   // 64 dimensions of a piece
  static constexpr int kOCol = 2 * kN;                // TMEM: two S / P buffers, then O
};

// One block of packed rows of one (sequence, key-value head).
struct Item {
  int valid;                // 0: no more work
  int q0, k0;               // first row of the sequence, first key of the item
  int nq, nk, skip;         // rows and keys of the sequence, its keys before the item's
  int h, blk;
  int tiles, first;         // key tiles; the first of them that holds a key some row does not see
  int part, parts, slot;    // of the block's keys; where the part's sums go
  uint32_t odd[16];         // keys of tiles first .. first + 3 with values that are not finite (128 bits each)
};

struct Bars {
  uint64_t item_full[2], item_empty[2], odd_ready[2];
  uint64_t q_full[2], q_empty[2], next_full;          // per 128-row tile
  // an edge tile (values that some row does not see) lands on v_edge, not kv_full: the helpers wait for it, and the
  // MMA warp for v_fixed.  Both advance only with edge tiles, so a phase cannot pass unseen
  uint64_t kv_full[8], kv_empty[8], v_edge[8], v_fixed[8];
  uint64_t s_full[2], p_half[2], p_ready[2], o_done[2], m_ready[2], o_free, both;
  uint64_t mma_end;                                   // the MMAs of a CTA that gives up
};

struct Shared {
  uint4 next;               // answer to the request for another work item
  Bars bar;
  Item item[2];
  uint32_t tmem;
  int abort;
  float m[128], l[2][128];  // D = 256: shared reference points, and each warpgroup's sums at the end
};

// The tiles need 1024-byte alignment: the kernel has no static shared memory, so
// its dynamic part begins at such an address (else the call ends with NaN).
template <int D, bool ONE>
constexpr int smem_bytes() { return Cfg<D, ONE>::kQBytes + Cfg<D, ONE>::kSlots * Cfg<D, ONE>::kSlot + static_cast<int>(sizeof(Shared)); }
static_assert(smem_bytes<128, false>() <= 232448 && smem_bytes<128, true>() <= 232448 && smem_bytes<256, true>() <= 232448, "shared memory of a CTA");

// try_wait without a suspend hint: with the hint of the other kernels' waits a
// warp saw a completed phase 400 to 500 cycles late, which is on the critical
// path here twice per step.
__device__ __forceinline__ bool try_wait(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// A last bounded wait, for what is still in flight when the others gave up.
__device__ __forceinline__ void drain(uint64_t *bar, uint32_t parity) {
  for (int tries = 0; tries < 1000 && !wm_tc::mbar_try(bar, parity); ++tries) {}
}

// Bounded wait of a whole warp: all its lanes return the same answer.  A wait
// that runs out makes every other wait of the CTA end, too.
__device__ __forceinline__ bool wait(Shared *sh, uint64_t *bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
  const unsigned long long t0 = wm_tc::gtimer();
  while (true) {
    for (int i = 0; i < 64; ++i)
      if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
    const bool late = wm_tc::gtimer() - t0 > wm_tc::kWaitNs;
    if (late) *reinterpret_cast<volatile int *>(&sh->abort) = 1;
    if (__any_sync(0xffffffffu, late || *reinterpret_cast<volatile int *>(&sh->abort) != 0)) return false;
  }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Shared memory operands by the low half of their descriptors (start address,
// panel distance); the high half, 8-row groups 1024 B apart in the 128-byte
// swizzle, is the same for all.  K-major: rows of 128 B, 16 values further along
// K are 32 B.  MN-major (V): rows of 64 values along MN, panels of 64 MN values
// kPanel apart, 16 keys further along K are 2048 B.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t saddr, uint32_t panel) { return ((saddr & 0x3FFFFu) >> 4) | ((panel >> 4) << 16); }

// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}

// kind::f16 instruction descriptor: bf16 x bf16 -> f32, M = 128; B MN-major for PV
__host__ __device__ constexpr uint32_t idesc_bf16(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

#define WM_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define WM_U8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])

__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : WM_R8(r, 0), WM_R8(r, 8), WM_R8(r, 16), WM_R8(r, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      WM_U8(r, 0), WM_U8(r, 8), WM_U8(r, 16), WM_U8(r, 24)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void store32(void *p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), WM_U8(r, 0) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Keys that packed row R of a block sees (0 for rows behind the sequence).
__device__ __forceinline__ int visible(const PromptArgs &a, int nq, int nk, int R) {
  const int i = R / a.G;
  if (!a.causal) return nk;
  const int n = i + 1 + nk - nq;
  return n < 0 ? 0 : (n < nk ? n : nk);
}

__device__ __forceinline__ void seq_bounds(const PromptArgs &a, int b, int &q0, int &nq, int &k0, int &nk) {
  q0 = min(max(a.cu_q[b], 0), a.Tq);
  nq = max(min(a.cu_q[b + 1], a.Tq) - q0, 0);
  k0 = min(max(a.cu_k[b], 0), a.Tk);
  nk = max(min(a.cu_k[b + 1], a.Tk) - k0, 0);
}

// Position of value tile j among the 2 n tiles of an item, which come in the order
// in which the MMA warp needs them.
template <bool ONE>
__device__ __forceinline__ int pos_v(int j, int n) { return ONE ? (j == n - 1 ? 2 * n - 1 : 2 * j + 2) : 2 * j + 1; }

// Work items are the blocks of the grid: a CTA that has started its item asks the
// hardware for a block that has not been launched yet and takes its number over
// (cluster launch control), so items are handed out in order to whoever is free,
// without a counter in memory.
__device__ __forceinline__ void ask_next(Shared *sh) {
  mbar_expect_tx(&sh->bar.next_full, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(&sh->next)),
               "r"(smem_u32(&sh->bar.next_full))
               : "memory");
}
// The block number taken over, or -1 if none was left.
__device__ __forceinline__ int read_next(Shared *sh) {
  uint32_t got, x = 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(smem_u32(&sh->next))
      : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the next answer overwrites this one
  return got ? static_cast<int>(x) : -1;
}

// Work item number x by one warp: blocks of all sequences from the last block of
// the last sequence backwards (within a causal sequence the longest first), heads
// innermost.
//
// SP: blocks are split over their keys, every block of a sequence into the same
// number of equal parts of at most c key tiles.  With c = (all blocks' tiles) /
// (SMs - blocks) there are at most as many parts as SMs, in whatever proportions
// the sequences' lengths stand: one wave.  With more blocks than half of the SMs
// the divisor stays there: equal blocks are then not split (two waves of halves
// take as long), and long ones among short ones are cut down to twice the mean load.
template <int D, bool ONE, bool SP>
__device__ __forceinline__ void find_item(const PromptArgs &a, int x, Item *out) {
  using C = Cfg<D, ONE>;
  const int lane = threadIdx.x & 31;
  auto blocks = [&](int nq) { return (static_cast<unsigned>(nq) * static_cast<unsigned>(a.G) + (C::kRows - 1)) / C::kRows; };
  auto key_tiles = [&](int nk) { return (static_cast<unsigned>(nk) + (C::kN - 1)) / C::kN; };
  unsigned c = 1u;
  if constexpr (SP) {
    int64_t nb = 0, nt = 0;
    for (int b = x < 0 ? a.B : lane; b < a.B; b += 32) {
      int q0, nq, k0, nk;
      seq_bounds(a, b, q0, nq, k0, nk);
      nb += blocks(nq);
      nt += static_cast<int64_t>(blocks(nq)) * key_tiles(nk);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      nb += __shfl_xor_sync(0xffffffffu, nb, d);
      nt += __shfl_xor_sync(0xffffffffu, nt, d);
    }
    const int64_t room = max(max(a.sms - nb * a.Hkv, static_cast<int64_t>(a.sms / 2)), static_cast<int64_t>(1));
    c = static_cast<unsigned>(max((nt * a.Hkv + room - 1) / room, static_cast<int64_t>(kLeastTiles)));
  }
  unsigned blk = static_cast<unsigned>(x) / static_cast<unsigned>(a.Hkv);
  const int h = static_cast<int>(static_cast<unsigned>(x) - blk * static_cast<unsigned>(a.Hkv));
  for (int hi = x < 0 ? 0 : a.B; hi > 0; hi -= 32) {  // lane l: sequence hi - 1 - l
    const int b = hi - 1 - lane;
    int q0 = 0, nq = 0, k0 = 0, nk = 0;
    if (b >= 0) seq_bounds(a, b, q0, nq, k0, nk);
    unsigned parts = 1u;
    if constexpr (SP) parts = min(max((key_tiles(nk) + c - 1u) / c, 1u), static_cast<unsigned>(a.slots));
    unsigned s = blocks(nq) * parts;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned o = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += o;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, s > blk);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        int k = static_cast<int>(s - 1 - blk);        // block within the sequence, last first
        unsigned part = 0u;
        if constexpr (SP) {
          part = static_cast<unsigned>(k) % parts;
          k = static_cast<int>(static_cast<unsigned>(k) / parts);
        }
        const int R0 = k * C::kRows;
        const int R1 = min(R0 + C::kRows, nq * a.G) - 1;
        const int n0 = visible(a, nq, nk, R0), n1 = visible(a, nq, nk, R1);
        int j0 = 0, j1 = (n1 + C::kN - 1) / C::kN, first = n0 / C::kN;
        if constexpr (SP) {
          const unsigned n = static_cast<unsigned>(j1), each = n / parts, more = n % parts;   // the first `more` parts have one more
          j0 = static_cast<int>(part * each + min(part, more));
          j1 = j0 + static_cast<int>(each + (part < more ? 1u : 0u));
          first = max(first - j0, 0);
        }
        out->valid = 1;
        out->q0 = q0;
        out->k0 = k0 + j0 * C::kN;
        out->nq = nq;
        out->nk = nk;
        out->skip = j0 * C::kN;
        out->h = h;
        out->blk = k;
        out->tiles = j1 - j0;
        out->first = first;
        out->part = static_cast<int>(part);
        out->parts = static_cast<int>(parts);
        out->slot = x;
      }
      if (lane < 16) out->odd[lane] = 0u;
      return;
    }
    blk -= __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) out->valid = 0;                      // x < 0 or past the last block
}

template <int D, bool ONE, bool SP>
__global__ void __launch_bounds__(kThreads, 1)
    k_attn_prompt(PromptArgs a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v) {
  using C = Cfg<D, ONE>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Shared &sh = *reinterpret_cast<Shared *>(smem + C::kQBytes + C::kSlots * C::kSlot);
  const uint32_t q_s = smem_u32(smem), kv_s = q_s + C::kQBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    Bars &b = sh.bar;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b.item_full[i], 1);
      mbar_init(&b.item_empty[i], 8 + 1 + 2);         // softmax, MMA and helper warps
      mbar_init(&b.odd_ready[i], kHelpers);
      mbar_init(&b.q_full[i], a.q_tma ? 1 : kHelpers);
      mbar_init(&b.q_empty[i], 1);
      mbar_init(&b.s_full[i], 1);
      mbar_init(&b.p_half[i], 128);
      mbar_init(&b.p_ready[i], 128);
      mbar_init(&b.o_done[i], 1);
      mbar_init(&b.m_ready[i], 128);
    }
    mbar_init(&b.next_full, 1);
    mbar_init(&b.o_free, 256);
    mbar_init(&b.both, 256);
    mbar_init(&b.mma_end, 1);
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&b.kv_full[i], 1);
      mbar_init(&b.kv_empty[i], 1);
      mbar_init(&b.v_edge[i], 1);
      mbar_init(&b.v_fixed[i], kHelpers);
    }
    sh.abort = (smem_u32(smem) & 1023u) != 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8 && lane == 0) {
    for (const CUtensorMap *m : {&map_q, &map_k, &map_v})
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  Bars &bar = sh.bar;
  WM_PDL_WAIT();                                      // the set-up above overlaps the end of the kernel before

  if (sh.abort) {
  } else if (warp >= 8) {
    // 384 threads at 168 registers are launched: 256 x 208 + 128 x 88 is the same sum
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      // ------------------------------------------------- items and TMA loads
      uint32_t g = 0u;                                // pieces loaded so far
      uint32_t asked = 0u;                            // requests for another item
      uint32_t edge_ph = 0u, edge_last = 0u;          // per slot: phase of v_edge, and whether the last load was an edge tile
      int it = 0;
      for (int x = static_cast<int>(blockIdx.x);; ++it) {
        const int sl = it & 1;
        if (!wait(&sh, &bar.item_empty[sl], ((it >> 1) & 1) ^ 1)) break;
        Item *item = &sh.item[sl];
        find_item<D, ONE, SP>(a, x, item);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.item_full[sl]);
        if (!item->valid) break;
        if (elect_one()) ask_next(&sh);
        ++asked;
        const int n = item->tiles, first = item->first;
        bool ok = true;
        for (int p = 0; ok && p < 2 * n; ++p) {
          bool is_v;
          int j;
          if constexpr (C::kChain) {
            is_v = p == 2 * n - 1 || (p >= 2 && (p & 1) == 0);
            j = p == 0 ? 0 : (p == 2 * n - 1 ? n - 1 : ((p & 1) ? (p + 1) / 2 : (p - 2) / 2));
          } else {
            is_v = p & 1;
            j = p >> 1;
          }
          const bool edge = is_v && j >= first;
#pragma unroll
          for (int part = 0; ok && part < C::kParts; ++part, ++g) {
            const int slot = static_cast<int>(g % C::kSlots);
            ok = wait(&sh, &bar.kv_empty[slot], ((g / C::kSlots) & 1u) ^ 1u);
            if (!ok) break;
            if (elect_one()) {
              uint64_t *full = edge ? &bar.v_edge[slot] : &bar.kv_full[slot];
              const uint32_t dst = kv_s + slot * C::kSlot;
              const int row = item->k0 + j * C::kN;
              mbar_expect_tx(full, C::kSlot);
              if (is_v) {
#pragma unroll
                for (int d = 0; d < D / 64; ++d) tma_load_3d(dst + d * C::kVPanel, &map_v, d * 64, item->h, row + part * C::kVKeys, full);
              } else {
#pragma unroll
                for (int d = 0; d < C::kKDims / 64; ++d)
                  tma_load_3d(dst + d * C::kKPanel, &map_k, part * C::kKDims + d * 64, item->h, row, full);
              }
              if (edge) mbar_arrive(&bar.kv_full[slot]);
            }
            edge_ph ^= edge ? 1u << slot : 0u;
            edge_last = edge ? edge_last | (1u << slot) : edge_last & ~(1u << slot);
            __syncwarp();
          }
        }
        if (!ok || !wait(&sh, &bar.next_full, it & 1)) break;
        x = read_next(&sh);
        __syncwarp();
      }
      // loads and the request in flight when the others gave up must land before the CTA leaves
      if (*reinterpret_cast<volatile int *>(&sh.abort)) {
        if (asked) drain(&bar.next_full, (asked - 1) & 1u);
        for (uint32_t i = g > C::kSlots ? g - C::kSlots : 0u; i < g; ++i) {
          const int slot = static_cast<int>(i % C::kSlots);
          const bool edge = (edge_last >> slot) & 1u;
          uint64_t *full = edge ? &bar.v_edge[slot] : &bar.kv_full[slot];
          const uint32_t ph = edge ? ((edge_ph >> slot) & 1u) ^ 1u : (i / C::kSlots) & 1u;
          drain(full, ph);
        }
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------- MMAs
      // One thread issues, but the whole warp keeps the state, and what it reads from shared memory goes
      // through a warp reduction: the compiler then sees uniform values, and descriptors and addresses stay
      // in uniform registers.  With state in ordinary registers each MMA took about 130 cycles to issue,
      // twice its time on the tensor core.
      constexpr uint32_t id_s = idesc_bf16(C::kN, false), id_o = idesc_bf16(D, true);
      struct Ring {
        int slot;
        uint32_t ph;
        __device__ __forceinline__ void next(int d) {
          slot += d;
          if (slot >= C::kSlots) {
            slot -= C::kSlots;
            ph ^= 1u;
          }
        }
      };
      Ring base{0, 0u};                               // slot of this item's first piece
      uint32_t o_ph = 1u;                             // phase of o_free: of the last item that had keys
      uint32_t fixed = 0u, pph = 0u;                  // phase bits: v_fixed per slot, P per buffer
      const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const int sl = it & 1;
        ok = wait(&sh, &bar.item_full[sl], (it >> 1) & 1);
        if (!ok) break;
        const Item *item = &sh.item[sl];
        const int n = __reduce_max_sync(0xffffffffu, item->tiles), first = __reduce_max_sync(0xffffffffu, item->first);
        const int valid = __reduce_max_sync(0xffffffffu, item->valid);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.item_empty[sl]);
        if (!valid) break;
        const int steps = n * C::kTiles;
        // key tiles come at positions 0, 2, 4, ... and value tiles at 1, 3, ...; at D = 256 at 0, 1, 3, 5, ... and
        // 2, 4, ..., 2 n - 2, 2 n - 1
        Ring rk = base, rv = base;
        rv.next(C::kChain && n > 1 ? 2 * C::kParts : C::kParts);
        auto issue_s = [&](int s) {
          const int j = C::kChain ? s : s >> 1, w = C::kChain ? 0 : s & 1;
          if (j == 0 && !wait(&sh, &bar.q_full[w], it & 1)) return false;
          Ring at = rk;
#pragma unroll
          for (int part = 0; part < C::kParts; ++part, at.next(1)) {
            if (!wait(&sh, &bar.kv_full[at.slot], at.ph)) return false;
            tc_fence_after();
            const uint32_t qa = desc_k(q_s + w * (128 * D * 2) + part * (C::kKDims / 64) * 16384), kb = desc_k(kv_s + at.slot * C::kSlot);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < C::kKDims / 16; ++kk) {
                const uint32_t step = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;       // both panels are 16 KB
                mma_ss(tm + (s & 1) * C::kN, qa + step, kb + step, id_s, (part | kk) != 0);
              }
              if (C::kChain || w == 1) tc_commit(&bar.kv_empty[at.slot]);
              if (part == C::kParts - 1) {
                tc_commit(&bar.s_full[s & 1]);
                if (s >= steps - C::kTiles) tc_commit(&bar.q_empty[w]);
              }
            }
            __syncwarp();
          }
          if (C::kChain || w == 1) rk.next(C::kChain && j == 0 ? C::kParts : 2 * C::kParts);
          return true;
        };
        if (steps == 0)                               // nothing to read Q for
          for (int w = 0; ok && w < C::kTiles; ++w) {
            ok = wait(&sh, &bar.q_full[w], it & 1);
            if (ok && lane == 0) mbar_arrive(&bar.q_empty[w]);
          }
        for (int s = 0; ok && s < 2 && s < steps; ++s) ok = issue_s(s);
        // The last O has been read.  Items without keys have none and take no part in this: the softmax warps run
        // through them without this warp, two of them would pass two phases before it looks
        if (ok && steps > 0) {
          ok = wait(&sh, &bar.o_free, o_ph);
          o_ph ^= 1u;
        }
        for (int s = 0; ok && s < steps; ++s) {
          const int j = C::kChain ? s : s >> 1, w = C::kChain ? 0 : s & 1, buf = s & 1;
          // the keys of P's first half are multiplied while the softmax still works on the second
          const uint32_t o = tm + C::kOCol + w * D, p = tm + buf * C::kN;
          Ring at = rv;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half == 0 || C::kParts == 2) {
              if (half == 1) at.next(1);
              ok = ok && wait(&sh, &bar.kv_full[at.slot], at.ph);
              if (ok && j >= first && w == 0) {
                ok = wait(&sh, &bar.v_fixed[at.slot], (fixed >> at.slot) & 1u);
                fixed ^= 1u << at.slot;
              }
            }
            ok = ok && wait(&sh, half ? &bar.p_ready[buf] : &bar.p_half[buf], (pph >> buf) & 1u);
            if (!ok) break;
            tc_fence_after();
            const uint32_t vb = desc_mn(kv_s + at.slot * C::kSlot, C::kVPanel);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < C::kN / 32; ++kk) {
                const int kp = half * (C::kN / 32) + kk, kv = C::kParts == 2 ? kk : kp;
                mma_ts(o, p + kp * 8, vb + kv * (2048 >> 4), id_o, (j | kp) != 0);
              }
              if (half == 1 && (C::kChain || s >= steps - 2)) tc_commit(&bar.o_done[buf]);
              if (C::kParts == 2 || (half == 1 && (C::kChain || w == 1))) tc_commit(&bar.kv_empty[at.slot]);
            }
            __syncwarp();
          }
          if (!ok) break;
          pph ^= 1u << buf;
          if (s == steps - 1) {                       // the item's last piece
            base = at;
            base.next(1);
          }
          if (C::kChain || w == 1) rv.next(C::kChain && j == n - 2 ? C::kParts : 2 * C::kParts);
          if (s + 2 < steps) ok = issue_s(s + 2);
        }
      }
      if (*reinterpret_cast<volatile int *>(&sh.abort)) {
        if (elect_one()) tc_commit(&bar.mma_end);
        __syncwarp();
        drain(&bar.mma_end, 0u);
      }
    } else {
      // --------------------------------- query rows, and values of edge tiles
      const int ht = tid - 320;
      uint32_t g0 = 0u, edge_ph = 0u;                 // pieces before this item, phases of v_edge
      uint32_t q_loads = 0u;                          // tiles of Q loaded by TMA so far
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const int sl = it & 1;
        ok = wait(&sh, &bar.item_full[sl], (it >> 1) & 1);
        if (!ok) break;
        Item *item = &sh.item[sl];
        if (!item->valid) break;
        const int n = item->tiles, first = item->first, nk = item->nk - item->skip;
        const int64_t rows = static_cast<int64_t>(item->nq) * a.G;
        for (int w = 0; ok && w < C::kTiles; ++w) {
          ok = wait(&sh, &bar.q_empty[w], (it & 1) ^ 1);
          if (!ok) break;
          const int R0 = item->blk * C::kRows + w * 128;
          const uint32_t qt = q_s + w * (128 * D * 2);
          if (a.q_tma) {
            // rows behind the sequence bring other rows' values; they are computed and not stored
            if (warp == 10 && elect_one()) {
              mbar_expect_tx(&bar.q_full[w], 128 * D * 2);
#pragma unroll
              for (int d = 0; d < D / 64; ++d)
                tma_load_3d(qt + d * 16384, &map_q, d * 64, item->h * a.G, item->q0 + R0 / a.G, &bar.q_full[w]);
            }
            __syncwarp();
            ++q_loads;
            continue;
          }
          constexpr int per = D / 8;                  // 16-byte pieces of a row
          constexpr int kStep = kHelpers / per;       // rows that the helpers copy at once
          const int c = ht % per;
          int r = ht / per, i = (R0 + r) / a.G, hg = R0 + r - i * a.G;
          const wm_bf16 *base = a.q + static_cast<int64_t>(item->q0) * a.q_stride + static_cast<int64_t>(item->h) * a.G * D + c * 8;
#pragma unroll 4
          for (; r < 128; r += kStep) {
            const bool in = R0 + r < rows;
            const wm_bf16 *src = base + (in ? i * a.q_stride + static_cast<int64_t>(hg) * D : 0);
            const uint32_t dst = qt + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
            for (hg += kStep; hg >= a.G; hg -= a.G) ++i;
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(&bar.q_full[w]);
        }
        for (int y = first * C::kParts; ok && y < n * C::kParts; ++y) {
          const int j = y / C::kParts, part = y % C::kParts;
          const int slot = static_cast<int>((g0 + pos_v<ONE>(j, n) * C::kParts + part) % C::kSlots);
          ok = wait(&sh, &bar.v_edge[slot], (edge_ph >> slot) & 1u);
          if (!ok) break;
          edge_ph ^= 1u << slot;
          uint4 *vt = reinterpret_cast<uint4 *>(smem + C::kQBytes + slot * C::kSlot);
          const int live = nk - j * C::kN;
          for (int x = ht; x < C::kSlot / 16; x += kHelpers) {
            const int r = part * C::kVKeys + (x >> 3) % C::kVKeys;    // key of this 16-byte piece
            if (r >= live) {
              vt[x] = make_uint4(0u, 0u, 0u, 0u);
              continue;
            }
            const uint4 v = vt[x];
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {             // exponent bits all ones
              const bool lo = (w[e] & 0x7f80u) == 0x7f80u, hi = (w[e] & 0x7f800000u) == 0x7f800000u;
              odd |= lo | hi;
              w[e] = (lo ? 0u : w[e] & 0xffffu) | (hi ? 0u : w[e] & 0xffff0000u);
            }
            if (odd) {
              vt[x] = make_uint4(w[0], w[1], w[2], w[3]);
              if (j - first < 4) atomicOr(&item->odd[(j - first) * 4 + (r >> 5)], 1u << (r & 31));
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(&bar.v_fixed[slot]);
        }
        mbar_arrive(&bar.odd_ready[sl]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.item_empty[sl]);
        g0 += 2 * n * C::kParts;
      }
      if (*reinterpret_cast<volatile int *>(&sh.abort))
        for (uint32_t i = q_loads > C::kTiles ? q_loads - C::kTiles : 0u; i < q_loads; ++i)
          drain(&bar.q_full[i % C::kTiles], (i / C::kTiles) & 1u);
    }
  } else {
    // ------------------------------------------------- softmax, one row each
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int w = warp >> 2, r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem + lanes + w * C::kN;
    const uint32_t o_t = tmem + lanes + C::kOCol + (C::kChain ? 0 : w * D);
    uint32_t sph = 0u;                                // phase of this warpgroup's S
    // D = 256: steps of the items before on each buffer, the phases of o_done and m_ready; else the
    // items before that had keys, the phase of o_done
    uint32_t done[2] = {0u, 0u};
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int sl = it & 1;
      ok = wait(&sh, &bar.item_full[sl], (it >> 1) & 1);
      if (!ok) break;
      const Item *item = &sh.item[sl];
      if (!item->valid) break;
      const int n = item->tiles, first = item->first, nq = item->nq, nk = item->nk;
      const int steps = n * C::kTiles;
      const int R = item->blk * C::kRows + (C::kChain ? 0 : w * 128) + r;
      const bool live = R < static_cast<int64_t>(nq) * a.G;
      const int see = live ? visible(a, nq, nk, R) - item->skip : 0;     // of the item's keys
      float m = kNegInf, l = 0.0f;

      for (int s = w; ok && s < steps; s += 2) {
        const int j = C::kChain ? s : s >> 1;
        ok = wait(&sh, &bar.s_full[w], sph);
        if (!ok) break;
        sph ^= 1u;
        tc_fence_after();
        uint32_t x[C::kN / 32][32];
#pragma unroll
        for (int c = 0; c < C::kN / 32; ++c) tmem_ld32(x[c], s_t + c * 32);
        tmem_wait_ld();
        if (j >= first) {
          const int room = see - j * C::kN;
#pragma unroll
          for (int c = 0; c < C::kN; ++c)
            if (c >= room) x[c >> 5][c & 31] = __float_as_uint(kNegInf);
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = __uint_as_float(x[0][c]);
#pragma unroll
        for (int c = 4; c + 8 <= C::kN; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mx[e] = max3(mx[e], __uint_as_float(x[(c + 2 * e) >> 5][(c + 2 * e) & 31]), __uint_as_float(x[(c + 2 * e + 1) >> 5][(c + 2 * e + 1) & 31]));
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(x[C::kN / 32 - 1][28 + e]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
        if constexpr (C::kChain) {
          if (s > 0) {                                // the reference point as the other warpgroup left it
            ok = wait(&sh, &bar.m_ready[w ^ 1], (done[w ^ 1] + ((s - 1) >> 1)) & 1u);
            if (!ok) break;
            const float mo = *reinterpret_cast<volatile float *>(&sh.m[r]);
            if (mo != m) {
              l *= m == kNegInf ? 0.0f : ex2(m - mo);
              m = mo;
            }
          }
        }
        const bool grow = top > m + kSlack || (m == kNegInf && top > m);
        const float f = grow ? (m == kNegInf ? 0.0f : ex2(m - top)) : 1.0f;
        if (grow) {
          m = top;
          l *= f;
        }
        if constexpr (C::kChain) {
          *reinterpret_cast<volatile float *>(&sh.m[r]) = m;
          mbar_arrive(&bar.m_ready[w]);
        }
        // O holds PV of the steps before.  With two tiles S(s) followed PV(s - 2), the last one on this O, in
        // the MMA warp's order, so it is complete; at D = 256 the last one is PV(s - 1)
        if (j > 0 && __any_sync(0xffffffffu, grow)) {
          if constexpr (C::kChain) {
            ok = wait(&sh, &bar.o_done[w ^ 1], (done[w ^ 1] + ((s - 1) >> 1)) & 1u);
            if (!ok) break;
            tc_fence_after();
          }
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(o, o_t + c);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st32(o_t + c, o);
          }
        }
        const float base = m == kNegInf ? 0.0f : m;
        const float2 sc = make_float2(a.scale2, a.scale2), nb = make_float2(-base, -base);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[C::kN / 4];                      // half of the keys
#pragma unroll
          for (int i = 0; i < C::kN / 4; ++i) {
            const int c = h * (C::kN / 2) + 2 * i;
            float2 e = wm_fma2(make_float2(__uint_as_float(x[c >> 5][c & 31]), __uint_as_float(x[(c + 1) >> 5][(c + 1) & 31])), sc, nb);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[i & 1] = wm_add2(sum[i & 1], e);
            p[i] = bf16x2(e.x, e.y);
          }
          tmem_st32(s_t + h * 32, p);
          if (h == 0) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bar.p_half[w]);
          }
        }
        l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bar.p_ready[w]);
      }
      if (!ok) break;

      // --------------------------------------------------------- epilogue
      if (steps > 0) {
        const int last = C::kChain ? (steps - 1) & 1 : w;
        ok = wait(&sh, &bar.o_done[last], (done[last] + (C::kChain ? (steps - 1) >> 1 : 0)) & 1u);
        if (!ok) break;
        done[0] += C::kChain ? (steps + 1) >> 1 : 1;
        done[1] += C::kChain ? steps >> 1 : 1;
      }
      ok = wait(&sh, &bar.odd_ready[sl], (it >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if constexpr (C::kChain) {
        // both warpgroups' sums at the last reference point; two phases of `both` per item
        mbar_arrive(&bar.both);
        ok = wait(&sh, &bar.both, 0);
        if (!ok) break;
        if (steps > 0) {
          const float ml = *reinterpret_cast<volatile float *>(&sh.m[r]);
          if (m != ml) l *= m == kNegInf ? 0.0f : ex2(m - ml);          // a sum of NaN scores stays NaN
          m = ml;
        }
        sh.l[w][r] = l;
        mbar_arrive(&bar.both);
        ok = wait(&sh, &bar.both, 1);
        if (!ok) break;
        l = sh.l[0][r] + sh.l[1][r];
      }
      uint32_t any = 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) any |= item->odd[i];
      const float inv = see > 0 ? 1.0f / l : 0.0f;
      const int i = R / a.G, hg = R - i * a.G;
      const int64_t head = (static_cast<int64_t>(item->q0) + i) * a.Hq + item->h * a.G + hg;
      constexpr int kCols = C::kChain ? D / 2 : D;    // at D = 256 each warpgroup writes half of every row
      const int col0 = C::kChain ? w * kCols : 0;
      for (int c = col0; c < col0 + kCols; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(o, o_t + c);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (live && any) {                            // values that are not finite, for the rows that see them
          for (int t = 0; t < 16; ++t)
            for (uint32_t bits = item->odd[t]; bits; bits &= bits - 1) {
              const int key = (first + (t >> 2)) * C::kN + (t & 3) * 32 + __ffs(bits) - 1;
              if (key >= see) continue;
              const wm_bf16 *vp = a.v + (static_cast<int64_t>(item->k0) + key) * a.v_stride + static_cast<int64_t>(item->h) * D + c;
              for (int e = 0; e < 32; ++e) {
                const float x = wm_bf16_to_f32(vp[e]);
                if (!(fabsf(x) <= 3.4028234663852886e38f)) {
#pragma unroll
                  for (int y = 0; y < 32; ++y)
                    if (y == e) o[y] = __float_as_uint(__uint_as_float(o[y]) + x);
                }
              }
            }
        }
        if (SP && item->parts > 1) {
          uint32_t *dst = reinterpret_cast<uint32_t *>(a.part_o) +
                          (static_cast<int64_t>(item->slot) * C::kRows + (R - item->blk * C::kRows)) * D + c;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t y[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) y[z] = o[8 * e + z];
            if (live) store32(dst + 8 * e, y);
          }
          __syncwarp();
          continue;
        }
        // whole 32-byte sectors: 16-byte stores to 32 rows at a time took twice as long
        wm_bf16 *dst = a.out + head * D + c;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t y[8];
#pragma unroll
          for (int z = 0; z < 8; ++z) {
            const float lo = __uint_as_float(o[16 * e + 2 * z]), hi = __uint_as_float(o[16 * e + 2 * z + 1]);
            y[z] = see > 0 ? bf16x2(lo * inv, hi * inv) : 0u;
          }
          if (live) store32(dst + 16 * e, y);
        }
        __syncwarp();                                 // the TMEM loads are whole-warp instructions
      }
      if (SP && item->parts > 1) {
        if (live && (!C::kChain || w == 0))
          a.part_ml[static_cast<int64_t>(item->slot) * C::kRows + (R - item->blk * C::kRows)] = make_float2(m, l);
      } else if (live && a.lse && (!C::kChain || w == 0)) a.lse[head] = see > 0 ? (m + log2f(l)) * kLn2 : kNegInf;
      tc_fence_before();
      if (steps > 0) mbar_arrive(&bar.o_free);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.item_empty[sl]);
    }
  }
  __syncthreads();
  if (*reinterpret_cast<volatile int *>(&sh.abort)) { // a wait ran out: no result passes for one
    const int64_t heads = static_cast<int64_t>(a.Tq) * a.Hq;
    wm_giveup::poison(a.out, heads * D, a.lse, heads, SP ? a.part_ml : nullptr, static_cast<int64_t>(a.slots) * C::kRows, tid, kThreads);
  }
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// The parts of split blocks joined with weights 2^(m_part - m).  A CTA per work
// item: those of one block share its rows, a warp takes one row at a time.
constexpr int kJoinThreads = 512;
template <int D, bool ONE>
__global__ void __launch_bounds__(kJoinThreads) k_attn_prompt_join(PromptArgs a) {
  using C = Cfg<D, ONE>;
  constexpr int kV = D / 32;                          // values of a lane, in pieces of kW
  constexpr int kW = kV < 4 ? kV : 4;
  using Piece = typename std::conditional<kW == 2, float2, float4>::type;
  __shared__ Item item;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  WM_PDL_WAIT();
  if (warp == 0) find_item<D, ONE, true>(a, static_cast<int>(blockIdx.x), &item);
  __syncthreads();
  if (!item.valid || item.parts < 2) return;
  // part y is in slot slot0 - y Hkv; of malformed, overlapping sequences some have no slot
  const int64_t slot0 = item.slot + static_cast<int64_t>(item.part) * a.Hkv;
  const int y0 = slot0 < a.slots ? 0 : static_cast<int>((slot0 - a.slots) / a.Hkv) + 1;
  const int r1 = static_cast<int>(static_cast<int64_t>(C::kRows) * (item.part + 1) / item.parts);
  for (int r = static_cast<int>(static_cast<int64_t>(C::kRows) * item.part / item.parts) + warp; r < r1; r += kJoinThreads / 32) {
    const int R = item.blk * C::kRows + r;
    if (R >= static_cast<int64_t>(item.nq) * a.G) break;
    auto at = [&](int y) { return (slot0 - static_cast<int64_t>(y) * a.Hkv) * C::kRows + r; };
    float m = kNegInf;
    for (int y = y0 + lane; y < item.parts; y += 32) m = fmaxf(m, a.part_ml[at(y)].x);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    float l = 0.0f, o[kV] = {};
#pragma unroll 4
    for (int y = y0; y < item.parts; ++y) {
      const float2 ml = a.part_ml[at(y)];
      const Piece *po = reinterpret_cast<const Piece *>(a.part_o + at(y) * D) + lane;
      // never 0 for a seen part, so that an infinite value shows as such
      const float f = ml.x == kNegInf ? 0.0f : fmaxf(ex2(ml.x - m), 1.17549435e-38f);
      l += ml.x == kNegInf ? ml.y : f * ml.y;         // no key of the part seen: 0, or NaN of NaN scores
#pragma unroll
      for (int i = 0; i < kV / kW; ++i) {
        const Piece v = po[32 * i];
        if (ml.x == kNegInf) continue;
        o[kW * i] += f * v.x;
        o[kW * i + 1] += f * v.y;
        if constexpr (kW == 4) {
          o[kW * i + 2] += f * v.z;
          o[kW * i + 3] += f * v.w;
        }
      }
    }
    const bool sees = visible(a, item.nq, item.nk, R) > 0;
    const float inv = sees ? 1.0f / l : 0.0f;
    const int t = R / a.G;
    const int64_t head = (static_cast<int64_t>(item.q0) + t) * a.Hq + item.h * a.G + (R - t * a.G);
#pragma unroll
    for (int i = 0; i < kV / kW; ++i)
#pragma unroll
      for (int e = 0; e < kW; e += 2)
        *reinterpret_cast<uint32_t *>(a.out + head * D + 32 * kW * i + kW * lane + e) =
            sees ? bf16x2(o[kW * i + e] * inv, o[kW * i + e + 1] * inv) : 0u;
    if (a.lse && lane == 0) a.lse[head] = sees ? (m + log2f(l)) * kLn2 : kNegInf;
  }
}

// [tokens, heads, D] bf16 with `stride` values between tokens, boxes of 64
// dimensions x box_heads heads x box_rows tokens; tokens behind the last read as
// zeros.
int make_map3(CUtensorMap *map, const void *base, int D, int heads, int64_t tokens, int64_t stride, int box_heads, int box_rows) {
  auto fn = wm_tc::encode_fn();
  if (!fn) return wm::fail(WM_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(stride) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return wm::fail(WM_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return WM_OK;
}

// Rows of a block.  D = 256 has TMEM for one tile.  At D = 64 and 128 a block takes
// one tile where the sequences' rows fill no more than that on average: the second
// tile's products would be wasted.
// Two tiles -> one (32/8 heads of 128, us): 37 sequences of 32 rows on 4096 keys 151
// -> 107, 32 of 4 rows on 4000 and one of 512 190 -> 123; at 64 rows of 4 heads each
// on their own keys 17 -> 21, 8 sequences of 2048 289 -> 392, as K and V are read
// twice as often and each step waits for one softmax.
int block_rows(int B, int Tq, int Hq, int Hkv, int D) {
  return D == 256 || static_cast<int64_t>(Tq) * (Hq / Hkv) <= 128ll * B ? 128 : 256;
}

// Work items of a call without splitting, at most: one partial block per sequence
// beyond the rows' own blocks.
int64_t most_items(int B, int Tq, int Hq, int Hkv, int D) {
  return (static_cast<int64_t>(Tq) * (Hq / Hkv) / block_rows(B, Tq, Hq, Hkv, D) + B) * Hkv;
}

// Slots for the parts of split blocks, 0 where none is split.  With fewer blocks
// than SMs the rest would idle (32/8 heads of 128, us): 64 rows on 32,768 keys 453
// -> 52, 512 rows 460 -> 257; 16 rows on 4096 keys 63 -> 19, on 2048 36 -> 17; two
// sequences on 1024 each 22 -> 19, hence the least count.  The join costs 6 us where
// nothing turns out to be split, so one sequence with more blocks than half of the
// SMs, which never is, goes without; several may be ragged (16 rows each, 15
// sequences of 500 and one of 32,768 keys: 453 -> 63).
int split_slots(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  const int64_t most = most_items(B, Tq, Hq, Hkv, D), sms = wm::sm_count();
  if (Tk < kSplitKeys || Tk / (kSplitKeys / 2) < B || 2 * most >= (B == 1 ? sms : 3 * sms)) return 0;
  return static_cast<int>(std::max(sms, most + sms / 2));
}


size_t slot_bytes(int rows, int D) { return static_cast<size_t>(rows) * (D + 2) * sizeof(float); }

template <int D, bool ONE, bool SP>
int launch_as(const PromptArgs &a, int64_t grid, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t stream) {
  cudaError_t e = wm::allow_smem<k_attn_prompt<D, ONE, SP>>(smem_bytes<D, ONE>());
  if (e == cudaSuccess)
    e = wm::launch_pdl(k_attn_prompt<D, ONE, SP>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem_bytes<D, ONE>(), stream, a, mq, mk,
                       mv);
  if constexpr (SP)
    if (e == cudaSuccess) e = wm::launch_pdl(k_attn_prompt_join<D, ONE>, dim3(static_cast<unsigned>(grid)), dim3(kJoinThreads), 0, stream, a);
  if (e != cudaSuccess) return wm::fail(WM_ERR_CUDA, std::string("wattn_prompt: ") + cudaGetErrorString(e));
  return wm::check_launch("wattn_prompt");
}

template <int D, bool ONE>
int launch(const PromptArgs &a, const wm_bf16 *k, int64_t k_stride, cudaStream_t stream) {
  using C = Cfg<D, ONE>;
  CUtensorMap mq, mk, mv;
  if (int rc = make_map3(&mq, a.q, D, a.Hq, a.Tq, a.q_stride, a.q_tma ? a.G : 1, a.q_tma ? 128 / a.G : 128)) return rc;
  // without keys no tile is loaded; the maps then describe one row of q
  const bool any = a.Tk > 0;
  if (int rc = make_map3(&mk, any ? k : a.q, D, any ? a.Hkv : 1, any ? a.Tk : 1, any ? k_stride : D, 1, C::kN)) return rc;
  if (int rc = make_map3(&mv, any ? a.v : a.q, D, any ? a.Hkv : 1, any ? a.Tk : 1, any ? a.v_stride : D, 1, C::kVKeys)) return rc;
  if (a.slots) return launch_as<D, ONE, true>(a, a.slots, mq, mk, mv, stream);
  const int64_t most = most_items(a.B, a.Tq, a.Hq, a.Hkv, D);
  WM_REQUIRE(most <= INT32_MAX, "prompt attention: too many rows");
  return launch_as<D, ONE, false>(a, std::max<int64_t>(most, 1), mq, mk, mv, stream);
}

}  // namespace

extern "C" {

size_t wattn_prompt_workspace_size(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  if (B <= 0 || Tq <= 0 || Tk < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128 && D != 256)) return 0;
  return split_slots(B, Tq, Tk, Hq, Hkv, D) * slot_bytes(block_rows(B, Tq, Hq, Hkv, D), D);
}

int wattn_prompt(const wm_bf16 *q, const wm_bf16 *k, const wm_bf16 *v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                 const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k, int B, int Tq, int Tk, int Hq, int Hkv, int D,
                 float scale, int causal, wm_bf16 *out, float *lse, void *workspace, size_t ws_bytes, wm_stream_t stream) {
  wm::clear_error();
  WM_REQUIRE(B >= 0 && Tq >= 0 && Tk >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0,
             "prompt attention: the query heads must be a multiple of the key-value heads");
  WM_REQUIRE(D == 64 || D == 128 || D == 256, "prompt attention: head dimension 64, 128 or 256");
  WM_REQUIRE(scale > 0.0f && scale * kLog2e <= 3.4028234663852886e38f, "prompt attention: the scale must be positive and finite");
  if (B == 0 || Tq == 0) return WM_OK;
  WM_REQUIRE(q && out && cu_seqlens_q && cu_seqlens_k && (Tk == 0 || (k && v)), "prompt attention: missing input or output");
  WM_REQUIRE(q_stride >= static_cast<int64_t>(Hq) * D && k_stride >= static_cast<int64_t>(Hkv) * D &&
                 v_stride >= static_cast<int64_t>(Hkv) * D && q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 &&
                 wm::aligned(q, 16) && wm::aligned(k, 16) && wm::aligned(v, 16) && wm::aligned(out, 32),
             "prompt attention: token rows must be 16-byte aligned and hold their heads, the output 32-byte aligned");
  WM_REQUIRE(static_cast<int64_t>(Tq) * (Hq / Hkv) <= INT32_MAX - 256, "prompt attention: too many rows per key-value head");
  const int slots = split_slots(B, Tq, Tk, Hq, Hkv, D);
  const int rows = block_rows(B, Tq, Hq, Hkv, D);
  if (ws_bytes < slots * slot_bytes(rows, D)) return wm::fail(WM_ERR_WORKSPACE, "prompt attention: workspace too small");
  WM_REQUIRE(slots == 0 || (workspace && wm::aligned(workspace, 256)), "prompt attention: the workspace must be 256-byte aligned");
  float *ws = static_cast<float *>(workspace);
  const int64_t sums = static_cast<int64_t>(slots) * rows;
  const PromptArgs a{q, v, q_stride, v_stride, cu_seqlens_q, cu_seqlens_k, B, Tq, Tk, Hq, Hkv, Hq / Hkv, causal,
                     128 % (Hq / Hkv) == 0, scale * kLog2e, out, lse, slots, wm::sm_count(), ws, slots ? reinterpret_cast<float2 *>(ws + sums * D) : nullptr};
  const bool one = rows == 128;
  if (D == 64) return one ? launch<64, true>(a, k, k_stride, stream) : launch<64, false>(a, k, k_stride, stream);
  if (D == 128) return one ? launch<128, true>(a, k, k_stride, stream) : launch<128, false>(a, k, k_stride, stream);
  return launch<256, true>(a, k, k_stride, stream);
}

}  // extern "C"
