// The paged key-value cache shared by its append, attention and eviction
// kernels: row formats, page lookups and the argument checks of the entry
// points.
//
// A cache tensor is a pool [n_pages, Hkv, page_size, D]: the rows of one head
// within a page are contiguous, so a tile of up to page_size keys is one run of
// bytes.  Entry e of sequence b lies in page page_table[b, e / page_size], slot
// e % page_size.  Page sizes are multiples of 16, so an aligned tile of 16 keys
// never crosses a page.
#pragma once

#include "wm_common.cuh"

namespace wm_paged {

__host__ __device__ constexpr int row_bytes(int fmt, int D) { return fmt == WKV_BF16 ? 2 * D : D; }
// bytes of one row's scales
__host__ __device__ constexpr int scale_bytes(int fmt, int D) {
  return fmt == WKV_FP8_F32_B64 ? 4 * (D / 64) : (fmt == WKV_MXFP8_B32 ? D / 32 : 0);
}

inline bool is_paged_fmt(int fmt) { return fmt == WKV_BF16 || fmt == WKV_FP8_F32_B64 || fmt == WKV_MXFP8_B32; }

struct Pool {
  void *k, *v;               // [n_pages, Hkv, page_size, D] rows
  void *ks, *vs;             // their scales, or null
  const int32_t *table;      // [B, max_pages]
  int n_pages, page_size, max_pages, Hkv;
};

inline int check_pool(const Pool &p, int B, int D, int fmt) {
  WM_REQUIRE(is_paged_fmt(fmt), "paged cache rows are bf16, fp8_f32_b64 or mxfp8");
  WM_REQUIRE(D == 64 || D == 128 || D == 256, "paged cache: head dimension 64, 128 or 256");
  WM_REQUIRE(B >= 0 && p.Hkv > 0 && p.n_pages >= 0 && p.max_pages >= 0, "paged cache: negative or empty shape");
  WM_REQUIRE(p.page_size > 0 && p.page_size % 16 == 0, "paged cache: the page size must be a multiple of 16");
  WM_REQUIRE(static_cast<int64_t>(p.max_pages) * p.page_size <= INT32_MAX, "paged cache: a sequence holds at most 2^31 - 1 entries");
  if (B == 0) return WM_OK;
  WM_REQUIRE(p.k && p.v && p.table, "paged cache: missing cache or page table");
  WM_REQUIRE((fmt == WKV_BF16) == (p.ks == nullptr) && (fmt == WKV_BF16) == (p.vs == nullptr),
             "paged cache: quantized rows need scales, bf16 rows take none");
  WM_REQUIRE(wm::aligned(p.k, 16) && wm::aligned(p.v, 16) && wm::aligned(p.ks, 16) && wm::aligned(p.vs, 16) &&
                 wm::aligned(p.table, 4),
             "paged cache: caches and scales must be 16-byte aligned");
  return WM_OK;
}

}  // namespace wm_paged
