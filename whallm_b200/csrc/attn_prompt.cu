// Attention of packed prompts: grouped heads, causal (aligned at the end, so new
// tokens may continue a longer history) or full.
//
//   row i of a sequence with nq rows and nk keys sees the keys j <= i + nk - nq
//   (causal) or all nk;  s_j = scale q.k_j,  lse = log sum_j exp(s_j),
//   out = sum_j exp(s_j - lse) v_j;  a row that sees no key: out 0, lse -inf.
//
// One warp per (row, head) on CUDA cores, one pass with a running maximum.
#include <algorithm>

#include "wm_common.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PromptArgs {
  const wm_bf16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const int32_t *cu_q, *cu_k;
  int B, Tq, Tk, Hq, Hkv, causal;
  float scale2;
  wm_bf16 *out;
  float *lse;
};

template <int D>
__global__ void __launch_bounds__(256) k_attn_prompt_rows(PromptArgs a) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(a.Tq) * a.Hq;
  for (int64_t x = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; x < n; x += ((int64_t)gridDim.x * blockDim.x) >> 5) {
    const int t = static_cast<int>(x / a.Hq), h = static_cast<int>(x - static_cast<int64_t>(t) * a.Hq), hk = h / (a.Hq / a.Hkv);
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid] <= t) lo = mid; else hi = mid;
    }
    const int q0 = a.cu_q[lo], q1 = a.cu_q[lo + 1];
    if (t < q0 || t >= q1) continue;
    const int k0 = max(a.cu_k[lo], 0), k1 = min(a.cu_k[lo + 1], a.Tk);
    const int last = a.causal ? min(k1, k0 + (t - q0) + (k1 - k0) - (q1 - q0) + 1) : k1;
    float q[V], o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      q[i] = wm_bf16_to_f32(a.q[t * a.q_stride + h * D + i * 32 + lane]) * a.scale2;
      o[i] = 0.0f;
    }
    float m = -__builtin_huge_valf(), l = 0.0f;
    for (int64_t j = k0; j < last; ++j) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) s = fmaf(q[i], wm_bf16_to_f32(a.k[j * a.k_stride + hk * D + i * 32 + lane]), s);
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      const float top = fmaxf(m, s), f = m == top ? 1.0f : exp2f(m - top), p = exp2f(s - top);
      m = top;
      l = l * f + p;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(o[i], f, p * wm_bf16_to_f32(a.v[j * a.v_stride + hk * D + i * 32 + lane]));
    }
    const float inv = last > k0 ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) a.out[(static_cast<int64_t>(t) * a.Hq + h) * D + i * 32 + lane] = wm_f32_to_bf16(o[i] * inv);
    if (a.lse && lane == 0) a.lse[x] = last > k0 ? (m + log2f(l)) * kLn2 : -__builtin_huge_valf();
  }
}

}  // namespace

extern "C" {

int wattn_prompt(const wm_bf16 *q, const wm_bf16 *k, const wm_bf16 *v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                 const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k, int B, int Tq, int Tk, int Hq, int Hkv, int D,
                 float scale, int causal, wm_bf16 *out, float *lse, wm_stream_t stream) {
  wm::clear_error();
  WM_REQUIRE(B >= 0 && Tq >= 0 && Tk >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0,
             "prompt attention: the query heads must be a multiple of the key-value heads");
  WM_REQUIRE(D == 64 || D == 128 || D == 256, "prompt attention: head dimension 64, 128 or 256");
  WM_REQUIRE(scale > 0.0f && scale <= 3.4028234663852886e38f, "prompt attention: the scale must be positive and finite");
  if (B == 0 || Tq == 0) return WM_OK;
  WM_REQUIRE(q && out && cu_seqlens_q && cu_seqlens_k && (Tk == 0 || (k && v)), "prompt attention: missing input or output");
  WM_REQUIRE(q_stride >= static_cast<int64_t>(Hq) * D && k_stride >= static_cast<int64_t>(Hkv) * D &&
                 v_stride >= static_cast<int64_t>(Hkv) * D && q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 &&
                 wm::aligned(q, 16) && wm::aligned(k, 16) && wm::aligned(v, 16) && wm::aligned(out, 16),
             "prompt attention: token rows must be 16-byte aligned and hold their heads");
  const PromptArgs a{q, k, v, q_stride, k_stride, v_stride, cu_seqlens_q, cu_seqlens_k, B, Tq, Tk, Hq, Hkv, causal,
                     scale * kLog2e, out, lse};
  const int64_t want = (static_cast<int64_t>(Tq) * Hq + 7) / 8;
  const int grid = static_cast<int>(std::min<int64_t>(want, static_cast<int64_t>(wm::sm_count()) * 64));
  if (D == 64) k_attn_prompt_rows<64><<<grid, 256, 0, stream>>>(a);
  else if (D == 128) k_attn_prompt_rows<128><<<grid, 256, 0, stream>>>(a);
  else k_attn_prompt_rows<256><<<grid, 256, 0, stream>>>(a);
  return wm::check_launch("wattn_prompt");
}

}  // extern "C"
