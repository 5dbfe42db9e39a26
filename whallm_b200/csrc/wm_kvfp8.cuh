// The e4m3 KV row quantizer, shared by the row kernels (formats.cu, where its
// arithmetic is explained) and the paged cache's append (kv_paged.cu).  Both are
// compiled with -fmad=false: the bytes and scales are the same wherever a row is
// quantized.
#pragma once

#include "wm_common.cuh"

namespace wm_kv {

constexpr float kFp8MaxInv = 0x1.24924ap-9f;  // float32(1/448)  (fakequant.py:34)
constexpr float kFp8Floor = 0x1.a36e2ep-14f;  // float32(1e-4)   (packed_cache.py:34)

// floor(log2 a) for positive finite a (subnormals included) == Swift Float.exponent
__device__ __forceinline__ int floor_log2(float a) {
  uint32_t b = __float_as_uint(a);
  uint32_t ex = (b >> 23) & 255u;
  if (ex != 0) return static_cast<int>(ex) - 127;
  uint32_t m = b & 0x7fffffu;
  return (31 - __clz(static_cast<int>(m))) - 149;
}

// 2^k as float for k in [-149, 127], exact
__device__ __forceinline__ float pow2i(int k) {
  if (k >= -126) return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
  return __uint_as_float(1u << (k + 149));
}

// ceil(log2 x) via IEEE bits for positive normal x (fakequant.py:47-52)
__device__ __forceinline__ int ceil_log2_bits(float x) {
  uint32_t b = __float_as_uint(x);
  int e = static_cast<int>((b >> 23) & 255u) - 127;
  return e + ((b & 0x7fffffu) != 0 ? 1 : 0);
}

template <int FMT>
struct Fp8Fmt {
  static constexpr int kG = FMT == WKV_FP8_F32_B64 ? 8 : 4;   // threads per scale block
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}

__device__ __forceinline__ float clamp448(float q) { return fminf(fmaxf(q, -448.0f), 448.0f); }

// NV (8 or 16) consecutive values of one thread; i indexes NV-value chunks.
template <int FMT, int NV>
__device__ __forceinline__ void kv_fp8_quant(const uint4 (&u)[NV / 8], int64_t i, unsigned gmask, int lane,
                                             uint8_t *__restrict__ payload, void *__restrict__ scales) {
  constexpr int G = Fp8Fmt<FMT>::kG * 8 / NV;   // threads per scale block
  float v[NV];
#pragma unroll
  for (int k = 0; k < NV / 8; ++k) {
    v[8 * k + 0] = wm_bf16lo(u[k].x); v[8 * k + 1] = wm_bf16hi(u[k].x);
    v[8 * k + 2] = wm_bf16lo(u[k].y); v[8 * k + 3] = wm_bf16hi(u[k].y);
    v[8 * k + 4] = wm_bf16lo(u[k].z); v[8 * k + 5] = wm_bf16hi(u[k].z);
    v[8 * k + 6] = wm_bf16lo(u[k].w); v[8 * k + 7] = wm_bf16hi(u[k].w);
  }
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) amax = fmaxf(amax, fabsf(v[j]));
#pragma unroll
  for (int m = 1; m < G; m <<= 1) amax = fmaxf(amax, __shfl_xor_sync(gmask, amax, m));
  const bool first = (lane & (G - 1)) == 0;
  float q[NV];
  if (FMT == WKV_FP8_F32_B64) {
    // Quotients by Markstein's correction: with y = RN(1/b) and q0 = RN(a * y)
    // within an ulp of a / b, the remainder a - q0 * b is exact in one fma and
    // RN(q0 + rem * y) is the correctly rounded a / b, as long as the remainder
    // does not underflow -- true for blocks whose maximum is at least 2^-80
    // (quotients below 2^-10, the only ones whose remainders could, encode to
    // a signed zero either way).  Smaller blocks divide exactly.  The sign is
    // the value's (for +-0); .satfinite saturates as the clamp to +-448 did.
    if (amax >= 0x1p-80f) {
      const float s0 = amax * kFp8MaxInv;
      const float s = fmaf(fmaf(-s0, 448.0f, amax), kFp8MaxInv, s0);     // RN(amax / 448)
      if (first) static_cast<float *>(scales)[i / G] = s;
      const float r = __frcp_rn(s);
      // value pairs on packed f32x2 arithmetic: each lane rounds as the scalar mul / fma do
      const float2 r2 = make_float2(r, r), ns2 = make_float2(-s, -s);
#pragma unroll
      for (int j = 0; j < NV; j += 2) {
        const float2 vv = make_float2(v[j], v[j + 1]);
        const float2 q0 = wm_mul2(vv, r2);
        const float2 qq = wm_fma2(wm_fma2(q0, ns2, vv), r2, q0);
        q[j] = __uint_as_float((__float_as_uint(qq.x) & 0x7fffffffu) | (__float_as_uint(v[j]) & 0x80000000u));
        q[j + 1] = __uint_as_float((__float_as_uint(qq.y) & 0x7fffffffu) | (__float_as_uint(v[j + 1]) & 0x80000000u));
      }
    } else {
      const float s = __fdiv_rn(amax, 448.0f);
      if (first) static_cast<float *>(scales)[i / G] = s;
#pragma unroll
      for (int j = 0; j < NV; ++j) q[j] = s > 0.0f ? clamp448(__fdiv_rn(v[j], s)) : 0.0f;
    }
  } else if (FMT == WKV_FP8_UE8M0_B32) {
    const int e = ceil_log2_bits(fmaxf(amax, kFp8Floor) * kFp8MaxInv);
    if (first) static_cast<uint8_t *>(scales)[i / G] = static_cast<uint8_t>(e + 127);
    const float f = pow2i(-e);
#pragma unroll
    for (int j = 0; j < NV; ++j) q[j] = clamp448(v[j] * f);
  } else {
    const bool zero = amax == 0.0f;
    const int e = zero ? 0 : max(-127, min(127, floor_log2(amax) - 8));
    if (first) static_cast<uint8_t *>(scales)[i / G] = zero ? 0 : static_cast<uint8_t>(e + 127);
    const float f = pow2i(-e);
#pragma unroll
    for (int j = 0; j < NV; ++j) q[j] = zero ? 0.0f : clamp448(v[j] * f);
  }
  uint32_t w[NV / 4];
#pragma unroll
  for (int k = 0; k < NV / 4; ++k) w[k] = e4m3x2(q[4 * k], q[4 * k + 1]) | (e4m3x2(q[4 * k + 2], q[4 * k + 3]) << 16);
  if constexpr (NV == 16) __stcs(reinterpret_cast<uint4 *>(payload) + i, make_uint4(w[0], w[1], w[2], w[3]));
  else __stcs(reinterpret_cast<uint2 *>(payload) + i, make_uint2(w[0], w[1]));
}

}  // namespace wm_kv
