// What a kernel leaves behind when one of its bounded waits ran out (internal
// header; also compiled for the host by the tests).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace wm_giveup {

// Thread `first` of `step`: NaN in every output of an attention call -- out in
// bf16, lse (may be null) and the sums of the parts (may be null) -- so that no
// element which the call did not come to passes for a result.
__host__ __device__ inline void poison(uint16_t *out, int64_t n_out, float *lse, int64_t n_lse, float2 *part_ml, int64_t n_parts,
                                       int first, int step) {
  const float nan = __builtin_nanf("");
  for (int64_t i = first; i < n_out; i += step) out[i] = 0x7FC0;
  if (lse)
    for (int64_t i = first; i < n_lse; i += step) lse[i] = nan;
  if (part_ml)
    for (int64_t i = first; i < n_parts; i += step) part_ml[i] = make_float2(0.0f, nan);
}

}  // namespace wm_giveup
