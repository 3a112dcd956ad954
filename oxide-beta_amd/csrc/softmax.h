// softmax.h -- what the losses over rows of logits share (internal to the library).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace oxh {
namespace softmax {

// evaluation.rs:622-636: finite, non-negative, integral and below `classes`.
__device__ __forceinline__ bool target_index(float t, uint64_t classes, uint64_t &index) {
  if (!isfinite(t) || t < 0.0f || t - truncf(t) != 0.0f) return false;
  if (t >= 18446744073709551616.0f) return false;
  const uint64_t i = static_cast<uint64_t>(t);
  if (i >= classes) return false;
  index = i;
  return true;
}

// exp(d) for d = x - rowmax <= 0, within ~1.5 ulp: 2^(d * log2 e) with the product carried as
// hi + lo (an exact fma residual plus d times the tail of log2 e), the hardware 2^x (v_exp_f32,
// 1 ulp) on the fraction |f| <= 0.5 + 2^-24, and the integer part applied by ldexp.  NaN
// propagates; d below -200 (including -inf) gives 0, as expf does.
__device__ __forceinline__ float exp_nonpos(float d) {
  constexpr float kLog2eHi = 1.44269502162933349609375f;  // nearest float to log2(e)
  constexpr float kLog2eLo = 1.925963033500011e-08f;      // log2(e) - kLog2eHi
  d = d < -200.0f ? -200.0f : d;
  const float hi = d * kLog2eHi;
  const float lo = fmaf(d, kLog2eLo, fmaf(d, kLog2eHi, -hi));
  const float n = rintf(hi);
  const float f = (hi - n) + lo;  // hi - n is exact
  return ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n));
}

}  // namespace softmax
}  // namespace oxh
