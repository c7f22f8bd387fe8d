// The factor of clipped gradients, scale * coefficient, for grad_clip.cu and the clipped sweep of sgd_fused.cu.
#pragma once
#include <cuda_runtime.h>

namespace rb {

// A value is taken times `back`, then times `by`. A product below the normal numbers of fp32 would have lost bits that matter where
// values are above 2^100: it is made 2^64 times as large and `back` is 2^-64, which loses nothing of values that large; else 1.
struct ClipFactor {
  float by, back;
};
__device__ __forceinline__ ClipFactor clip_factor(float scale, float coef) {
  const float f = scale * coef;
  if (fabsf(f) >= 0x1p-126f) return {f, 1.f};
  return {scale * 0x1p64f * coef, 0x1p-64f};
}

}  // namespace rb
