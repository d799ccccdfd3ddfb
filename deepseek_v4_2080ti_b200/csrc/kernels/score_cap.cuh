// The cap of attention scores: s -> tanh(k s), relative error below 1e-6 (NaN stays).  The quotient alone would lose what is small against 1.
#pragma once
#include <cuda_runtime.h>

namespace b200 {

// Where |k s| <= 1: z P(z^2), P an interpolation of tanh(z) / z at six Chebyshev points.
__device__ __forceinline__ float score_cap_small(float s, float k) {
  const float z = s * k, u = z * z;
  float y = fmaf(u, -0.0030582291074097f, 0.0167208556085825f);
  y = fmaf(y, u, -0.0515859872102737f);
  y = fmaf(y, u, 0.1328072100877762f);
  y = fmaf(y, u, -0.3332895040512085f);
  return fmaf(y, u, 0.9999994039535522f) * z;
}
__device__ __forceinline__ float score_cap(float s, float k) {
  const float z = s * k;
  return fabsf(z) <= 1.f ? score_cap_small(s, k) : 1.f - 2.f * __fdividef(1.f, 1.f + exp2f(z * 2.885390081777927f));
}

}  // namespace b200
