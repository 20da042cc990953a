// Scale rule of the block-scaled e4m3 quantisation, shared by the quantisation
// kernels and the norm that quantises its output.
#pragma once

#include "common.cuh"

namespace rlb {

constexpr float kFp8Max = 448.f;

// Smallest power of two >= s (s > 0, finite): bump the exponent when any
// mantissa bit is set.
__device__ __forceinline__ float pow2_ceil(float s) {
  uint32_t b = __float_as_uint(s);
  if (b & 0x007fffffu) {
    b = (b & 0xff800000u) + 0x00800000u;
  }
  return __uint_as_float(b & 0xff800000u);
}

__device__ __forceinline__ float fp8_scale(float amax, bool pow2) {
  float s = fmaxf(amax, 1e-12f) / kFp8Max;
  return pow2 ? pow2_ceil(s) : s;
}

}  // namespace rlb
