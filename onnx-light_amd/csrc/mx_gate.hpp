// The activation of a gated product, shared by the streaming kernel and the GEMM.
#pragma once

#include <hip/hip_runtime.h>

#include "decoder.hpp"

namespace onnxl_amd {
namespace mx {

// In fp32, from the hardware's exponential and reciprocal (an ulp each).  An exponent is
// rounded as a number of its size, |g| for SiLU and about g^2 for the others, so the result's
// relative error grows with it, to 2^-19 (1 + g^2) at most, and past e^87 it is 0; 16 or 8 bits
// hide it where the result is not many orders below the largest.  A NaN stays one.
__device__ __forceinline__ float Activate(float g, int kind) {
  constexpr float kLog2e = 1.44269504f;
  if (kind == kRelu) return g < 0.f ? 0.f : g;
  // 0.5 g (1 + erf(g / sqrt 2)), without the difference that cancels for g < 0
  if (kind == kGelu) return 0.5f * g * erfcf(-0.70710678f * g);
  // 0.5 (1 + tanh v) = 1 / (1 + e^-2v)
  const float v = kind == kSilu ? g : 1.59576912f * (g + 0.044715f * g * g * g);
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
}

}  // namespace mx
}  // namespace onnxl_amd
