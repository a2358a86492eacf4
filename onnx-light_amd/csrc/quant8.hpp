// Scales and codes of blocks quantized on the device, shared by the RMS norm,
// the MX quantizer and the key / value cache.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace onnxl_amd {

constexpr float kInt8Max = 127.f, kFp8Max = 448.f;
constexpr float kMinNormal = 0x1p-126f;

// The scale of a block: codes are round(y * inv) and stand for code * scale.
struct BlockScale {
  float scale, inv;
  uint8_t e8m0;
};

// scale = top / qmax, inv = 1 / scale.  A scale below the smallest normal
// number counts as zero, with zero codes (its inverse would overflow); a top
// that is not finite gives a NaN scale, again with zero codes.
__device__ __forceinline__ BlockScale ScaleOf(float top, float qmax) {
  BlockScale s{top / qmax, 0.f, 0};
  if (!(top < __builtin_huge_valf()))
    s.scale = __builtin_nanf("");
  else if (s.scale < kMinNormal)
    s.scale = 0.f;
  else
    s.inv = 1.f / s.scale;
  return s;
}

// E8M0: e = floor(log2 top) - emax (the exponent of the element type's
// largest value: 8 for E4M3, 2 for E2M1), at least -127, stored as e + 127; a
// top that is not finite gives 255, the format's NaN, with zero codes.  A
// power of two scales a value exactly, so the codes have a single rounding.
__device__ __forceinline__ BlockScale MxScaleOf(float top, int emax) {
  const int biased = (int)(__builtin_bit_cast(uint32_t, top) >> 23);  // top >= 0
  if (biased == 255) return BlockScale{__builtin_nanf(""), 0.f, 255};
  // a subnormal top (biased 0) is below 2^-126: its e is below -127 too
  const int e = biased > emax ? biased - emax : 0;
  const float scale = e ? __builtin_bit_cast(float, (uint32_t)e << 23) : 0x1p-127f;
  const float inv = __builtin_bit_cast(float, (uint32_t)(254 - e) << 23);
  return BlockScale{scale, inv, (uint8_t)e};
}

// Nearest code, ties to even; v is finite, or 0 * NaN in a block without a
// finite scale, whose codes are 0.
__device__ __forceinline__ uint8_t Int8Code(float v) {
  const float c = __builtin_rintf(fminf(fmaxf(v, -kInt8Max), kInt8Max));
  return v == v ? (uint8_t)(int8_t)(int)c : 0;
}

// Two E4M3 codes in bits 0-15: the conversion gives NaN past 464, so values
// are clamped to the largest first.
__device__ __forceinline__ unsigned Fp8Codes2(float a, float b) {
  a = a == a ? __builtin_amdgcn_fmed3f(a, -kFp8Max, kFp8Max) : 0.f;
  b = b == b ? __builtin_amdgcn_fmed3f(b, -kFp8Max, kFp8Max) : 0.f;
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
__device__ __forceinline__ uint8_t Fp8Code(float v) { return (uint8_t)Fp8Codes2(v, 0.f); }

// Two E2M1 codes in bits 0-7, saturating, ties to even.
__device__ __forceinline__ unsigned Fp4Codes2(float a, float b) {
  a = a == a ? a : 0.f;
  b = b == b ? b : 0.f;
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, 1.f, 0) & 0xffu;
}

}  // namespace onnxl_amd
