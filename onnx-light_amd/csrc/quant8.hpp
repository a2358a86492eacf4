// Scales and codes of blocks quantized on the device, shared by the RMS norm,
// the MX quantizer and the key / value cache.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace onnxl_amd {

constexpr float kInt8Max = 127.f, kFp8Max = 448.f;
constexpr float kMinNormal = 0x1p-126f;

// The scale of a block: codes are round(y * inv) and stand for code * scale.  With a
// FLOAT scale inv and the product are rounded, to within 2^-23 of y / scale, so a
// quotient that near the middle between two codes may take either of them; of
// 16-bit values exact middles are no rarity (y qmax / max), and these roundings
// decide them, not ties to even.  A division per value would take ten instructions
// for one.
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

// Nearest codes, ties to even, of v = y * inv of a block with a FLOAT scale.
// |v| is at most the largest code (and an ulp), which no rounding leaves.  In a
// block whose scale is NaN v may be NaN: its codes mean nothing.
__device__ __forceinline__ unsigned Int8Codes4(float a, float b, float c, float d) {
  const unsigned lo = __builtin_amdgcn_perm((unsigned)(int)__builtin_rintf(b), (unsigned)(int)__builtin_rintf(a), 0x0c0c0400u);
  const unsigned hi = __builtin_amdgcn_perm((unsigned)(int)__builtin_rintf(d), (unsigned)(int)__builtin_rintf(c), 0x04000c0cu);
  return lo | hi;
}
__device__ __forceinline__ unsigned Fp8Codes4(float a, float b, float c, float d) {
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// MX blocks: v = x * 2^-e may pass the largest code, and the conversion gives
// NaN past 464, so it is clamped.
__device__ __forceinline__ float ClampFp8(float v) { return __builtin_amdgcn_fmed3f(v, -kFp8Max, kFp8Max); }

// Two E2M1 codes in bits 0-7, saturating.
__device__ __forceinline__ unsigned Fp4Codes2(float a, float b) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, 1.f, 0) & 0xffu;
}

// Codes of eight values of an MX block; a block without a finite scale has zero
// codes.
__device__ __forceinline__ uint2 MxFp8Codes8(const float (&v)[8], const BlockScale &s) {
  float c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = ClampFp8(v[j] * s.inv);
  const bool none = s.e8m0 == 255;
  return make_uint2(none ? 0u : Fp8Codes4(c[0], c[1], c[2], c[3]), none ? 0u : Fp8Codes4(c[4], c[5], c[6], c[7]));
}
__device__ __forceinline__ unsigned MxFp4Codes8(const float (&v)[8], const BlockScale &s) {
  unsigned c = 0;
#pragma unroll
  for (int j = 0; j < 8; j += 2) c |= Fp4Codes2(v[j] * s.inv, v[j + 1] * s.inv) << (4 * j);
  return s.e8m0 == 255 ? 0u : c;
}

}  // namespace onnxl_amd
