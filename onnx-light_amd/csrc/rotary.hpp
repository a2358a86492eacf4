// Rotation of a head's dimensions by position, shared by the rotary embedding
// and the cache's append.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"

namespace onnxl_amd {

// The table row of token `row`, -1 where its position has none.
__device__ __forceinline__ int64_t RotaryRow(const RotaryTable &t, int64_t row, int64_t without_ids) {
  int64_t p = without_ids;
  if (t.ids) p = t.ids64 ? static_cast<const int64_t *>(t.ids)[row] : (int64_t) static_cast<const int32_t *>(t.ids)[row];
  return p >= 0 && p < t.positions ? p : -1;
}

// N consecutive values of type DT as floats.
template <int DT, int N> __device__ __forceinline__ void Widen(const void *base, int64_t at, float (&v)[N]) {
  if constexpr (DT == kFloat) {
    __builtin_memcpy(v, static_cast<const float *>(base) + at, 4 * N);
  } else {
    uint16_t u[N];
    __builtin_memcpy(u, static_cast<const uint16_t *>(base) + at, 2 * N);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = DT == kFloat16 ? F16ToF32(u[i]) : Bf16ToF32(u[i]);
  }
}

// N values of the tables from pair i of row `pos` on; NaN where there is no row.
template <int DT, int N>
__device__ __forceinline__ void TableValues(const RotaryTable &t, int64_t pos, int i, float (&c)[N], float (&s)[N]) {
  if (pos < 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) c[j] = s[j] = __builtin_nanf("");
    return;
  }
  const int64_t at = pos * t.half + i;
  if (t.f32) {
    Widen<kFloat, N>(t.cos, at, c);
    Widen<kFloat, N>(t.sin, at, s);
  } else {
    Widen<DT, N>(t.cos, at, c);
    Widen<DT, N>(t.sin, at, s);
  }
}

}  // namespace onnxl_amd
