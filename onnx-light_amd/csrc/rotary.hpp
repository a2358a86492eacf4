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

template <int DT, int N> __device__ __forceinline__ void Narrow(void *base, int64_t at, const float (&v)[N]) {
  if constexpr (DT == kFloat) {
    __builtin_memcpy(static_cast<float *>(base) + at, v, 4 * N);
  } else {
    uint16_t u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = DT == kFloat16 ? F32ToF16(v[i]) : F32ToBf16(v[i]);
    __builtin_memcpy(static_cast<uint16_t *>(base) + at, u, 2 * N);
  }
}

// The same past the caches: only for whole lines at a time.
template <int DT> __device__ __forceinline__ void NarrowStream(void *base, int64_t at, const float (&v)[8]) {
  constexpr int W = DT == kFloat ? 2 : 1;
  typedef unsigned w4u __attribute__((ext_vector_type(4), aligned(2)));
  w4u r[W];
#pragma unroll
  for (int i = 0; i < 4 * W; ++i) {
    if constexpr (DT == kFloat)
      r[i / 4][i % 4] = __builtin_bit_cast(unsigned, v[i]);
    else
      r[0][i] = DT == kFloat16 ? F32ToF16(v[2 * i]) | (unsigned)F32ToF16(v[2 * i + 1]) << 16
                               : F32ToBf16(v[2 * i]) | (unsigned)F32ToBf16(v[2 * i + 1]) << 16;
  }
  char *y = static_cast<char *>(base) + at * (DT == kFloat ? 4 : 2);
#pragma unroll
  for (int i = 0; i < W; ++i) __builtin_nontemporal_store(r[i], reinterpret_cast<w4u *>(y + 16 * i));
}

// Sixteen values a thread and head: eight pairs (i, d / 2 + i) or as many dimensions
// that stay; where pairs are neighbours two eights half the head apart, each of which
// turns or stays, so that the loads and the stores of neighbouring threads are one
// piece.  A thread takes its part of the token's table rows once for HEADS heads, whose
// values are all on their way before the first is turned.
struct Sixteen {
  float a[8], b[8];
};
__device__ __forceinline__ void Turn(float &a, float &b, float c, float s) {
  const float t = a * c - b * s;
  b = a * s + b * c;
  a = t;
}
// four neighbouring pairs, from dimension `dim` on
template <int DT, int HEADS, bool B>
__device__ __forceinline__ void TurnEight(const RotaryTable &t, int64_t pos, int dim, Sixteen (&v)[HEADS]) {
  if (dim >= 2 * t.half) return;
  float c[4], s[4];
  TableValues<DT, 4>(t, pos, dim / 2, c, s);
#pragma unroll
  for (int h = 0; h < HEADS; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float *x = B ? v[h].b : v[h].a;
      Turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
    }
}

// Part g of D / 16 of the heads first, first + step, .. (HEADS of them, below `heads`) of a
// token, which begin at xat + head * xpitch of x, and so of y; d and D are multiples of 16.
template <int DT, int HEADS, bool INTER>
__device__ __forceinline__ void RotateHeads(const RotaryTable &t, const void *x, int64_t xat, int64_t xpitch, void *y, int64_t yat,
                                            int64_t ypitch, int first, int step, int heads, int D, int g, int64_t pos, bool stream) {
  const int turning = t.half / 8;
  const bool turns = INTER ? 8 * g < 2 * t.half : g < turning;  // the first eight, and so anything
  if (!turns && x == y) return;
  const int da = INTER || turns ? 8 * g : 2 * t.half + 8 * (g - turning);
  const int db = da + (INTER ? D / 2 : turns ? t.half : D / 2 - t.half);
  Sixteen v[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const int64_t row = xat + min(first + h * step, heads - 1) * xpitch;
    Widen<DT, 8>(x, row + da, v[h].a);
    Widen<DT, 8>(x, row + db, v[h].b);
  }
  if (turns) {
    if constexpr (INTER) {
      TurnEight<DT, HEADS, false>(t, pos, da, v);
      TurnEight<DT, HEADS, true>(t, pos, db, v);
    } else {
      float c[8], s[8];
      TableValues<DT, 8>(t, pos, 8 * g, c, s);
#pragma unroll
      for (int h = 0; h < HEADS; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) Turn(v[h].a[i], v[h].b[i], c[i], s[i]);
    }
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (first + h * step >= heads) break;
    const int64_t row = yat + (first + h * step) * ypitch;
    if (stream) {
      NarrowStream<DT>(y, row + da, v[h].a);
      NarrowStream<DT>(y, row + db, v[h].b);
    } else {
      Narrow<DT, 8>(y, row + da, v[h].a);
      Narrow<DT, 8>(y, row + db, v[h].b);
    }
  }
}

}  // namespace onnxl_amd
