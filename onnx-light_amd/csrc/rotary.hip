// Rotary positions: the tables of cosines and sines, and the rotation.
#include "rotary.hpp"

namespace onnxl_amd {
namespace {

constexpr double kTwoPi = 6.283185307179586476925;

// Angle per position of pair i, in turns.
__device__ double TurnsPerPosition(const RotaryTablesParams &p, int i) {
  const int d = 2 * p.half;
  double base = p.base;
  if (p.scaling == kRotaryNtk) base *= pow(p.factor, (double)d / (d - 2));
  const double f = pow(base, -2.0 * i / d);
  double keep = 1.0;  // the share of the frequency that stays; the rest is divided by the factor
  if (p.scaling == kRotaryLinear) keep = 0.0;
  if (p.scaling == kRotaryByParts) keep = (p.original * f / kTwoPi - p.turns_slow) / (p.turns_fast - p.turns_slow);
  if (p.scaling == kRotaryYarn) {
    const double per = d / (2 * log(base));
    const double lo = fmax(floor(per * log(p.original / (p.turns_fast * kTwoPi))), 0.0);
    const double hi = fmin(ceil(per * log(p.original / (p.turns_slow * kTwoPi))), d - 1.0);
    keep = 1.0 - (i - lo) / fmax(hi - lo, 0.001);
  }
  keep = fmin(fmax(keep, 0.0), 1.0);
  return (f * keep + f / p.factor * (1.0 - keep)) / kTwoPi;
}

template <int DT> __device__ __forceinline__ void Put(void *base, int64_t at, float v) {
  if constexpr (DT == kFloat)
    static_cast<float *>(base)[at] = v;
  else
    static_cast<uint16_t *>(base)[at] = DT == kFloat16 ? F32ToF16(v) : F32ToBf16(v);
}

template <int DT> __global__ __launch_bounds__(256) void RotaryTablesKernel(const RotaryTablesParams p) {
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / 1);
  const int i = blockIdx.y;
  const double turns = TurnsPerPosition(p, i);
  for (int64_t pos = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; pos < p.positions; pos += step) {
    const double t = pos * turns;
    double s, c;
    sincospi(2.0 * (t - rint(t)), &s, &c);
    Put<DT>(p.cos, pos * p.half + i, (float)(c * p.magnitude));
    Put<DT>(p.sin, pos * p.half + i, (float)(s * p.magnitude));
  }
}

// A pair or a dimension that stays per thread.
template <int DT> __global__ __launch_bounds__(256) void RotaryKernel(const RotaryParams p) {
  const int per_head = p.D - p.t.half;
  const int64_t i = (p.first + blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.tokens * p.heads * per_head) return;
  const int64_t row = i / per_head;  // of the layout
  const int j = (int)(i % per_head);
  const int64_t token = p.by_head ? row / (p.heads * p.seq) * p.seq + row % p.seq : row / p.heads;
  const int64_t at = row * p.D;
  if (j >= p.t.half) {
    float v[1];
    Widen<DT, 1>(p.x, at + p.t.half + j, v);
    Put<DT>(p.y, at + p.t.half + j, v[0]);
    return;
  }
  const int64_t ia = at + (p.t.interleaved ? 2 * j : j), ib = p.t.interleaved ? ia + 1 : ia + p.t.half;
  float a[1], b[1], c[1], s[1];
  Widen<DT, 1>(p.x, ia, a);
  Widen<DT, 1>(p.x, ib, b);
  TableValues<DT, 1>(p.t, RotaryRow(p.t, token, token), j, c, s);
  Put<DT>(p.y, ia, a[0] * c[0] - b[0] * s[0]);
  Put<DT>(p.y, ib, a[0] * s[0] + b[0] * c[0]);
}

}  // namespace

void LaunchRotaryTables(const RotaryTablesParams &p, hipStream_t stream) {
  const dim3 grid((unsigned)std::min<int64_t>((p.positions + 255) / 256, 1024), (unsigned)p.half);
  if (p.dtype == kFloat)
    RotaryTablesKernel<kFloat><<<grid, 256, 0, stream>>>(p);
  else if (p.dtype == kFloat16)
    RotaryTablesKernel<kFloat16><<<grid, 256, 0, stream>>>(p);
  else
    RotaryTablesKernel<kBfloat16><<<grid, 256, 0, stream>>>(p);
}

void LaunchRotaryEmbedding(const RotaryParams &whole, hipStream_t stream) {
  RotaryParams p = whole;
  const int64_t threads = p.tokens * p.heads * (p.D - p.t.half);
  LaunchInPieces((threads + 255) / 256, 256, [&](int64_t first, unsigned count) {
    p.first = first;
    if (p.dtype == kFloat)
      RotaryKernel<kFloat><<<count, 256, 0, stream>>>(p);
    else if (p.dtype == kFloat16)
      RotaryKernel<kFloat16><<<count, 256, 0, stream>>>(p);
    else
      RotaryKernel<kBfloat16><<<count, 256, 0, stream>>>(p);
  });
}

}  // namespace onnxl_amd
