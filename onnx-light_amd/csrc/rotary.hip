// Rotary positions: the tables of cosines and sines, and the rotation.
#include "rotary.hpp"

namespace onnxl_amd {
namespace {

constexpr double kTwoPi = 6.283185307179586476925;

// Angle per position of pair i, in turns.
__device__ __forceinline__ double TurnsPerPosition(const RotaryTablesParams &p, int i) {
  const double f = exp(-(double)i / p.half * p.log_base);
  double keep = 1.0;  // the share of the frequency that stays; the rest is divided by the factor
  if (p.scaling == kRotaryLinear) keep = 0.0;
  if (p.scaling == kRotaryByParts) keep = (p.original * f / kTwoPi - p.turns_slow) / (p.turns_fast - p.turns_slow);
  if (p.scaling == kRotaryYarn) keep = 1.0 - (i - p.low) / fmax(p.high - p.low, 0.001);
  keep = fmin(fmax(keep, 0.0), 1.0);
  return (keep == 1.0 ? f : f * keep + f / p.factor * (1.0 - keep)) / kTwoPi;
}

// Cosine and sine of an angle in turns: the nearest quarter turn is taken off in 64
// bits, so that far positions lose nothing, and what is left, at most an eighth, has
// its series in fp32 (the first terms left out are 2e-9 and 2e-10).
__device__ __forceinline__ void CosSin(double turns, float &c, float &s) {
  const double quarters = rint(4.0 * turns);
  const float x = (float)((turns - 0.25 * quarters) * kTwoPi), z = x * x;
  const float si = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float co = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
  const int q = (int)quarters & 3;  // positions are below 2^31, a position at most 1 / (2 pi) turns
  const float a = q & 1 ? si : co, b = q & 1 ? co : si;
  c = q == 1 || q == 2 ? -a : a;
  s = q >= 2 ? -b : b;
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

// Bound by the stores.  A thread has N pairs of every step-th position and their
// frequencies in registers; the threads of a position write its rows in one piece.
template <int DT, int N> __global__ __launch_bounds__(256) void RotaryTablesKernel(const RotaryTablesParams p, int per_row) {
  const int rows = 256 / per_row, r = threadIdx.x / per_row, i = (blockIdx.y * per_row + threadIdx.x % per_row) * N;
  if (r >= rows || i >= p.half) return;
  double turns[N];
#pragma unroll
  for (int j = 0; j < N; ++j) turns[j] = TurnsPerPosition(p, i + j);
  const int64_t step = (int64_t)gridDim.x * rows, first = (int64_t)blockIdx.x * rows + r;
  double place = (double)first;
  for (int64_t pos = first; pos < p.positions; pos += step, place += (double)step) {
    float c[N], s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      CosSin(place * turns[j], c[j], s[j]);
      c[j] *= p.magnitude;
      s[j] *= p.magnitude;
    }
    Narrow<DT, N>(p.cos, pos * p.half + i, c);
    Narrow<DT, N>(p.sin, pos * p.half + i, s);
  }
}

// Any sizes: a pair or a dimension that stays per thread.
template <int DT> __global__ __launch_bounds__(256) void RotaryAnyKernel(const RotaryParams p) {
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
    Narrow<DT, 1>(p.y, at + p.t.half + j, v);
    return;
  }
  const int64_t ia = at + (p.t.interleaved ? 2 * j : j), ib = p.t.interleaved ? ia + 1 : ia + p.t.half;
  float a[1], b[1], c[1], s[1];
  Widen<DT, 1>(p.x, ia, a);
  Widen<DT, 1>(p.x, ib, b);
  TableValues<DT, 1>(p.t, RotaryRow(p.t, token, token), j, c, s);
  const float ya[1] = {a[0] * c[0] - b[0] * s[0]}, yb[1] = {a[0] * s[0] + b[0] * c[0]};
  Narrow<DT, 1>(p.y, ia, ya);
  Narrow<DT, 1>(p.y, ib, yb);
}

// Sixteen values a thread and head: eight pairs (i, d / 2 + i) or as many dimensions
// that stay; where pairs are neighbours two eights half the head apart, each of which
// turns or stays, so that the loads and the stores of neighbouring threads are one
// piece.  Bound by memory: a thread takes its part of the token's table rows once for
// HEADS heads, whose values are all on their way before the first is turned.
// 2 x 40 x 8191 x 128 fp16, us, one head a thread | two | four | eight: 77 | 71 | 73 | 77.
// Stores go past the caches where each is of whole lines (`stream`), past them | not:
// 62.9 | 69.1 interleaved, half of the head turning, 65.2 | 71.5 in halves, all of it; not
// where half of it turns in halves, lines in two pieces: 77.2 | 72.0.
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
template <int DT, int HEADS, bool INTER>
__global__ __launch_bounds__(256) void RotaryKernel(const RotaryParams p, int groups, int per_block, bool stream) {
  const int r = threadIdx.x / groups, g = threadIdx.x % groups;
  const int64_t token = (p.first + blockIdx.x) * per_block + r;
  if (r >= per_block || token >= p.tokens) return;
  const int turning = p.t.half / 8, h0 = blockIdx.y * HEADS;
  const bool turns = INTER ? 8 * g < 2 * p.t.half : g < turning;  // the first eight, and so anything
  if (!turns && p.x == p.y) return;
  const int da = INTER || turns ? 8 * g : 2 * p.t.half + 8 * (g - turning);
  const int db = da + (INTER ? p.D / 2 : turns ? p.t.half : p.D / 2 - p.t.half);
  int64_t at = token * p.heads * p.D, pitch = p.D;
  if (p.by_head) {
    const int64_t b = p.tokens <= 0x7fffffff ? (unsigned)token / (unsigned)p.seq : token / p.seq;
    at = (b * p.heads * p.seq + (token - b * p.seq)) * p.D;
    pitch = p.seq * p.D;
  }
  Sixteen v[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const int64_t row = at + min(h0 + h, p.heads - 1) * pitch;
    Widen<DT, 8>(p.x, row + da, v[h].a);
    Widen<DT, 8>(p.x, row + db, v[h].b);
  }
  if (turns) {
    const int64_t pos = RotaryRow(p.t, token, token);
    if constexpr (INTER) {
      TurnEight<DT, HEADS, false>(p.t, pos, da, v);
      TurnEight<DT, HEADS, true>(p.t, pos, db, v);
    } else {
      float c[8], s[8];
      TableValues<DT, 8>(p.t, pos, 8 * g, c, s);
#pragma unroll
      for (int h = 0; h < HEADS; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) Turn(v[h].a[i], v[h].b[i], c[i], s[i]);
    }
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (h0 + h >= p.heads) break;
    const int64_t row = at + (h0 + h) * pitch;
    if (stream) {
      NarrowStream<DT>(p.y, row + da, v[h].a);
      NarrowStream<DT>(p.y, row + db, v[h].b);
    } else {
      Narrow<DT, 8>(p.y, row + da, v[h].a);
      Narrow<DT, 8>(p.y, row + db, v[h].b);
    }
  }
}

template <int DT, int HEADS> void LaunchHeads(RotaryParams p, int groups, hipStream_t st) {
  const int per_block = 256 / groups, line = 128 / (DT == kFloat ? 4 : 2);
  // the runs of a head that its threads write at once: whole lines of an aligned y
  const bool runs = p.t.interleaved ? p.D / 2 % line == 0 : p.t.half % line == 0 && (p.D / 2 - p.t.half) % line == 0;
  const bool stream = HEADS > 1 && runs && reinterpret_cast<uintptr_t>(p.y) % 128 == 0;
  LaunchInPieces((p.tokens + per_block - 1) / per_block, 256, [&](int64_t first, unsigned count) {
    p.first = first;
    const dim3 grid(count, (unsigned)((p.heads + HEADS - 1) / HEADS));
    if (p.t.interleaved)
      RotaryKernel<DT, HEADS, true><<<grid, 256, 0, st>>>(p, groups, per_block, stream);
    else
      RotaryKernel<DT, HEADS, false><<<grid, 256, 0, st>>>(p, groups, per_block, stream);
  });
}

template <int DT> void LaunchTables(const RotaryTablesParams &p, hipStream_t stream) {
  const bool four = p.half % 4 == 0;
  const int pairs = four ? p.half / 4 : p.half, per_row = std::min(pairs, 256), rows = 256 / per_row;
  const int64_t blocks = (p.positions + rows - 1) / rows;
  // enough to fill the chip; more positions go round, with the frequencies kept
  const dim3 grid((unsigned)std::min<int64_t>(blocks, 8 * 256), (unsigned)((pairs + per_row - 1) / per_row));
  if (four)
    RotaryTablesKernel<DT, 4><<<grid, 256, 0, stream>>>(p, per_row);
  else
    RotaryTablesKernel<DT, 1><<<grid, 256, 0, stream>>>(p, per_row);
}

template <int DT> void LaunchRotation(RotaryParams p, hipStream_t stream) {
  const int d = 2 * p.t.half, groups = d / 16 + (p.D - d) / 16;
  if (d % 16 == 0 && p.D % 16 == 0 && groups <= 256 && p.heads < 65536) {
    // Two heads a thread where that leaves every CU eight waves a SIMD.
    if (p.tokens * groups * p.heads >= 4 * 256 * 1024)
      LaunchHeads<DT, 2>(p, groups, stream);
    else
      LaunchHeads<DT, 1>(p, groups, stream);
    return;
  }
  const int64_t threads = p.tokens * p.heads * (p.D - p.t.half);
  LaunchInPieces((threads + 255) / 256, 256, [&](int64_t first, unsigned count) {
    p.first = first;
    RotaryAnyKernel<DT><<<count, 256, 0, stream>>>(p);
  });
}

}  // namespace

void LaunchRotaryTables(const RotaryTablesParams &p, hipStream_t stream) {
  if (p.dtype == kFloat)
    LaunchTables<kFloat>(p, stream);
  else if (p.dtype == kFloat16)
    LaunchTables<kFloat16>(p, stream);
  else
    LaunchTables<kBfloat16>(p, stream);
}

void LaunchRotaryEmbedding(const RotaryParams &p, hipStream_t stream) {
  if (p.dtype == kFloat)
    LaunchRotation<kFloat>(p, stream);
  else if (p.dtype == kFloat16)
    LaunchRotation<kFloat16>(p, stream);
  else
    LaunchRotation<kBfloat16>(p, stream);
}

}  // namespace onnxl_amd
