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

// Bound by the stores: 1000003 positions of 128 dimensions in fp32, 512 MB, 104 us, 4.9
// TB/s, and 101.5 without the arithmetic (1829 with library functions in 64 bits for
// every value).  A thread has N pairs of every step-th position and their
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

// Any sizes: a pair or a dimension that stays per thread, whose place costs divisions in 64
// bits.  8192 tokens of 32 heads of 80, 20 turning, bfloat16, 61 us, 1.4 TB/s (32 turning, by
// sixteens, 17 to 19 us); 64 tokens 2.9, the launch.
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

// Sixteen values a thread and head (RotateHeads).  Bound by memory.
// 2 x 40 x 8191 x 128 fp16, us, one head a thread | two | four | eight: 77 | 71 | 73 | 77.
// Stores go past the caches where each is of whole lines (`stream`), past them | not:
// 62.9 | 69.1 interleaved, half of the head turning, 65.2 | 71.5 in halves, all of it; not
// where half of it turns in halves, lines in two pieces: 77.2 | 72.0.
template <int DT, int HEADS, bool INTER>
__global__ __launch_bounds__(256) void RotaryKernel(const RotaryParams p, int groups, int per_block, bool stream) {
  const int r = threadIdx.x / groups, g = threadIdx.x % groups;
  const int64_t token = (p.first + blockIdx.x) * per_block + r;
  if (r >= per_block || token >= p.tokens) return;
  int64_t at = token * p.heads * p.D, pitch = p.D;
  if (p.by_head) {
    const int64_t b = p.tokens <= 0x7fffffff ? (unsigned)token / (unsigned)p.seq : token / p.seq;
    at = (b * p.heads * p.seq + (token - b * p.seq)) * p.D;
    pitch = p.seq * p.D;
  }
  RotateHeads<DT, HEADS, INTER>(p.t, p.x, at, pitch, p.y, at, pitch, blockIdx.y * HEADS, 1, p.heads, p.D, g,
                                RotaryRow(p.t, token, token), stream);
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
