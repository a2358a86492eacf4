// Microscaled 4-bit products: quantization of 16-bit activations to MXFP8 or
// MXFP4 and the product, plain or gated, with MXFP4 weights on the block-scaled
// matrix cores.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "mx_gemm.hpp"
#include "mx_stream.hpp"
#include "quant8.hpp"

namespace onnxl_amd {
namespace {

// Eight values per thread, four neighbouring threads per block.  Where `tiles`
// is given the output is the GEMM's (mx_gemm.hpp): scales there, rows padded to
// whole steps with zero codes of scale 1.
template <int DT, bool FP4> __device__ __forceinline__ void QuantizeRow8(const MxQuantParams &p, uint8_t *tiles, int64_t i) {
  const int64_t steps = (p.K + 255) / 256, per_row = tiles ? steps * 32 : p.K / 8, row = i / per_row, k8 = i % per_row;
  if (k8 * 8 >= p.K) {
    if constexpr (FP4)
      *reinterpret_cast<unsigned *>(p.y + i * 4) = 0;
    else
      *reinterpret_cast<uint2 *>(p.y + i * 8) = make_uint2(0, 0);
    if (k8 % 4 == 0) tiles[mx::ScaleTileAt(row, k8 / 4, steps)] = 127;
    return;
  }
  const int64_t at = row * p.K + k8 * 8;
  float v[8];
  if constexpr (DT == kFloat) {
    const float *x = static_cast<const float *>(p.x) + at;
    __builtin_memcpy(v, x, 32);
  } else {
    uint16_t u[8];
    __builtin_memcpy(u, static_cast<const uint16_t *>(p.x) + at, 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = DT == kFloat16 ? F16ToF32(u[j]) : Bf16ToF32(u[j]);
  }
  // the largest magnitude as bits: a NaN is larger than any number, and stays
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
  top = max(top, (unsigned)__shfl_xor((int)top, 1));
  top = max(top, (unsigned)__shfl_xor((int)top, 2));
  const BlockScale s = MxScaleOf(__builtin_bit_cast(float, top), FP4 ? 2 : 8);
  if constexpr (FP4)
    *reinterpret_cast<unsigned *>(p.y + i * 4) = MxFp4Codes8(v, s);
  else
    *reinterpret_cast<uint2 *>(p.y + i * 8) = MxFp8Codes8(v, s);
  if (k8 % 4 == 0) {
    if (tiles)
      tiles[mx::ScaleTileAt(row, k8 / 4, steps)] = s.e8m0;
    else
      p.scale[i / 4] = s.e8m0;
  }
}

template <int DT> __global__ __launch_bounds__(256) void MxQuantizeKernel(const MxQuantParams p) {
  const int64_t i = (p.first + blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.rows * (p.K / 8)) return;
  if (p.fp4)
    QuantizeRow8<DT, true>(p, nullptr, i);
  else
    QuantizeRow8<DT, false>(p, nullptr, i);
}

// ---------------------------------------------------------------------------
// The GEMM's operands: b's scales (and a's, where a comes as codes) in tiles,
// and a quantized where it has 16 bits, in one launch.

// Eight blocks (a step) of one row per thread; blocks past the row's end get
// the scale 1, for their codes read as zeros.
__device__ __forceinline__ void TileScales(const uint8_t *scale, uint8_t *tiles, int64_t rows, int64_t K, int64_t i) {
  const int64_t steps = (K + 255) / 256, blocks = K / 32, row = i % rows, t = i / rows;
  const uint8_t *s = scale + row * blocks + t * 8;
  uint8_t b[8];
  if (t * 8 + 8 <= blocks) {
    __builtin_memcpy(b, s, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = t * 8 + j < blocks ? s[j] : 127;
  }
  unsigned *d = reinterpret_cast<unsigned *>(tiles) + (row / 32 * steps + t) * 64 + row % 32;
  d[0] = b[0] | b[2] << 8 | b[4] << 16 | (unsigned)b[6] << 24;
  d[32] = b[1] | b[3] << 8 | b[5] << 16 | (unsigned)b[7] << 24;
}

struct MxOperands {
  MxQuantParams q;            // a to be quantized: x set
  const uint8_t *a, *a_scale, *b_scale;
  const uint8_t *up_scale;    // of the second weight of a gated product, or nullptr
  uint8_t *codes;             // a's codes with padded rows, where K is not whole steps
  uint8_t *a_tiles, *b_tiles, *up_tiles;
  int64_t M, N, K;
  int64_t b_groups;           // workgroups of b's part
  int64_t first;              // the launch's first workgroup
};

template <int DT> __global__ __launch_bounds__(256) void MxOperandsKernel(const MxOperands p) {
  const int64_t steps = (p.K + 255) / 256, group = p.first + blockIdx.x;
  if (group < p.b_groups) {
    const int64_t i = group * 256 + threadIdx.x;
    if (i < p.N * steps)
      TileScales(p.b_scale, p.b_tiles, p.N, p.K, i);
    else if (p.up_scale && i < 2 * p.N * steps)
      TileScales(p.up_scale, p.up_tiles, p.N, p.K, i - p.N * steps);
    return;
  }
  const int64_t i = (group - p.b_groups) * 256 + threadIdx.x;
  if (!p.q.x) {
    if (i < p.M * steps) TileScales(p.a_scale, p.a_tiles, p.M, p.K, i);
    if (!p.codes) return;
    const int64_t bytes = p.q.fp4 ? p.K / 2 : p.K, pitch = steps * (p.q.fp4 ? 128 : 256);
    const int64_t row = i / (pitch / 16), c = i % (pitch / 16) * 16;
    if (row >= p.M) return;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c < bytes) v = *reinterpret_cast<const uint4 *>(p.a + row * bytes + c);
    *reinterpret_cast<uint4 *>(p.codes + row * pitch + c) = v;
    return;
  }
  if (i >= p.M * steps * 32) return;
  if (p.q.fp4)
    QuantizeRow8<DT, true>(p.q, p.a_tiles, i);
  else
    QuantizeRow8<DT, false>(p.q, p.a_tiles, i);
}

}  // namespace

void LaunchMxQuantize(const MxQuantParams &whole, hipStream_t stream) {
  MxQuantParams p = whole;
  LaunchInPieces((p.rows * (p.K / 8) + 255) / 256, 256, [&](int64_t first, unsigned count) {
    p.first = first;
    if (p.x_dtype == kFloat)
      MxQuantizeKernel<kFloat><<<count, 256, 0, stream>>>(p);
    else if (p.x_dtype == kFloat16)
      MxQuantizeKernel<kFloat16><<<count, 256, 0, stream>>>(p);
    else
      MxQuantizeKernel<kBfloat16><<<count, 256, 0, stream>>>(p);
  });
}

namespace {

int64_t Ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of a product's weight, or of both weights of a gated one.
int64_t WeightRows(const MxMatMulParams &p) { return p.output ? 2 * p.N : p.N; }

// Scratch: codes (where they are not a's own) and scale tiles of a, scale tiles
// of b and of the second weight.
struct MxScratch {
  size_t codes, a_tiles, b_tiles;
  explicit MxScratch(const MxMatMulParams &p)
      : codes(p.x || p.K % 256 ? Scratch::Round((size_t)(p.M * Ceil(p.K, 256) * (p.a_fp4 ? 128 : 256))) : 0),
        a_tiles(Scratch::Round((size_t)mx::ScaleTileBytes(p.M, p.K))),
        b_tiles(Scratch::Round((size_t)mx::ScaleTileBytes(p.N, p.K))) {}
};

template <bool A4, int MB, int NB, int STAGES, int WM, int WN> void LaunchGemm(const mx::GemmArgs &g, int output, hipStream_t s) {
  using S = mx::Shape<A4, MB, NB, STAGES, WM, WN>;
  const dim3 grid((unsigned)(Ceil(g.M, S::BM) * Ceil(g.N, output ? S::BN / 2 : S::BN)));
  if constexpr (WM * WN == 8) {
    if (output == kGatedMx)
      mx::GemmKernel<A4, MB, NB, STAGES, WM, WN, kGatedMx><<<grid, 512, 0, s>>>(g);
    else if (output == kGated)
      mx::GemmKernel<A4, MB, NB, STAGES, WM, WN, kGated><<<grid, 512, 0, s>>>(g);
  }
  if (output == kPlain) mx::GemmKernel<A4, MB, NB, STAGES, WM, WN><<<grid, 64 * WM * WN, 0, s>>>(g);
}

// Large tiles (256 x 256, 128 x 256 for E4M3 activations) feed more MFMAs per
// byte, small ones (128 x 128) leave fewer CUs idle; E4M3 has 128 x 192 between
// them.  A round of small, middle and large ones takes about 20, 24 and 29 parts of
// time (of the small ones two fit a CU for E2M1), and the shortest sum is taken.
// us, large / small: MXFP4 4096 x 4096 x 4096 47 / 56, 4096 x 8192 x 8192 149 / 190, gated
// 1000 x 4096 x 14336 89 / 94; MXFP8 2000 x 4096 x 4096 37.5 / 44.6, 4096 x 4096 x 4096 72 / 81,
// 700 x 8192 x 8192 51 / 60, gated 1000 x 4096 x 14336 131 / 134, 1000 x 2048 x 5632 40.6 / 38.3
// (the rule's loss).  Middle / small: 1000 x 4096 x 6144 31.4 / 37.2.  With four waves large /
// small MXFP4 1000 x 4096 x 6144 38 / 25, large / middle / small MXFP8 256 x 4096 x 4096 27 /
// 24 / 21, 1000 x 4096 x 6144 33 / 30 / 41.
//
// A small tile has as many stages as LDS has room for, since a step of its own takes
// less time than a load: three for E4M3, and for E2M1 four, where there are no more tiles
// than CUs, else two, so that two workgroups share a CU.  us, two stages | more: MXFP8
// 128 x 4096 x 4096 20.5 | 18.2, 1000 x 14336 x 4096 66.9 | 61.7; MXFP4 128 x 4096 x
// 4096 18.5 | 14.4, 1000 x 14336 x 4096 53.6 | 45.0, but 1000 x 4096 x 6144 25.7 | 30.3,
// 2000 x 4096 x 4096 30.4 | 35.9.
//
// Tiles have eight waves, two a SIMD, of which one multiplies while the other waits or
// stores.  Four read less of LDS, which wins along a long K of E4M3 by large tiles.
// us, four waves | eight, large tiles: MXFP4 4096 x 8192 x 8192 153 | 149, 1000 x 4096 x
// 14336 44.4 | 39.8, gated 4096 x 8192 x 14336 572 | 472; MXFP8 1000 x 4096 x 14336 62 | 58,
// 16384 x 4096 x 4096 278 | 270, 2000 x 8192 x 8192 118 | 117, 4096 x 8192 x 8192 234 | 243,
// 1000 x 14336 x 14336 181 | 193, gated 500 x 4096 x 14336 72.6 | 63.0, 4096 x 8192 x 14336
// 821 | 811.  Small ones: MXFP8 128 x 4096 x 4096 18.2 | 16.5, 1000 x 14336 x 4096 60.7 |
// 60.6; MXFP4 128 x 4096 x 4096 14.4 | 13.1, 2000 x 4096 x 4096 30.7 | 31.1, gated 33 x 5120 x
// 13001 27.6 | 23.7.  (Three blocks of 32 columns, the middle tile's, are not two waves' to
// share.)
enum class Tiles { kSmall, kMiddle, kLarge };
Tiles TilesOf(const MxMatMulParams &p) {
  const int64_t cus = Ctx().num_cus;
  // a gated tile has half the columns, of two weights
  auto rounds = [&](int64_t m, int64_t n, int64_t at_once) {
    return Ceil(Ceil(p.M, m) * Ceil(p.N, p.output ? n / 2 : n), at_once * cus);
  };
  const int64_t small = 20 * rounds(128, 128, p.a_fp4 ? 2 : 1), large = 29 * rounds(p.a_fp4 ? 256 : 128, 256, 1);
  if (!p.a_fp4 && !p.output && 24 * rounds(128, 192, 1) < std::min(small, large)) return Tiles::kMiddle;
  return large <= small ? Tiles::kLarge : Tiles::kSmall;
}

// Few rows take the streaming kernel, whose time goes with the weight's bytes and
// the row tiles; the GEMM's one round of tiles goes with K alone, and a wide
// weight fills it.  us, rows x K x N, stream | GEMM (gated: N of each weight):
//   MXFP4  32 x 4096 x 14336 14.8 | 13.7    20 x 8192 x 28672 45.6 | 38.2
//          36 x 2048 x 8192 8.1 | 9.5       40 x 8192 x 8192 18.1 | 19.7
//          40 x 11008 x 8192 22.1 | 24.0    48 x 4096 x 11008 17.7 | 14.4
//          64 x 2048 x 8192 8.6 | 9.7       64 x 4096 x 6144 12.5 | 12.9
//          64 x 4096 x 8192 12.9 | 13.1     52 x 8192 x 5632 22.0 | 19.6
//          64 x 11008 x 4096 21.0 | 23.4
//   MXFP8  20 x 8192 x 28672 45.5 | 42.1    32 x 4096 x 14336 18.1 | 16.7
//          36 x 2048 x 8192 8.9 | 11.1      48 x 4096 x 6144 15.6 | 15.8
//          48 x 4096 x 8192 18.3 | 16.1     40 x 11008 x 8192 35.2 | 31.8
//          64 x 4096 x 4096 15.8 | 15.7     64 x 4096 x 6144 18.7 | 15.9
//          64 x 11008 x 4096 28.7 | 31.4
//   gated, MXFP4
//          32 x 4096 x 8192 15.2 | 15.4     24 x 4096 x 11008 21.6 | 18.2
//          33 x 2048 x 8192 11.1 | 11.7     33 x 4096 x 8192 18.0 | 15.5
//          48 x 4096 x 5632 18.3 | 15.2     33 x 5120 x 13001 32.1 | 23.7
//          64 x 4096 x 4096 13.6 | 14.7
//   gated, MXFP8
//          32 x 4096 x 8192 19.5 | 18.7     24 x 4096 x 11008 21.7 | 20.8
//          20 x 8192 x 11008 36.0 | 35.7
bool Streams(const MxMatMulParams &p) {
  if (p.M <= 16 || p.M > 64) return p.M <= 16;
  const int64_t rows = WeightRows(p), K = std::max<int64_t>(p.K, 1);
  // MXFP8 output takes four row tiles, which more than 32 rows leave no registers for
  if (p.output == kGatedMx) return p.M <= 32;
  if (p.M <= 32) return rows < 14336;
  // where rows * K of the one takes as long as K and a launch of the other
  if (p.a_fp4) return rows < (p.M > 48 ? 3000 + 19000000 / K : 7000 + 16000000 / K);
  return rows < 3500 + 10000000 / K;
}

// Up to this many values every workgroup quantizes its activations itself
// (eight at a time per thread); a launch for all costs 2 to 4 us.  us, MXFP8, itself |
// in a launch, by N:
//               2048        4096       8192        14336       28672
//   1 x 4096    4.7 | 7.4   5.0 | 7.5   6.3 | 8.1    9.9 | 11.6  16.6 | 18.7
//   2 x 4096    4.8 | 7.3   5.1 | 7.8   7.3 | 8.1   11.7 | 11.9  20.5 | 19.4
//   4 x 4096    6.3 | 7.3   6.3 | 8.0   9.5 | 8.5   15.6 | 12.5  25.8 | 20.3
//   8 x 4096    8.8 | 7.5   8.8 | 8.2  13.3 | 8.9   23.1 | 13.3  37.9 | 21.9
//   8 x 2048    5.6 | 7.5   5.6 | 7.3   7.1 | 7.1   12.6 | 9.7   21.0 | 14.7
//   1 x 8192    6.5 | 8.8   9.4 | 9.4  16.9 | 14.8  20.7 | 25.0  41.0 | 35.4
//   2 x 8192    7.8 | 9.1  11.4 | 9.7  20.5 | 15.2  24.3 | 25.5  45.2 | 36.2
// The rule does not look at N, with which the workgroups that repeat the work grow:
// it holds up to 8192 values and for narrow weights, and loses up to 35 % between
// that and its end by wide ones.
constexpr int64_t kOwnQuant = 16384;
bool OwnQuant(const MxMatMulParams &p) { return p.x && p.M <= 16 && p.M * Ceil(p.K, 512) * 512 <= kOwnQuant; }

// How the streaming kernel covers a problem: row tiles of 16 nt rows of the
// weight, `split` workgroups of `waves` waves for each.
struct StreamPlan {
  int nt, mt, waves, split;
  int64_t tiles;
};

StreamPlan PlanStream(const MxMatMulParams &p) {
  StreamPlan s;
  const int64_t chunks = Ceil(p.K, 512);
  s.mt = (int)Ceil(p.M, 16);
  // Activations from memory are read by every wave for itself, all over the chip
  // the same ones at about the same time, and cost as much per 16 rows as the
  // weight: several row tiles share a read, while a wave for every CU's SIMD is
  // left.  More than these do not fit the registers of two waves per SIMD.  us,
  // K = 4096, N = 14336, with these | with one: 8 rows 13.3 | 15.0, 16 rows 15.0 |
  // 18.3, MXFP4 32 rows 14.7 | 19.1, 48 rows 18.2 | 24.0.
  // A gated product's row tiles come in pairs, for MXFP8 blocks in two.
  const int least = p.output == kGatedMx ? 4 : p.output ? 2 : 1;
  s.nt = OwnQuant(p) ? least : s.mt == 1 ? 2 : s.mt <= (p.a_fp4 ? 3 : 2) ? 4 : 2;
  while (s.nt > 1 && Ceil(WeightRows(p), 16 * s.nt) * chunks < 4 * Ctx().num_cus) s.nt /= 2;
  s.nt = std::max(s.nt, least);
  s.waves = s.nt == 4 ? 4 : 8;
  s.tiles = Ceil(WeightRows(p), 16 * s.nt);
  // as many as give every wave one chunk, while there are not more than about
  // two rounds of them
  s.split = (int)std::max<int64_t>(1, std::min<int64_t>(Ceil(chunks, s.waves), 32 * Ctx().num_cus / (s.waves * s.tiles)));
  return s;
}

template <bool A4, int NT, int MT, bool QUANT, int OUT> void LaunchStream(const mx::StreamArgs &a, const StreamPlan &s, hipStream_t st) {
  const int64_t chunks = Ceil(a.K, 512);
  const size_t codes = QUANT ? (size_t)(a.M * chunks * ((A4 ? 256 : 512) + 16)) : 0;
  const size_t lds = std::max(codes, (size_t)NT * MT * s.waves * 1024);
  LaunchInPieces(s.tiles, 64 * s.waves, [&](int64_t first, unsigned count) {
    mx::StreamArgs p = a;
    p.first = (int)first;
    mx::StreamKernel<A4, NT, MT, QUANT, OUT><<<dim3(count, (unsigned)s.split), 64 * s.waves, lds, st>>>(p);
  });
}

template <bool A4, int MT, int OUT> void LaunchStreamRows(const mx::StreamArgs &a, const StreamPlan &s, hipStream_t st) {
  constexpr bool kFour = MT == 2 || (A4 && MT == 3);
  if constexpr (OUT == kGatedMx) {
    if constexpr (MT <= 2) LaunchStream<A4, 4, MT, false, OUT>(a, s, st);
  } else if (kFour && s.nt == 4) {
    LaunchStream<A4, kFour ? 4 : 2, MT, false, OUT>(a, s, st);
  } else if (OUT == kGated || s.nt == 2) {
    LaunchStream<A4, 2, MT, false, OUT>(a, s, st);
  } else {
    LaunchStream<A4, OUT == kPlain ? 1 : 2, MT, false, OUT>(a, s, st);
  }
}

template <bool A4, int OUT> void LaunchStreamOf(const mx::StreamArgs &a, bool own, const StreamPlan &s, hipStream_t st) {
  if (own)
    LaunchStream<A4, OUT == kPlain ? 1 : OUT == kGated ? 2 : 4, 1, true, OUT>(a, s, st);
  else if (s.mt == 1)
    LaunchStreamRows<A4, 1, OUT>(a, s, st);
  else if (s.mt == 2)
    LaunchStreamRows<A4, 2, OUT>(a, s, st);
  else if (s.mt == 3)
    LaunchStreamRows<A4, 3, OUT>(a, s, st);
  else
    LaunchStreamRows<A4, 4, OUT>(a, s, st);
}

template <int OUT> void LaunchStreams(const mx::StreamArgs &a, bool a_fp4, bool own, const StreamPlan &s, hipStream_t st) {
  a_fp4 ? LaunchStreamOf<true, OUT>(a, own, s, st) : LaunchStreamOf<false, OUT>(a, own, s, st);
}

}  // namespace

size_t MxMatMulScratchBytes(const MxMatMulParams &p) {
  if (Streams(p)) {
    const size_t codes = p.x && !OwnQuant(p) ? Scratch::Round((size_t)(p.M * p.K)) + Scratch::Round((size_t)(p.M * p.K / 32)) : 0;
    const StreamPlan s = PlanStream(p);
    return codes + (s.split > 1 ? (size_t)s.tiles * s.split * s.nt * s.mt * 1024 : 0);
  }
  const MxScratch s(p);
  return s.codes + s.a_tiles + (p.output ? 2 : 1) * s.b_tiles;
}

void LaunchMxMatMul(const MxMatMulParams &p, void *scratch, hipStream_t stream) {
  if (Streams(p)) {
    const StreamPlan plan = PlanStream(p);
    mx::StreamArgs a{p.x, p.a, p.a_scale, p.b, p.b_scale, static_cast<uint16_t *>(p.y), (int)p.M, (int)p.N, (int)p.K,
                     p.x_dtype == kBfloat16, p.y_bf16, plan.split, nullptr, nullptr, 0, p.up, p.up_scale, p.activation,
                     p.y_scale};
    const bool own = OwnQuant(p);
    uint8_t *codes = static_cast<uint8_t *>(scratch), *scales = codes + Scratch::Round((size_t)(p.M * p.K));
    if (a.split > 1) {
      a.part = reinterpret_cast<float *>(p.x && !own ? scales + Scratch::Round((size_t)(p.M * p.K / 32)) : codes);
      a.done = Ctx().ws.Counters((size_t)plan.tiles);
    }
    if (p.x && !own) {
      LaunchMxQuantize(MxQuantParams{p.x, codes, scales, p.M, p.K, p.x_dtype, p.a_fp4, 0}, stream);
      a.a = codes;
      a.as = scales;
    }
    if (p.output == kGatedMx)
      LaunchStreams<kGatedMx>(a, p.a_fp4, own, plan, stream);
    else if (p.output)
      LaunchStreams<kGated>(a, p.a_fp4, own, plan, stream);
    else
      LaunchStreams<kPlain>(a, p.a_fp4, own, plan, stream);
    return;
  }
  const MxScratch s(p);
  uint8_t *codes = static_cast<uint8_t *>(scratch), *a_tiles = codes + s.codes, *b_tiles = a_tiles + s.a_tiles;
  uint8_t *up_tiles = b_tiles + s.b_tiles;
  const int64_t steps = Ceil(p.K, 256);
  MxOperands o{};
  o.a_scale = p.a_scale;
  o.b_scale = p.b_scale;
  o.a_tiles = a_tiles;
  o.b_tiles = b_tiles;
  o.up_scale = p.up_scale;
  o.up_tiles = up_tiles;
  o.M = p.M;
  o.N = p.N;
  o.K = p.K;
  o.b_groups = Ceil(WeightRows(p) * steps, 256);
  o.q = MxQuantParams{p.x, codes, nullptr, p.M, p.K, p.x_dtype, p.a_fp4, 0};
  o.a = p.a;
  o.codes = s.codes ? codes : nullptr;
  // a thread per 8 values to quantize, or 16 bytes of codes to copy, or a step's scales
  const int64_t a_threads = p.M * steps * (p.x ? 32 : !s.codes ? 1 : p.a_fp4 ? 8 : 16);
  // K = 0: no operands, no launch, sums of nothing
  LaunchInPieces(o.b_groups + Ceil(a_threads, 256), 256, [&](int64_t first, unsigned count) {
    o.first = first;
    if (p.x_dtype == kFloat16)
      MxOperandsKernel<kFloat16><<<count, 256, 0, stream>>>(o);
    else
      MxOperandsKernel<kBfloat16><<<count, 256, 0, stream>>>(o);
  });
  const mx::GemmArgs g{s.codes ? codes : p.a, p.b, a_tiles, b_tiles, static_cast<uint16_t *>(p.y), p.M, p.N, p.K, p.y_bf16,
                       (p.output == kGatedMx || p.N % 8 == 0) && reinterpret_cast<uintptr_t>(p.y) % 16 == 0, p.up, up_tiles,
                       p.activation, p.y_scale};
  const Tiles tiles = TilesOf(p);
  if (tiles == Tiles::kLarge && p.a_fp4)
    LaunchGemm<true, 4, 2, 2, 2, 4>(g, p.output, stream);
  else if (tiles == Tiles::kLarge && (p.output || p.K < 8192))
    LaunchGemm<false, 2, 2, 2, 2, 4>(g, p.output, stream);
  else if (tiles == Tiles::kLarge)
    LaunchGemm<false, 2, 4, 2, 2, 2>(g, kPlain, stream);
  else if (tiles == Tiles::kMiddle)
    LaunchGemm<false, 2, 3, 2, 2, 2>(g, kPlain, stream);
  else if (!p.a_fp4)
    LaunchGemm<false, 1, 2, 3, 4, 2>(g, p.output, stream);
  else if (Ceil(p.M, 128) * Ceil(p.N, p.output ? 64 : 128) <= Ctx().num_cus)
    LaunchGemm<true, 1, 2, 4, 4, 2>(g, p.output, stream);
  else
    LaunchGemm<true, 1, 2, 2, 4, 2>(g, p.output, stream);
}

}  // namespace onnxl_amd
