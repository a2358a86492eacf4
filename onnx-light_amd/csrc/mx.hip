// Microscaled 4-bit products: quantization of 16-bit activations to MXFP8 or
// MXFP4 and the product with MXFP4 weights on the block-scaled matrix cores.
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
  uint8_t *codes;             // a's codes with padded rows, where K is not whole steps
  uint8_t *a_tiles, *b_tiles;
  int64_t M, N, K;
  int64_t b_groups;           // workgroups of b's part
  int64_t first;              // the launch's first workgroup
};

template <int DT> __global__ __launch_bounds__(256) void MxOperandsKernel(const MxOperands p) {
  const int64_t steps = (p.K + 255) / 256, group = p.first + blockIdx.x;
  if (group < p.b_groups) {
    const int64_t i = group * 256 + threadIdx.x;
    if (i < p.N * steps) TileScales(p.b_scale, p.b_tiles, p.N, p.K, i);
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

// Scratch: codes (where they are not a's own) and scale tiles of a, scale tiles
// of b.
struct MxScratch {
  size_t codes, a_tiles, b_tiles;
  explicit MxScratch(const MxMatMulParams &p)
      : codes(p.x || p.K % 256 ? Scratch::Round((size_t)(p.M * Ceil(p.K, 256) * (p.a_fp4 ? 128 : 256))) : 0),
        a_tiles(Scratch::Round((size_t)mx::ScaleTileBytes(p.M, p.K))),
        b_tiles(Scratch::Round((size_t)mx::ScaleTileBytes(p.N, p.K))) {}
};

template <bool A4, int MB, int NB> void LaunchGemm(const mx::GemmArgs &g, hipStream_t s) {
  using S = mx::Shape<A4, MB, NB>;
  mx::GemmKernel<A4, MB, NB><<<dim3((unsigned)(Ceil(g.M, S::BM) * Ceil(g.N, S::BN))), 256, 0, s>>>(g);
}

// Large tiles (256 x 256, 128 x 256 for E4M3 activations) feed more MFMAs per
// byte, small ones (128 x 128) leave fewer CUs idle; E4M3 has 128 x 192 between
// them.  A round of small, middle and large ones takes about 20, 24 and 29 parts of
// time (of the small ones two fit a CU for E2M1), and the shortest sum is taken.
// us, large / small: MXFP4 1000 x 4096 x 6144 38 / 25, 4096 x 8192 x 8192 156 /
// 184.  Large / middle / small: MXFP8 256 x 4096 x 4096 27 / 24 / 21, 1000 x 4096 x
// 6144 33 / 30 / 41, 2048 x 4096 x 4096 39 / 51 / 45, 4096 x 8192 x 8192 234 / 278 /
// 311.
enum class Tiles { kSmall, kMiddle, kLarge };
Tiles TilesOf(const MxMatMulParams &p) {
  const int64_t cus = Ctx().num_cus;
  auto rounds = [&](int64_t m, int64_t n, int64_t at_once) { return Ceil(Ceil(p.M, m) * Ceil(p.N, n), at_once * cus); };
  const int64_t small = 20 * rounds(128, 128, p.a_fp4 ? 2 : 1), large = 29 * rounds(p.a_fp4 ? 256 : 128, 256, 1);
  if (!p.a_fp4 && 24 * rounds(128, 192, 1) < std::min(small, large)) return Tiles::kMiddle;
  return large <= small ? Tiles::kLarge : Tiles::kSmall;
}

// Few rows take the streaming kernel, whose time goes with the weight's bytes and
// the row tiles; the GEMM's one round of tiles goes with K alone, and a wide
// weight fills it.  us, rows x K x N, stream | GEMM:
//   MXFP4  32 x 4096 x 14336 14.7 | 18.6    48 x 4096 x 14336 18.1 | 18.5
//          56 x 4096 x 14336 20.8 | 18.6    64 x 2048 x 16384 14.9 | 13.1
//          64 x 8192 x 8192 27.1 | 28.2     64 x 11008 x 4096 20.9 | 33.9
//   MXFP8  36 x 2048 x 8192 8.6 | 13.1      40 x 11008 x 8192 35.2 | 39.4
//          40 x 4096 x 14336 27.3 | 20.7    33 x 8192 x 28672 81.4 | 51.5
//          64 x 4096 x 6144 18.5 | 19.5     64 x 4096 x 8192 21.9 | 19.8
bool Streams(const MxMatMulParams &p) {
  if (p.M <= 32 || p.M > 64) return p.M <= 32;
  if (p.a_fp4) return p.M <= 48 || p.N < 12288;
  return p.N < (p.M <= 48 ? 11264 : 7168);
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
  s.nt = OwnQuant(p) ? 1 : s.mt == 1 ? 2 : s.mt <= (p.a_fp4 ? 3 : 2) ? 4 : 2;
  while (s.nt > 1 && Ceil(p.N, 16 * s.nt) * chunks < 4 * Ctx().num_cus) s.nt /= 2;
  s.waves = s.nt == 4 ? 4 : 8;
  s.tiles = Ceil(p.N, 16 * s.nt);
  // as many as give every wave one chunk, while there are not more than about
  // two rounds of them
  s.split = (int)std::max<int64_t>(1, std::min<int64_t>(Ceil(chunks, s.waves), 32 * Ctx().num_cus / (s.waves * s.tiles)));
  return s;
}

template <bool A4, int NT, int MT, bool QUANT> void LaunchStream(const mx::StreamArgs &a, const StreamPlan &s, hipStream_t st) {
  const int64_t chunks = Ceil(a.K, 512);
  const size_t codes = QUANT ? (size_t)(a.M * chunks * ((A4 ? 256 : 512) + 16)) : 0;
  const size_t lds = std::max(codes, (size_t)NT * MT * s.waves * 1024);
  LaunchInPieces(s.tiles, 64 * s.waves, [&](int64_t first, unsigned count) {
    mx::StreamArgs p = a;
    p.first = (int)first;
    mx::StreamKernel<A4, NT, MT, QUANT><<<dim3(count, (unsigned)s.split), 64 * s.waves, lds, st>>>(p);
  });
}

template <bool A4, int MT> void LaunchStreamRows(const mx::StreamArgs &a, const StreamPlan &s, hipStream_t st) {
  constexpr bool kFour = MT == 2 || (A4 && MT == 3);
  if (kFour && s.nt == 4)
    LaunchStream<A4, kFour ? 4 : 2, MT, false>(a, s, st);
  else if (s.nt == 2)
    LaunchStream<A4, 2, MT, false>(a, s, st);
  else
    LaunchStream<A4, 1, MT, false>(a, s, st);
}

template <bool A4> void LaunchStreamOf(const mx::StreamArgs &a, bool own, const StreamPlan &s, hipStream_t st) {
  if (own)
    LaunchStream<A4, 1, 1, true>(a, s, st);
  else if (s.mt == 1)
    LaunchStreamRows<A4, 1>(a, s, st);
  else if (s.mt == 2)
    LaunchStreamRows<A4, 2>(a, s, st);
  else if (s.mt == 3)
    LaunchStreamRows<A4, 3>(a, s, st);
  else
    LaunchStreamRows<A4, 4>(a, s, st);
}

}  // namespace

size_t MxMatMulScratchBytes(const MxMatMulParams &p) {
  if (Streams(p)) {
    const size_t codes = p.x && !OwnQuant(p) ? Scratch::Round((size_t)(p.M * p.K)) + Scratch::Round((size_t)(p.M * p.K / 32)) : 0;
    const StreamPlan s = PlanStream(p);
    return codes + (s.split > 1 ? (size_t)s.tiles * s.split * s.nt * s.mt * 1024 : 0);
  }
  const MxScratch s(p);
  return s.codes + s.a_tiles + s.b_tiles;
}

void LaunchMxMatMul(const MxMatMulParams &p, void *scratch, hipStream_t stream) {
  if (Streams(p)) {
    const StreamPlan plan = PlanStream(p);
    mx::StreamArgs a{p.x, p.a, p.a_scale, p.b, p.b_scale, static_cast<uint16_t *>(p.y), (int)p.M, (int)p.N, (int)p.K,
                     p.x_dtype == kBfloat16, p.y_bf16, plan.split, nullptr, nullptr, 0};
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
    p.a_fp4 ? LaunchStreamOf<true>(a, own, plan, stream) : LaunchStreamOf<false>(a, own, plan, stream);
    return;
  }
  const MxScratch s(p);
  uint8_t *codes = static_cast<uint8_t *>(scratch), *a_tiles = codes + s.codes, *b_tiles = a_tiles + s.a_tiles;
  const int64_t steps = Ceil(p.K, 256);
  MxOperands o{};
  o.a_scale = p.a_scale;
  o.b_scale = p.b_scale;
  o.a_tiles = a_tiles;
  o.b_tiles = b_tiles;
  o.M = p.M;
  o.N = p.N;
  o.K = p.K;
  o.b_groups = Ceil(p.N * steps, 256);
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
                       p.N % 8 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0};
  const Tiles tiles = TilesOf(p);
  if (tiles == Tiles::kLarge)
    p.a_fp4 ? LaunchGemm<true, 4, 4>(g, stream) : LaunchGemm<false, 2, 4>(g, stream);
  else if (tiles == Tiles::kMiddle)
    LaunchGemm<false, 2, 3>(g, stream);
  else
    p.a_fp4 ? LaunchGemm<true, 2, 2>(g, stream) : LaunchGemm<false, 2, 2>(g, stream);
}

}  // namespace onnxl_amd
