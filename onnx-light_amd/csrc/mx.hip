// Microscaled 4-bit products: quantization of 16-bit activations to MXFP8 or
// MXFP4 and the product, plain or gated, with MXFP4 weights on the block-scaled
// matrix cores.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "mx_gemm.hpp"
#include "mx_plan.hpp"
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

using mx::Ceil;

mx::Sizes SizesOf(const MxMatMulParams &p) {
  return {p.M, p.N, p.K, p.x != nullptr, p.a_fp4 != 0, p.output, Ctx().num_cus};
}

// Scratch: codes (where they are not a's own) and scale tiles of a, scale tiles
// of b and of the second weight.
struct MxScratch {
  size_t codes, a_tiles, b_tiles;
  explicit MxScratch(const MxMatMulParams &p)
      : codes(p.x || p.K % 256 ? Scratch::Round((size_t)(p.M * Ceil(p.K, 256) * (p.a_fp4 ? 128 : 256))) : 0),
        a_tiles(Scratch::Round((size_t)mx::ScaleTileBytes(p.M, p.K))),
        b_tiles(Scratch::Round((size_t)mx::ScaleTileBytes(p.N, p.K))) {}
};

// Launches this kernel if it is the plan's.
template <bool A4, int MB, int NB, int STAGES, int WM, int WN> bool LaunchGemm(const mx::GemmArgs &g, const mx::GemmPlan &t, int output, hipStream_t s) {
  if (t.mb != MB || t.nb != NB || t.stages != STAGES || t.wm != WM || t.wn != WN) return false;
  using S = mx::Shape<A4, MB, NB, STAGES, WM, WN>;
  constexpr int kThreads = 64 * WM * WN;
  LaunchInPieces(Ceil(g.M, S::BM) * Ceil(g.N, output ? S::BN / 2 : S::BN), kThreads, [&](int64_t first, unsigned count) {
    mx::GemmArgs p = g;
    p.first = (int)first;
    if constexpr (WM * WN == 8) {
      if (output == kGatedMx)
        mx::GemmKernel<A4, MB, NB, STAGES, WM, WN, kGatedMx><<<count, kThreads, 0, s>>>(p);
      else if (output == kGated)
        mx::GemmKernel<A4, MB, NB, STAGES, WM, WN, kGated><<<count, kThreads, 0, s>>>(p);
    }
    if (output == kPlain) mx::GemmKernel<A4, MB, NB, STAGES, WM, WN><<<count, kThreads, 0, s>>>(p);
  });
  return true;
}

template <bool A4, int NT, int MT, bool QUANT, int OUT> void LaunchStream(const mx::StreamArgs &a, const mx::StreamPlan &s, hipStream_t st) {
  const int64_t chunks = Ceil(a.K, 512);
  const size_t codes = QUANT ? (size_t)(a.M * chunks * ((A4 ? 256 : 512) + 16)) : 0;
  const size_t lds = std::max(codes, (size_t)NT * MT * s.waves * 1024);
  LaunchInPieces(s.tiles, 64 * s.waves, [&](int64_t first, unsigned count) {
    mx::StreamArgs p = a;
    p.first = (int)first;
    mx::StreamKernel<A4, NT, MT, QUANT, OUT><<<dim3(count, (unsigned)s.split), 64 * s.waves, lds, st>>>(p);
  });
}

template <bool A4, int MT, int OUT> void LaunchStreamRows(const mx::StreamArgs &a, const mx::StreamPlan &s, hipStream_t st) {
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

template <bool A4, int OUT> void LaunchStreamOf(const mx::StreamArgs &a, bool own, const mx::StreamPlan &s, hipStream_t st) {
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

template <int OUT> void LaunchStreams(const mx::StreamArgs &a, bool a_fp4, bool own, const mx::StreamPlan &s, hipStream_t st) {
  a_fp4 ? LaunchStreamOf<true, OUT>(a, own, s, st) : LaunchStreamOf<false, OUT>(a, own, s, st);
}

}  // namespace

size_t MxMatMulScratchBytes(const MxMatMulParams &p) {
  const mx::Sizes sizes = SizesOf(p);
  if (mx::Streams(sizes)) {
    const size_t codes = p.x && !mx::OwnQuant(sizes) ? Scratch::Round((size_t)(p.M * p.K)) + Scratch::Round((size_t)(p.M * p.K / 32)) : 0;
    const mx::StreamPlan s = mx::PlanStream(sizes);
    return codes + (s.split > 1 ? (size_t)s.tiles * s.split * s.nt * s.mt * 1024 : 0);
  }
  const MxScratch s(p);
  return s.codes + s.a_tiles + (p.output ? 2 : 1) * s.b_tiles;
}

void LaunchMxMatMul(const MxMatMulParams &p, void *scratch, hipStream_t stream) {
  const mx::Sizes sizes = SizesOf(p);
  if (mx::Streams(sizes)) {
    const mx::StreamPlan plan = mx::PlanStream(sizes);
    mx::StreamArgs a{p.x, p.a, p.a_scale, p.b, p.b_scale, static_cast<uint16_t *>(p.y), (int)p.M, (int)p.N, (int)p.K,
                     p.x_dtype == kBfloat16, p.y_bf16, plan.split, nullptr, nullptr, 0, p.up, p.up_scale, p.activation,
                     p.y_scale};
    const bool own = mx::OwnQuant(sizes);
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
  o.b_groups = Ceil(mx::WeightRows(sizes) * steps, 256);
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
  const mx::GemmPlan t = mx::PlanGemm(sizes);
  const bool launched = p.a_fp4 ? LaunchGemm<true, 4, 2, 2, 2, 4>(g, t, p.output, stream) || LaunchGemm<true, 1, 2, 4, 4, 2>(g, t, p.output, stream) ||
                                      LaunchGemm<true, 1, 2, 2, 4, 2>(g, t, p.output, stream)
                                : LaunchGemm<false, 2, 2, 2, 2, 4>(g, t, p.output, stream) || LaunchGemm<false, 2, 4, 2, 2, 2>(g, t, p.output, stream) ||
                                      LaunchGemm<false, 2, 3, 2, 2, 2>(g, t, p.output, stream) || LaunchGemm<false, 1, 2, 3, 4, 2>(g, t, p.output, stream);
  if (!launched) throw DeviceError("internal: MX tiles without a kernel");
}

}  // namespace onnxl_amd
