// Microscaled 4-bit products: quantization of 16-bit activations to MXFP8 or
// MXFP4 and the product with MXFP4 weights on the block-scaled matrix cores.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "quant8.hpp"

namespace onnxl_amd {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

template <int DT> __device__ __forceinline__ float LoadX(const void *p, int64_t i) {
  if constexpr (DT == kFloat) return static_cast<const float *>(p)[i];
  if constexpr (DT == kFloat16) return F16ToF32(static_cast<const uint16_t *>(p)[i]);
  return Bf16ToF32(static_cast<const uint16_t *>(p)[i]);
}

// One block of 32 values per thread.
template <int DT> __global__ __launch_bounds__(256) void MxQuantizeKernel(const MxQuantParams p) {
  const int64_t blk = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (blk >= p.rows * (p.K / 32)) return;
  float v[32], top = 0.f;
  bool finite = true;
  for (int i = 0; i < 32; ++i) {
    v[i] = LoadX<DT>(p.x, blk * 32 + i);
    finite = finite && fabsf(v[i]) < __builtin_huge_valf();
    top = fmaxf(top, fabsf(v[i]));
  }
  const BlockScale s = MxScaleOf(finite ? top : __builtin_huge_valf(), p.fp4 ? 2 : 8);
  p.scale[blk] = s.e8m0;
  if (s.e8m0 == 255)
    for (int i = 0; i < 32; ++i) v[i] = 0.f;
  for (int i = 0; i < 32; i += 2) {
    if (p.fp4) {
      p.y[(blk * 32 + i) / 2] = (uint8_t)Fp4Codes2(v[i] * s.inv, v[i + 1] * s.inv);
    } else {
      p.y[blk * 32 + i] = Fp8Code(v[i] * s.inv);
      p.y[blk * 32 + i + 1] = Fp8Code(v[i + 1] * s.inv);
    }
  }
}

// One wave per 16 x 16 outputs, operands straight from memory.  Lane l holds
// row l % 16 of an operand: for E2M1 the 32 values from 32 (l / 16), for E4M3
// the 16 from 16 (l / 16) and the 16 from 64 + 16 (l / 16), and the scale of
// block l / 16 in both.
template <bool A4> __global__ __launch_bounds__(64) void MxMatMulKernel(const MxMatMulParams p) {
  const int lane = threadIdx.x, r = lane % 16, g = lane / 16;
  const int64_t m = (int64_t)blockIdx.y * 16 + r, n = (int64_t)blockIdx.x * 16 + r;
  const int64_t am = m < p.M ? m : p.M - 1, bn = n < p.N ? n : p.N - 1;
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  auto load = [&](const uint8_t *row, int64_t at, int64_t bytes, v8i &dst, int first) {
    for (int i = 0; i < 4; ++i)
      dst[first + i] = at + 4 * i + 4 <= bytes ? *reinterpret_cast<const int *>(row + at + 4 * i) : 0;
  };
  for (int64_t k = 0; k < p.K; k += 128) {
    v8i a = {0, 0, 0, 0, 0, 0, 0, 0}, b = {0, 0, 0, 0, 0, 0, 0, 0};
    load(p.b + bn * (p.K / 2), k / 2 + 16 * g, p.K / 2, b, 0);
    if constexpr (A4) {
      load(p.a + am * (p.K / 2), k / 2 + 16 * g, p.K / 2, a, 0);
    } else {
      load(p.a + am * p.K, k + 16 * g, p.K, a, 0);
      load(p.a + am * p.K, k + 64 + 16 * g, p.K, a, 4);
    }
    const int64_t blk = k / 32 + g, blocks = p.K / 32;
    const int sa = blk < blocks ? p.a_scale[am * blocks + blk] : 127;
    const int sb = blk < blocks ? p.b_scale[bn * blocks + blk] : 127;
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, A4 ? 4 : 0, 4, 0, sa, 0, sb);
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t mo = (int64_t)blockIdx.y * 16 + 4 * g + i;
    if (mo < p.M && n < p.N)
      static_cast<uint16_t *>(p.y)[mo * p.N + n] = p.y_bf16 ? F32ToBf16(acc[i]) : F32ToF16(acc[i]);
  }
}

}  // namespace

void LaunchMxQuantize(const MxQuantParams &p, hipStream_t stream) {
  const int64_t blocks = p.rows * (p.K / 32);
  if (blocks == 0) return;
  const dim3 grid((unsigned)((blocks + 255) / 256));
  if (p.x_dtype == kFloat)
    MxQuantizeKernel<kFloat><<<grid, 256, 0, stream>>>(p);
  else if (p.x_dtype == kFloat16)
    MxQuantizeKernel<kFloat16><<<grid, 256, 0, stream>>>(p);
  else
    MxQuantizeKernel<kBfloat16><<<grid, 256, 0, stream>>>(p);
}

void LaunchMxMatMul(const MxMatMulParams &p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.N + 15) / 16), (unsigned)((p.M + 15) / 16));
  if (p.a_fp4)
    MxMatMulKernel<true><<<grid, 64, 0, stream>>>(p);
  else
    MxMatMulKernel<false><<<grid, 64, 0, stream>>>(p);
}

}  // namespace onnxl_amd
