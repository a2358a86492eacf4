// RMS norm with the residual's addition and 8-bit output with scales: what a
// decoder layer runs in front of its quantized products.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "quant8.hpp"

namespace onnxl_amd {
namespace {

constexpr int kThreads = 256;

template <int DT> __device__ __forceinline__ float LoadX(const void *p, int64_t i) {
  if constexpr (DT == kFloat) return static_cast<const float *>(p)[i];
  if constexpr (DT == kFloat16) return F16ToF32(static_cast<const uint16_t *>(p)[i]);
  return Bf16ToF32(static_cast<const uint16_t *>(p)[i]);
}

__device__ __forceinline__ float BlockReduce(float v, float *s, bool max) {
  for (int o = 32; o > 0; o >>= 1) {
    const float w = __shfl_xor(v, o);
    v = max ? fmaxf(v, w) : v + w;
  }
  __syncthreads();
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  return max ? fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])) : (s[0] + s[1]) + (s[2] + s[3]);
}

// One workgroup per row, three passes over it: the sum of squares, then for
// each block its largest magnitude and its codes.
template <int DT> __global__ __launch_bounds__(kThreads) void RmsNormKernel(const RmsNormParams p) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x, at = row * p.D;
  const int tid = threadIdx.x;
  auto h_of = [&](int64_t i) -> float {
    const float x = LoadX<DT>(p.x, at + i);
    if (!p.residual) return x;
    const float h = x + LoadX<DT>(p.residual, at + i);
    if constexpr (DT == kFloat) return h;
    if constexpr (DT == kFloat16) return F16ToF32(F32ToF16(h));
    return Bf16ToF32(F32ToBf16(h));
  };
  float ss = 0.f;
  for (int64_t i = tid; i < p.D; i += kThreads) {
    const float h = h_of(i);
    ss += h * h;
  }
  const float rstd = 1.f / sqrtf(BlockReduce(ss, red, false) / (float)p.D + p.eps);
  auto y_of = [&](int64_t i) {
    const float w = p.weight_f32 ? static_cast<const float *>(p.weight)[i] : LoadX<DT>(p.weight, i);
    return h_of(i) * rstd * w;
  };
  for (int64_t b = 0; b < p.D; b += p.block) {
    float top = 0.f;
    bool finite = true;
    for (int64_t i = b + tid; i < b + p.block; i += kThreads) {
      const float y = fabsf(y_of(i));
      finite = finite && y < __builtin_huge_valf();
      top = fmaxf(top, y);
    }
    top = BlockReduce(finite ? top : __builtin_huge_valf(), red, true);
    const BlockScale s = p.scale_kind == kRnsE8M0 ? MxScaleOf(top, 8) : ScaleOf(top, p.y_fp8 ? 448.f : 127.f);
    if (tid == 0) {
      const int64_t si = row * (p.D / p.block) + b / p.block;
      if (p.scale_kind == kRnsE8M0)
        static_cast<uint8_t *>(p.scale)[si] = s.e8m0;
      else
        static_cast<float *>(p.scale)[si] = s.scale;
    }
    for (int64_t i = b + tid; i < b + p.block; i += kThreads)
      static_cast<uint8_t *>(p.y)[at + i] = p.y_fp8 ? Fp8Code(y_of(i) * s.inv) : Int8Code(y_of(i) * s.inv);
  }
  if (p.sum) {
    // last: it may be x's or the residual's own memory
    __syncthreads();
    for (int64_t i = tid; i < p.D; i += kThreads) {
      const float h = h_of(i);
      if constexpr (DT == kFloat) static_cast<float *>(p.sum)[at + i] = h;
      if constexpr (DT == kFloat16) static_cast<uint16_t *>(p.sum)[at + i] = F32ToF16(h);
      if constexpr (DT == kBfloat16) static_cast<uint16_t *>(p.sum)[at + i] = F32ToBf16(h);
    }
  }
}

}  // namespace

void LaunchRmsNormQuantize(const RmsNormParams &p, hipStream_t stream) {
  if (p.rows == 0) return;
  const dim3 grid((unsigned)p.rows);
  if (p.x_dtype == kFloat)
    RmsNormKernel<kFloat><<<grid, kThreads, 0, stream>>>(p);
  else if (p.x_dtype == kFloat16)
    RmsNormKernel<kFloat16><<<grid, kThreads, 0, stream>>>(p);
  else
    RmsNormKernel<kBfloat16><<<grid, kThreads, 0, stream>>>(p);
}

}  // namespace onnxl_amd
