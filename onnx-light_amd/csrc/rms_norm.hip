// RMS norm with the residual's addition and 8-bit output with scales: what a
// decoder layer runs in front of its quantized products.
//
// Bound by memory: x and the residual are read once, the sum and the codes
// written once.  A workgroup has a row and keeps it in registers between the
// sum of squares and the quantization; rows that do not fit are read again (from
// the caches) in pieces.  Every thread has groups of 8 consecutive values, so a
// scale block of 32, 64, 128 or 256 values is 4 .. 32 neighbouring threads of a
// wave and its maximum a few lane exchanges; a scale for the whole row is one
// more join in LDS.  The largest magnitude is found on the bit patterns, where a
// NaN is above every number.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "quant8.hpp"

namespace onnxl_amd {
namespace {

// 16 (8) bytes at any address.  x and the residual are read once and the sum is
// written for a later layer part: non-temporal, they displace nothing (8192 x
// 8192 with blocks of 128 141 -> 81 us, 5.8 TB/s; 88 with ordinary stores of the
// sum).  The codes are read by the next kernel and stay (non-temporal they cost
// the product behind a 1000-token norm 3 us).
typedef unsigned v4u __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned v2u __attribute__((ext_vector_type(2), aligned(1)));

// Eight values from i on as fp32; those from `end` on are 0.  Whole groups are
// one or two 16-byte loads from any address.
template <int DT, bool NT> __device__ __forceinline__ void Load8(const void *p, int64_t i, int64_t end, float (&v)[8]) {
  if constexpr (DT == kFloat) {
    const float *x = static_cast<const float *>(p);
    if (i + 8 <= end) {
      __builtin_memcpy(v, x + i, 32);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + j < end ? x[i + j] : 0.f;
    }
  } else {
    const uint16_t *x = static_cast<const uint16_t *>(p);
    uint16_t u[8] = {};
    if (i + 8 <= end) {
      const v4u raw = NT ? __builtin_nontemporal_load(reinterpret_cast<const v4u *>(x + i)) : *reinterpret_cast<const v4u *>(x + i);
      __builtin_memcpy(u, &raw, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < end) u[j] = x[i + j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = DT == kFloat16 ? F16ToF32(u[j]) : Bf16ToF32(u[j]);
  }
}

// v rounded to DT, written to p (where given) and left in v.
template <int DT> __device__ __forceinline__ void Round8(void *p, int64_t i, int64_t end, float (&v)[8]) {
  if constexpr (DT == kFloat) {
    if (!p) return;
    float *y = static_cast<float *>(p);
    if (i + 8 <= end) {
      __builtin_memcpy(y + i, v, 32);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < end) y[i + j] = v[j];
    }
  } else {
    uint16_t u[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      unsigned w;
      if constexpr (DT == kBfloat16) {
        asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(w) : "v"(v[j]), "v"(v[j + 1]));
      } else {
        w = __builtin_bit_cast(uint16_t, (_Float16)v[j]) | (unsigned)__builtin_bit_cast(uint16_t, (_Float16)v[j + 1]) << 16;
      }
      u[j] = (uint16_t)w;
      u[j + 1] = (uint16_t)(w >> 16);
      v[j] = DT == kFloat16 ? F16ToF32(u[j]) : __builtin_bit_cast(float, w << 16);
      v[j + 1] = DT == kFloat16 ? F16ToF32(u[j + 1]) : __builtin_bit_cast(float, w & 0xffff0000u);
    }
    if (!p) return;
    uint16_t *y = static_cast<uint16_t *>(p);
    if (i + 8 <= end) {
      v4u raw;
      __builtin_memcpy(&raw, u, 16);
      __builtin_nontemporal_store(raw, reinterpret_cast<v4u *>(y + i));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < end) y[i + j] = u[j];
    }
  }
}

__device__ __forceinline__ unsigned TopBits(const float (&v)[8]) {
  unsigned t = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) t = max(t, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
  return t;
}

// Codes of y = v * s.inv; those of a scale that is NaN are zero.
__device__ __forceinline__ void Store8(uint8_t *y, int64_t i, int64_t end, const float (&v)[8], const BlockScale &s,
                                       const RmsNormParams &p) {
  uint2 w;
  if (p.scale_kind == kRnsE8M0) {
    w = MxFp8Codes8(v, s);
  } else {
    float c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = v[j] * s.inv;
    w = p.y_fp8 ? make_uint2(Fp8Codes4(c[0], c[1], c[2], c[3]), Fp8Codes4(c[4], c[5], c[6], c[7]))
                : make_uint2(Int8Codes4(c[0], c[1], c[2], c[3]), Int8Codes4(c[4], c[5], c[6], c[7]));
    if (s.scale != s.scale) w = make_uint2(0, 0);
  }
  if (i + 8 <= end) {
    *reinterpret_cast<v2u *>(y + i) = v2u{w.x, w.y};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < end) y[i + j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j % 4)));
  }
}

// Sum (max) over the workgroup; s holds one value per wave.
template <int WAVES, bool MAX, typename T> __device__ __forceinline__ T Join(T v, T *s) {
  for (int o = 32; o > 0; o >>= 1) {
    const T w = __shfl_xor(v, o);
    v = MAX ? (v > w ? v : w) : v + w;
  }
  if constexpr (WAVES == 1) return v;
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v = MAX ? (v > s[w] ? v : s[w]) : v + s[w];
  return v;
}

// NG groups of 8 values per thread are kept; KEPT: they are the whole row.
template <int DT, int THREADS, int NG, bool KEPT>
__global__ __launch_bounds__(THREADS) void RmsNormKernel(const RmsNormParams p) {
  constexpr int WAVES = THREADS / 64, kStep = THREADS * 8;
  __shared__ float s_sum[WAVES];
  __shared__ unsigned s_top[WAVES];
  const int64_t row = p.first + blockIdx.x, at = row * p.D, end = at + p.D;
  const int tid = threadIdx.x;
  float v[NG][8];
  // h of the group from i on (past the end: zeros)
  auto load = [&](int64_t i, float (&h)[8], bool first) __attribute__((always_inline)) {
    Load8<DT, KEPT>(first || !p.sum ? p.x : p.sum, i, end, h);
    if (p.residual && (first || !p.sum)) {
      float r[8];
      Load8<DT, KEPT>(p.residual, i, end, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] += r[j];
      Round8<DT>(first ? p.sum : nullptr, i, end, h);
    }
  };
  auto times = [](float (&h)[8], float by) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] *= by;
  };
  float ss = 0.f;
  auto square = [&](const float (&h)[8]) __attribute__((always_inline)) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) t = __builtin_fmaf(h[j], h[j], t);
    ss += t;
  };
  if constexpr (KEPT) {
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int64_t i = at + k * kStep + tid * 8;
      if (i < end) {
        load(i, v[k], true);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < NG; ++k) square(v[k]);
  } else {
    for (int64_t i = at + tid * 8; i < end; i += kStep) {
      load(i, v[0], true);
      square(v[0]);
    }
  }
  ss = Join<WAVES, false>(ss, s_sum);
  // Squares of finite values may leave fp32.  The row is then multiplied by a power
  // of two, which the norm does not see, and its squares are added again: by 2^-80
  // where the sum is infinite (a square is below 2^96 then), by 2^90 where it is so
  // small that squares may have been lost, unless epsilon is far above them (sum and
  // epsilon are below 2^100 then).  No row of ordinary size comes here.
  float by = 1.f, eps = p.eps;
  if (!(ss < __builtin_huge_valf()) || (ss < 0x1p-80f && eps < 0x1p-80f)) {
    by = ss < 1.f ? 0x1p90f : 0x1p-80f;
    eps = p.eps * by * by;
    ss = 0.f;
    if constexpr (KEPT) {
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        times(v[k], by);
        square(v[k]);
      }
    } else {
      for (int64_t i = at + tid * 8; i < end; i += kStep) {
        load(i, v[0], false);
        times(v[0], by);
        square(v[0]);
      }
    }
    if constexpr (WAVES > 1) __syncthreads();  // the sums before were read
    ss = Join<WAVES, false>(ss, s_sum);
  }
  const float rstd = 1.f / sqrtf(ss / (float)p.D + eps);
  auto scale_by_weight = [&](int64_t i, float (&h)[8]) __attribute__((always_inline)) {
    float w[8];
    if (p.weight_f32)
      Load8<kFloat, false>(p.weight, i, p.D, w);
    else
      Load8<DT, false>(p.weight, i, p.D, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = h[j] * rstd * w[j];
  };
  const int64_t blocks = p.D / p.block;
  auto put_scale = [&](int64_t b, const BlockScale &s) __attribute__((always_inline)) {
    if (p.scale_kind == kRnsE8M0)
      static_cast<uint8_t *>(p.scale)[row * blocks + b] = s.e8m0;
    else
      static_cast<float *>(p.scale)[row * blocks + b] = s.scale;
  };
  auto scale_of = [&](unsigned top) __attribute__((always_inline)) {
    const float t = __builtin_bit_cast(float, top);
    return p.scale_kind == kRnsE8M0 ? MxScaleOf(t, 8) : ScaleOf(t, p.y_fp8 ? kFp8Max : kInt8Max);
  };
  uint8_t *y = static_cast<uint8_t *>(p.y);
  // one scale per block of neighbouring threads
  auto quantize_blocks = [&](int64_t i, float (&h)[8]) __attribute__((always_inline)) {
    unsigned top = TopBits(h);
    for (int o = 1; o < (int)p.block / 8; o <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    const BlockScale s = scale_of(top);
    if (i >= p.D) return;
    if (i % p.block == 0) put_scale(i / p.block, s);
    Store8(y, at + i, end, h, s, p);
  };
  const bool per_row = p.block == p.D && p.scale_kind == kRnsFloat;
  if constexpr (KEPT) {
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (k * kStep + tid * 8 < p.D) scale_by_weight(k * kStep + tid * 8, v[k]);
    if (!per_row) {
#pragma unroll
      for (int k = 0; k < NG; ++k) quantize_blocks(k * kStep + tid * 8, v[k]);
      return;
    }
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < NG; ++k) top = max(top, TopBits(v[k]));
    const BlockScale s = scale_of(Join<WAVES, true>(top, s_top));
    if (tid == 0) put_scale(0, s);
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (k * kStep + tid * 8 < p.D) Store8(y, at + k * kStep + tid * 8, end, v[k], s, p);
  } else {
    unsigned top = 0;
    // every thread takes every step: the block's maximum is a lane exchange
    for (int64_t i = tid * 8; i < (p.D + kStep - 1) / kStep * kStep; i += kStep) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[0][j] = 0.f;
      if (i < p.D) {
        load(at + i, v[0], false);
        if (by != 1.f) times(v[0], by);
        scale_by_weight(i, v[0]);
      }
      if (per_row)
        top = max(top, TopBits(v[0]));
      else
        quantize_blocks(i, v[0]);
    }
    if (!per_row) return;
    const BlockScale s = scale_of(Join<WAVES, true>(top, s_top));
    if (tid == 0) put_scale(0, s);
    for (int64_t i = tid * 8; i < p.D; i += kStep) {
      load(at + i, v[0], false);
      if (by != 1.f) times(v[0], by);
      scale_by_weight(i, v[0]);
      Store8(y, at + i, end, v[0], s, p);
    }
  }
}

template <int DT, int THREADS, int NG, bool KEPT> void LaunchRows(RmsNormParams p, hipStream_t s) {
  LaunchInPieces(p.rows, THREADS, [&](int64_t first, unsigned count) {
    p.first = first;
    RmsNormKernel<DT, THREADS, NG, KEPT><<<count, THREADS, 0, s>>>(p);
  });
}

template <int DT> void Launch(const RmsNormParams &p, hipStream_t s) {
  // As few threads as hold the row with one group of 8 values each, then more
  // groups; past the registers the row is read again.  4096 rows with residual,
  // bfloat16, us, the variant taken | the next: 512 values 5.2 | 7.7, 2048 12.8 |
  // 18.9, 8192 41.7 (5.6 TB/s) | 46.9, 16384 83.4 | 123.
  if (p.D <= 512)
    LaunchRows<DT, 64, 1, true>(p, s);
  else if (p.D <= 2048)
    LaunchRows<DT, 256, 1, true>(p, s);
  else if (p.D <= 8192)
    LaunchRows<DT, 512, 2, true>(p, s);
  else if (p.D <= 16384)
    LaunchRows<DT, 512, 4, true>(p, s);
  else
    LaunchRows<DT, 512, 1, false>(p, s);
}

}  // namespace

void LaunchRmsNormQuantize(const RmsNormParams &p, hipStream_t stream) {
  if (p.rows == 0) return;
  if (p.x_dtype == kFloat)
    Launch<kFloat>(p, stream);
  else if (p.x_dtype == kFloat16)
    Launch<kFloat16>(p, stream);
  else
    Launch<kBfloat16>(p, stream);
}

}  // namespace onnxl_amd
