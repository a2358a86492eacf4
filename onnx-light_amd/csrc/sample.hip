// A token from each row of logits and a given random number: temperature, top-k,
// top-p and min-p, then the first token, in order of index, at which the kept
// weights add up to more than the random number's share of their sum.
//
// A weight exp((x - max) / T) is a whole number of 2^-kUnit: sums of them have no
// order, so they are the same from run to run and however the work is split, and
// a row's tokens and the borders of top-p are decided exactly on them.  2^-42 of
// the largest weight is far below what separates two tokens' places, and a row of
// 2^21 tokens still adds up in 63 bits.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"

namespace onnxl_amd {
namespace {

constexpr int kUnit = 42, kThreads = 1024;
typedef unsigned long long u64;

// exp(-d), d >= 0, to about 2^-50: 2^k times the series of the rest, |r| <= ln 2 / 2.
__device__ __forceinline__ double ExpMinus(double d) {
  if (!(d < 700.0)) return 0.0;
  const double k = rint(d * 1.4426950408889634074);
  const double r = fma(k, 2.3190468138462996e-17, fma(k, 0.6931471805599453094, -d));
  double p = 1.0 / 479001600;
  p = fma(p, r, 1.0 / 39916800);
  p = fma(p, r, 1.0 / 3628800);
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, -(int)k);
}

template <int DT> __device__ __forceinline__ float Logit(const void *x, int64_t at) {
  if constexpr (DT == kFloat) return static_cast<const float *>(x)[at];
  const uint16_t u = static_cast<const uint16_t *>(x)[at];
  return DT == kFloat16 ? F16ToF32(u) : Bf16ToF32(u);
}

// Whole numbers in the order of the logits: NaN and -inf, which are never
// chosen, 0; the zeros equal.
__device__ __forceinline__ unsigned KeyOf(float x) {
  if (!(x > -__builtin_huge_valf())) return 0;
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float LogitOf(unsigned key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <typename T> __device__ __forceinline__ T WaveSum(T v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

struct Shared {
  u64 wave[kThreads / 64];
  u64 mass[256];
  unsigned count[256];
  u64 out[2];
  unsigned digit;
};

// The sum over the workgroup, for everybody.
__device__ __forceinline__ u64 GroupSum(Shared &s, u64 v) {
  v = WaveSum(v);
  __syncthreads();
  if (threadIdx.x % 64 == 0) s.wave[threadIdx.x / 64] = v;
  __syncthreads();
  u64 t = 0;
  for (int i = 0; i < kThreads / 64; ++i) t += s.wave[i];
  return t;
}

// A row as the kernels see it.
template <int DT> struct Row {
  const void *x;
  int64_t at;
  int vocab;
  float top;
  double inv;  // 1 / T
  __device__ unsigned Key(int i) const { return KeyOf(Logit<DT>(x, at + i)); }
  __device__ double Weight(unsigned key) const {
    const float v = LogitOf(key);
    return v == top ? 1.0 : ExpMinus(((double)top - (double)v) * inv);
  }
  __device__ u64 Whole(unsigned key) const { return (u64)rint(Weight(key) * (double)(u64(1) << kUnit)); }
};

// The smallest key among the first `want` whole units in the order of the keys, where every
// token above `floor` counts `unit(key)`: `above`, what the larger keys add up to.
template <int DT, bool MASS> __device__ unsigned Border(Shared &s, const Row<DT> &r, unsigned floor, u64 want, u64 &above) {
  unsigned prefix = 0;
  above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) s.mass[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < r.vocab; i += kThreads) {
      const unsigned k = r.Key(i);
      if (k < floor || k == 0 || (shift < 24 && k >> (shift + 8) != prefix >> (shift + 8))) continue;
      atomicAdd(&s.mass[k >> shift & 255], MASS ? r.Whole(k) : 1ull);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 sum = above;
      int d = 255;
      for (; d > 0 && sum + s.mass[d] < want; --d) sum += s.mass[d];
      s.out[0] = sum;
      s.digit = d;
    }
    __syncthreads();
    above = s.out[0];
    prefix |= s.digit << shift;
  }
  return prefix;
}

template <int DT> __global__ __launch_bounds__(kThreads) void SampleRowKernel(const SampleParams p) {
  __shared__ Shared s;
  const int tid = threadIdx.x;
  const int64_t row = p.first + blockIdx.x;
  Row<DT> r{p.x, row * p.vocab, p.vocab, 0.f, 1.0};
  auto answer = [&](int64_t token, float probability) {
    if (p.token64)
      static_cast<int64_t *>(p.token)[row] = token;
    else
      static_cast<int32_t *>(p.token)[row] = (int32_t)token;
    if (p.probability) p.probability[row] = probability;
  };

  // the largest logit; the lowest index that has it
  u64 best = 0;
  for (int i = tid; i < p.vocab; i += kThreads) {
    const u64 k = (u64)r.Key(i) << 32 | (0xffffffffu - (unsigned)i);
    best = k > best ? k : best;
  }
  for (int o = 32; o > 0; o >>= 1) {
    const u64 k = __shfl_xor(best, o);
    best = k > best ? k : best;
  }
  if (tid % 64 == 0) s.wave[tid / 64] = best;
  __syncthreads();
  for (int i = 0; i < kThreads / 64; ++i) best = s.wave[i] > best ? s.wave[i] : best;
  const unsigned top = (unsigned)(best >> 32);
  if (top == 0) {
    if (tid == 0) answer(-1, 0.f);
    return;
  }
  const float T = p.temperature ? p.temperature[row] : 1.f;
  if (!(T > 0.f)) {
    if (tid == 0) answer((int64_t)(0xffffffffu - (unsigned)best), 1.f);
    return;
  }
  r.top = LogitOf(top);
  r.inv = 1.0 / (double)T;

  // kept are the keys above `border`, and of those equal to it the first `ties`
  unsigned border = 1;
  u64 ties = (u64)p.vocab;
  u64 total;
  int64_t k = 0;
  if (p.top_k) k = p.k64 ? static_cast<const int64_t *>(p.top_k)[row] : (int64_t) static_cast<const int32_t *>(p.top_k)[row];
  if (k > 0 && k < p.vocab) {
    u64 above;
    border = Border<DT, false>(s, r, 1, (u64)k, above);
    ties = (u64)k - above;
  }
  auto mass = [&] {
    u64 sum = 0, equal = 0;
    for (int i = tid; i < p.vocab; i += kThreads) {
      const unsigned key = r.Key(i);
      if (key > border) sum += r.Whole(key);
      equal += key == border;
    }
    sum = GroupSum(s, sum);
    equal = GroupSum(s, equal);
    ties = equal < ties ? equal : ties;
    return border ? sum + ties * r.Whole(border) : sum;
  };
  total = mass();
  const float tp = p.top_p ? p.top_p[row] : 1.f;
  if (tp < 1.f) {
    // the token at which the weights before it reach top_p of all is the first left out
    double want = ceil((double)fmaxf(tp, 0.f) * (double)total);
    u64 above;
    const u64 need = want < 1.0 ? 1 : (u64)want;
    const unsigned b = Border<DT, true>(s, r, border, need, above);
    const u64 one = r.Whole(b), left = need > above ? need - above : 0;
    const u64 n = one ? (left + one - 1) / one : 1;
    ties = b == border && ties < n ? ties : n;
    border = b;
    total = mass();
  }
  const float mp = p.min_p ? p.min_p[row] : 0.f;
  const bool cut = mp > 0.f;
  const double least = fmin((double)mp, 1.0);

  // tiles of consecutive tokens, one a thread, up to the one that passes the share
  u64 want = 0, upto = 0, seen = 0;
  for (int pass = cut ? 0 : 1; pass < 2; ++pass) {
    if (pass == 1) {
      if (cut) total = upto;
      float u = p.uniform[row];
      u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
      want = (u64)((double)u * (double)total);
      if (want >= total) want = total - 1;
    }
    upto = seen = 0;
    for (int base = 0; base < p.vocab; base += kThreads) {
      const int i = base + tid;
      const unsigned key = i < p.vocab ? r.Key(i) : 0;
      const bool equal = key == border && key != 0;
      // which of the equal ones this is
      const u64 vote = __ballot(equal);
      const int lane = tid % 64;
      u64 before = seen + __popcll(vote & ((u64(1) << lane) - 1));
      __syncthreads();
      if (lane == 0) s.wave[tid / 64] = __popcll(vote);
      __syncthreads();
      for (int w = 0; w < kThreads / 64; ++w) {
        if (w < tid / 64) before += s.wave[w];
        seen += s.wave[w];
      }
      u64 mine = 0;
      if (key > border || (equal && before < ties)) mine = !cut || r.Weight(key) >= least ? r.Whole(key) : 0;
      const u64 sum = GroupSum(s, mine);
      if (pass == 1 && upto + sum > want) {
        u64 incl = mine;
        for (int o = 1; o < 64; o <<= 1) {
          const u64 v = __shfl_up(incl, o);
          if (lane >= o) incl += v;
        }
        for (int w = 0; w < tid / 64; ++w) incl += s.wave[w];
        incl += upto;
        if (incl > want && incl - mine <= want) answer(i, (float)(r.Weight(key) / ((double)total * 0x1p-42)));
        return;
      }
      upto += sum;
    }
  }
}

}  // namespace

size_t SampleScratchBytes(const SampleParams &) { return 0; }

void LaunchSampleTokens(const SampleParams &whole, void *, hipStream_t stream) {
  SampleParams p = whole;
  LaunchInPieces(p.rows, kThreads, [&](int64_t first, unsigned count) {
    p.first = first;
    if (p.dtype == kFloat)
      SampleRowKernel<kFloat><<<count, kThreads, 0, stream>>>(p);
    else if (p.dtype == kFloat16)
      SampleRowKernel<kFloat16><<<count, kThreads, 0, stream>>>(p);
    else
      SampleRowKernel<kBfloat16><<<count, kThreads, 0, stream>>>(p);
  });
}

}  // namespace onnxl_amd
