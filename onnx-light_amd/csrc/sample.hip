// A token from each row of logits and a given random number: temperature, top-k,
// top-p and min-p, then the first token, in order of index, at which the kept
// weights add up to more than the random number's share of their sum.
//
// A weight exp((x - max) / T) is a whole number of 2^-kUnit: sums of them have no
// order, so they are the same from run to run and however the work is split, and
// a row's tokens and the borders of top-p are decided exactly on them.  2^-42 of
// the largest weight is far below what separates two tokens' places, and a row of
// 2^21 tokens still adds up in 63 bits.
//
// Nothing is sorted.  What top-k and top-p keep are the tokens before a border in
// the order of the logits, which is found in steps: the row's largest logit; counts
// (top-k) or weights (top-p) in bins of equal width below it, and the bin with the
// border; the tokens of that bin, or of it and those above, in a list; their border
// by its bits.  The kept weights are added up in chunks of consecutive tokens, the
// chunk of the random number's share is found, and its token.  A row whose list
// would not fit has its border found by the bits of all its logits.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"

namespace onnxl_amd {
namespace {

constexpr int kUnit = 42, kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048, kList = 4096, kChunks = 1024;
constexpr float kOctaves = 44.f;  // of weights that the bins span; the last bin has the rest
typedef unsigned long long u64;

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

struct Shared {
  double power[32];  // 2^(-j / 32)
  u64 wave[kWaves];
  u64 digit[256];
  u64 chunk[kChunks];
  u64 bin[kBins];
  u64 list[kList];  // key << 32 | index
  u64 out[2];
  unsigned n, at;
};

// A row, and what its weights go by.
template <int DT> struct Row {
  const void *x;
  int64_t base;
  int vocab;
  float top, per_bin;  // the largest logit; bins a unit of it
  double octaves;      // log2(e) / T
  double least;        // min_p, 0: none
  const double *power;

  __device__ float At(int i) const {
    float v[1];
    Load<1>(i, v);
    return v[0];
  }
  template <int N> __device__ __forceinline__ void Load(int i, float (&v)[N]) const {
    if constexpr (DT == kFloat) {
      __builtin_memcpy(v, static_cast<const float *>(x) + base + i, 4 * N);
    } else {
      uint16_t u[N];
      __builtin_memcpy(u, static_cast<const uint16_t *>(x) + base + i, 2 * N);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = DT == kFloat16 ? F16ToF32(u[j]) : Bf16ToF32(u[j]);
    }
  }
  // 2^-t by a table of the 32nds and the series of the rest, |r| <= ln 2 / 64, to
  // about 2^-48
  __device__ __forceinline__ double Weight(float v) const {
    if (v == top) return 1.0;
    const double t = ((double)top - (double)v) * octaves;
    if (!(t < 1000.0)) return 0.0;
    const double k = rint(32.0 * t), r = (k * 0.03125 - t) * 0.6931471805599453094;
    double p = fma(r, 1.0 / 120, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const int i = (int)k;
    return ldexp(power[i & 31] * p, -(i >> 5));
  }
  __device__ static __forceinline__ u64 Whole(double w) { return (u64)rint(w * (double)(u64(1) << kUnit)); }
  // what min_p leaves of a token's weight
  __device__ __forceinline__ u64 Kept(float v) const {
    const double w = Weight(v);
    return w >= least ? Whole(w) : 0;
  }
  __device__ __forceinline__ int Bin(float v) const {
    const float b = (top - v) * per_bin;  // falls with v, as every rounding in it does
    return v == top ? 0 : b < (float)(kBins - 1) ? (int)b : kBins - 1;
  }
  // f(logits, first index, how many) for 16 bytes at a time, four of them on their way;
  // every thread of the workgroup comes by the same number of times
  template <typename F> __device__ __forceinline__ void Each(F &&f) const {
    constexpr int N = DT == kFloat ? 4 : 8, U = 4;
    for (int i0 = 0; i0 < vocab; i0 += U * N * kThreads) {
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + (u * kThreads + (int)threadIdx.x) * N;
        if (i + N <= vocab) {
          Load<N>(i, v[u]);
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) v[u][j] = i + j < vocab ? At(i + j) : -__builtin_huge_valf();
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) f(v[u], i0 + (u * kThreads + (int)threadIdx.x) * N, std::integral_constant<int, N>{});
    }
  }
};

template <typename T> __device__ __forceinline__ T WaveSum(T v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// Sums of all threads up to and with this one; `all` of all.
__device__ __forceinline__ u64 GroupScan(Shared &s, u64 v, u64 &all) {
  const int lane = threadIdx.x % 64;
  for (int o = 1; o < 64; o <<= 1) {
    const u64 w = __shfl_up(v, o);
    if (lane >= o) v += w;
  }
  __syncthreads();
  if (lane == 63) s.wave[threadIdx.x / 64] = v;
  __syncthreads();
  all = 0;
  u64 before = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < (int)threadIdx.x / 64) before += s.wave[w];
    all += s.wave[w];
  }
  return v + before;
}

// The 32-bit number at which units, counted from the largest numbers down, reach
// `want` (the smallest number, where they do not); `above`: the units of larger ones.
// visit(f) calls f(number, unit) for the workgroup's numbers.
template <typename V> __device__ unsigned Border(Shared &s, u64 want, u64 &above, V &&visit) {
  unsigned prefix = 0;
  above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) s.digit[threadIdx.x] = 0;
    __syncthreads();
    visit([&](unsigned number, u64 unit) __attribute__((always_inline)) {
      if (shift == 24 || number >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s.digit[number >> shift & 255], unit);
    });
    __syncthreads();
    if (threadIdx.x < 64) {
      // four digits a lane, the largest first
      const int lane = threadIdx.x;
      u64 d[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += d[j] = s.digit[255 - 4 * lane - j];
      u64 upto = sum;
      for (int o = 1; o < 64; o <<= 1) {
        const u64 w = __shfl_up(upto, o);
        if (lane >= o) upto += w;
      }
      const u64 reach = __ballot(above + upto >= want);
      if (lane == (reach ? __builtin_ctzll(reach) : 63)) {
        u64 a = above + upto - sum;
        int j = 0;
        for (; j < 3 && a + d[j] < want; ++j) a += d[j];
        s.out[0] = a;
        s.at = 255 - 4 * lane - j;
      }
    }
    __syncthreads();
    above = s.out[0];
    prefix |= s.at << shift;
  }
  return prefix;
}

// The token at which the weights up to it reach this is the last that top_p keeps.
__device__ __forceinline__ u64 WantOf(float top_p, u64 total) {
  const u64 w = (u64)ceil((double)fmaxf(top_p, 0.f) * (double)total);
  return w ? w : 1;
}

template <int DT> __global__ __launch_bounds__(kThreads) void SampleRowKernel(const SampleParams p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid % 64;
  const int64_t row = p.first + blockIdx.x;
  Row<DT> r{p.x, row * p.vocab, p.vocab, 0.f, 0.f, 0.0, 0.0, s.power};
  auto answer = [&](int64_t token, float probability) {
    if (p.token64)
      static_cast<int64_t *>(p.token)[row] = token;
    else
      static_cast<int32_t *>(p.token)[row] = (int32_t)token;
    if (p.probability) p.probability[row] = probability;
  };
  if (tid < 32) s.power[tid] = exp2(-tid / 32.0);

  // the largest logit, and the lowest index that has it
  u64 best = 0;
  r.Each([&](const auto &v, int i, auto n) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const u64 k = (u64)KeyOf(v[j]) << 32 | (0xffffffffu - (unsigned)(i + j));
      best = k > best ? k : best;
    }
  });
  for (int o = 32; o > 0; o >>= 1) {
    const u64 k = __shfl_xor(best, o);
    best = k > best ? k : best;
  }
  if (lane == 0) s.wave[tid / 64] = best;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) best = s.wave[i] > best ? s.wave[i] : best;
  const unsigned top = (unsigned)(best >> 32);
  const float T = p.temperature ? p.temperature[row] : 1.f;
  int64_t k = 0;
  if (p.top_k) k = p.k64 ? static_cast<const int64_t *>(p.top_k)[row] : (int64_t) static_cast<const int32_t *>(p.top_k)[row];
  if (k >= p.vocab) k = 0;
  if (top == 0 || !(T > 0.f) || k == 1) {
    if (tid == 0) answer(top == 0 ? -1 : (int64_t)(0xffffffffu - (unsigned)best), top == 0 ? 0.f : 1.f);
    return;
  }
  const float tp = p.top_p ? p.top_p[row] : 1.f, mp = p.min_p ? p.min_p[row] : 0.f;
  const bool cuts = tp < 1.f;
  r.top = LogitOf(top);
  r.octaves = 1.4426950408889634074 / (double)T;
  r.per_bin = (float)(r.octaves * (kBins / kOctaves));
  r.least = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;

  // the bin with the border, and how much is in those above: counts for top-k, weights
  // for top-p
  auto bin_of = [&](u64 want, u64 &above, u64 &in, u64 &all) {
    const u64 a = s.bin[2 * tid], b = s.bin[2 * tid + 1], upto = GroupScan(s, a + b, all);
    if (want > all) want = all;
    __syncthreads();
    if (upto >= want && upto - a - b < want) {
      const bool second = upto - b < want;
      s.at = 2 * tid + second;
      s.out[0] = second ? upto - b : upto - a - b;
      s.out[1] = second ? b : a;
    }
    __syncthreads();
    above = s.out[0];
    in = s.out[1];
    return (int)s.at;
  };
  auto clear = [&] {
    s.bin[2 * tid] = s.bin[2 * tid + 1] = 0;
    s.chunk[tid] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
  };
  clear();
  int border_bin = kBins;  // all below it in number is kept
  u64 above = 0, in = 0, all = 0, want = 0;
  if (k > 0) {
    r.Each([&](const auto &v, int, auto n) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < n; ++j)
        if (KeyOf(v[j])) atomicAdd(&s.bin[r.Bin(v[j])], 1ull);
    });
    __syncthreads();
    border_bin = bin_of((u64)k, above, in, all);
    if (all <= (u64)k) {
      k = 0;  // nothing to leave out
      border_bin = kBins;
      __syncthreads();
      clear();
    }
  }
  if (k <= 0 && cuts) {
    r.Each([&](const auto &v, int, auto n) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < n; ++j)
        if (KeyOf(v[j])) atomicAdd(&s.bin[r.Bin(v[j])], r.Whole(r.Weight(v[j])));
    });
    __syncthreads();
    u64 none;
    const u64 total = (bin_of(~u64(0), above, none, all), all);
    want = WantOf(tp, total);
    __syncthreads();
    border_bin = bin_of(want, above, none, all);
  }
  // top-k lists its bin and all above it, top-p its bin alone; what is kept for certain
  // goes to its chunk
  const int size = (p.vocab + kChunks * 8 - 1) / (kChunks * 8) * 8;  // tokens of a chunk
  const bool few = k > 0 && above + in <= kList;
  auto take = [&](bool listed, float v, int i) __attribute__((always_inline)) {
    const u64 vote = __ballot(listed);
    if (!vote) return;
    unsigned at = 0;
    if (lane == (int)__builtin_ctzll(vote)) at = atomicAdd(&s.n, (unsigned)__popcll(vote));
    at = __shfl(at, (int)__builtin_ctzll(vote)) + (unsigned)__popcll(vote & ((u64(1) << lane) - 1));
    if (listed && at < kList) s.list[at] = (u64)KeyOf(v) << 32 | (unsigned)i;
  };
  const bool by_list = k > 0 ? few : cuts;
  if (k <= 0 || few) {
    r.Each([&](const auto &v, int i, auto n) __attribute__((always_inline)) {
      u64 sum = 0;
#pragma unroll
      for (int j = 0; j < n; ++j) {
        const bool is = KeyOf(v[j]) != 0;
        const int b = r.Bin(v[j]);
        if (by_list) take(is && (k > 0 ? b <= border_bin : b == border_bin), v[j], i + j);
        if (k <= 0 && is && b < border_bin) sum += r.Kept(v[j]);
      }
      if (sum) atomicAdd(&s.chunk[i / size], sum);
    });
    __syncthreads();
  }
  // kept are the tokens with a larger key than `border`, and of those with that key the
  // ones up to index `last`
  unsigned border = 0, last = 0;
  const unsigned n = s.n;
  if (by_list && n <= kList) {
    constexpr int E = kList / kThreads;
    u64 e[E], w[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const unsigned i = j * kThreads + tid;
      e[j] = i < n ? s.list[i] : 0;
      w[j] = e[j] ? r.Whole(r.Weight(LogitOf((unsigned)(e[j] >> 32)))) : 0;
    }
    auto counts = [&](auto &&f) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (e[j]) f((unsigned)(e[j] >> 32), 1ull);
    };
    u64 over = 0, ties = ~u64(0);
    if (k > 0) {
      border = Border(s, (u64)k, over, counts);
      ties = (u64)k - over;
      if (cuts) {
        u64 mine = 0, total = 0;
#pragma unroll
        for (int j = 0; j < E; ++j)
          if ((unsigned)(e[j] >> 32) > border) mine += w[j];
        GroupScan(s, mine, total);
        want = WantOf(tp, total + ties * r.Whole(r.Weight(LogitOf(border))));
      }
      above = 0;
    }
    if (cuts) {
      const unsigned floor = border;
      const unsigned b = Border(s, want - above, over, [&](auto &&f) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (e[j] && (unsigned)(e[j] >> 32) >= floor) f((unsigned)(e[j] >> 32), w[j]);
      });
      const u64 one = r.Whole(r.Weight(LogitOf(b))), left = want - above > over ? want - above - over : 0;
      const u64 m = one ? (left + one - 1) / one : 1;
      ties = b == border && ties < m ? ties : m;
      border = b;
    }
    // the first `ties` of the equal ones: the largest numbers ~index
    u64 none;
    last = ~Border(s, ties, none, [&](auto &&f) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (e[j] && (unsigned)(e[j] >> 32) == border) f(~(unsigned)e[j], 1ull);
    });
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const unsigned key = (unsigned)(e[j] >> 32), i = (unsigned)e[j];
      if (key > border || (e[j] && key == border && i <= last)) {
        const u64 kept = r.Kept(LogitOf(key));
        if (kept) atomicAdd(&s.chunk[i / size], kept);
      }
    }
    __syncthreads();
  } else if (k > 0 || cuts) {
    // by the bits of all logits
    auto each = [&](auto &&f) {
      r.Each([&](const auto &v, int i, auto m) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < m; ++j) {
          const unsigned key = KeyOf(v[j]);
          if (key) f(key, v[j], i + j);
        }
      });
    };
    u64 over = 0, ties = ~u64(0), total = 0;
    if (k > 0) {
      border = Border(s, (u64)k, over, [&](auto &&f) { each([&](unsigned key, float, int) { f(key, 1ull); }); });
      ties = (u64)k - over;
      if (cuts) {
        u64 mine = 0;
        each([&](unsigned key, float v, int) {
          if (key > border) mine += r.Whole(r.Weight(v));
        });
        GroupScan(s, mine, total);
        want = WantOf(tp, total + ties * r.Whole(r.Weight(LogitOf(border))));
      }
    }
    if (cuts) {
      const unsigned floor = border;
      const unsigned b = Border(s, want, over, [&](auto &&f) {
        each([&](unsigned key, float v, int) {
          if (key >= floor) f(key, r.Whole(r.Weight(v)));
        });
      });
      const u64 one = r.Whole(r.Weight(LogitOf(b))), left = want > over ? want - over : 0;
      const u64 m = one ? (left + one - 1) / one : 1;
      ties = b == border && ties < m ? ties : m;
      border = b;
    }
    u64 none;
    last = ~Border(s, ties, none, [&](auto &&f) {
      each([&](unsigned key, float, int i) {
        if (key == border) f(~(unsigned)i, 1ull);
      });
    });
    __syncthreads();
    s.chunk[tid] = 0;
    __syncthreads();
    each([&](unsigned key, float v, int i) {
      if (key > border || (key == border && (unsigned)i <= last)) {
        const u64 kept = r.Kept(v);
        if (kept) atomicAdd(&s.chunk[i / size], kept);
      }
    });
    __syncthreads();
  }

  // the chunk, then the token, at which the kept weights pass the share
  u64 total;
  const u64 mine = s.chunk[tid], upto = GroupScan(s, mine, total);
  float u = p.uniform[row];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  u64 share = (u64)((double)u * (double)total);
  if (share >= total) share = total - 1;
  if (upto > share && upto - mine <= share) {
    s.at = tid;
    s.out[0] = share - (upto - mine);
  }
  __syncthreads();
  const int from = (int)s.at * size;
  u64 left = s.out[0];
  for (int i0 = 0; i0 < size; i0 += kThreads) {
    const int i = from + i0 + tid;
    u64 kept = 0;
    float v = 0.f;
    if (i0 + tid < size && i < p.vocab) {
      v = r.At(i);
      const unsigned key = KeyOf(v);
      if (key > border || (key != 0 && key == border && (unsigned)i <= last)) kept = r.Kept(v);
    }
    u64 sum;
    const u64 incl = GroupScan(s, kept, sum);
    if (incl > left && incl - kept <= left) answer(i, (float)(r.Weight(v) / ((double)total * 0x1p-42)));
    if (sum > left) return;
    left -= sum;
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
