// A token from each row of logits and a given random number: temperature, top-k,
// top-p and min-p, then the first token, in order of index, at which the kept
// weights add up to more than the random number's share of their sum.
//
// A weight exp((x - max) / T) is a whole number of 2^-42: sums of them have no
// order, so they are the same from run to run and however the work is split, and
// a row's tokens and the borders of top-p are decided exactly on them, by whole shares.  2^-42 of
// the largest weight is far below what separates two tokens' places, and a row of
// 2^21 tokens still adds up in 63 bits.
//
// The row is not sorted.  What top-k and top-p keep are the tokens before a border in
// the order of the logits, which is found in steps: the row's largest logit; counts
// (top-k) or weights (top-p) in bins of equal width below it, and the bin with the
// border; the tokens of that bin, or of it and those above, in a list, which is
// sorted.  The kept weights are added up in chunks of consecutive tokens, the
// chunk of the random number's share is found, and its token.  A row whose list
// would not fit has its border found by the bits of all its logits.
//
// Additions to LDS cost most, about a lane a clock: a top_k of a few hundred goes by the
// largest logits of many small groups instead of bins, and for top_p a sample of the row
// says from which logit on it has bins at all.
//
// A row's loads take little of it: 256 rows of 131072 bfloat16 logits with top_p 0.9, 67 MB,
// take 96 us, of which the vector unit issues on 60 %, a weight's number looked up for each
// token twice, and LDS is waited for.  One row of 128000 fp32 logits, top_k 50, 27 us: three
// launches of latencies.
//
// Many rows, or short ones, have a workgroup each; of few long ones a row is shared by
// several, in a launch for each step, whose last workgroup joins what they found.
#include <type_traits>

#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"

namespace onnxl_amd {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048, kList = 4096, kChunks = 1024;
constexpr int kCodes = 4096;      // bfloat16 numbers of a sign, 32 octaves, whose weights are kept
constexpr float kOctaves = 44.f;  // of weights that the bins span; the last bin has the rest
constexpr float kMaxFloat = 0x1.fffffep127f, kMinFloat = 0x1p-126f;
typedef unsigned long long u64;
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// Whole numbers in the order of the logits: NaN and -inf, which are never
// chosen, 0; the zeros equal.
__device__ __forceinline__ bool IsLogit(float x) { return x > -__builtin_huge_valf(); }
__device__ __forceinline__ unsigned KeyOf(float x) {
  if (!IsLogit(x)) return 0;
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float LogitOf(unsigned key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Shared {
  double power[64];  // 2^(-j / 64)
  u64 wave[kWaves];
  u64 digit[256];
  u64 chunk[kChunks];
  u64 bin[kBins];
  u64 list[kList];         // key << 32 | index
  u64 queue[kWaves][128];  // of a wave: logit << 32 | index, kept for certain
  u64 code[2][kCodes];     // weights of bfloat16 numbers, of both signs
  u64 out[2];
  unsigned votes[2][kWaves];
  unsigned n, at;
  int last;
};

// ---- sums over lanes and threads ----------------------------------------------

template <int CTRL, int ROWS> __device__ __forceinline__ u64 AddFrom(u64 v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((u64)hi << 32 | lo);
}
// Of a row of 16 lanes, in its last.
__device__ __forceinline__ u64 RowSum(u64 v) {
  v = AddFrom<0x111, 0xf>(v);
  v = AddFrom<0x112, 0xf>(v);
  v = AddFrom<0x114, 0xf>(v);
  return AddFrom<0x118, 0xf>(v);
}
// Sums of the lanes up to and with this one: inside rows of 16, then the last lane of a
// row to the next row, of the second to the third and fourth.
__device__ __forceinline__ u64 WaveScan(u64 v) {
  v = RowSum(v);
  v = AddFrom<0x142, 0xa>(v);
  return AddFrom<0x143, 0xc>(v);
}
// Sums of all threads up to and with this one; `all` of all.
__device__ __forceinline__ u64 GroupScan(Shared &s, u64 v, u64 &all) {
  v = WaveScan(v);
  __syncthreads();
  if (threadIdx.x % 64 == 63) s.wave[threadIdx.x / 64] = v;
  __syncthreads();
  u64 before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < (int)threadIdx.x / 64 ? s.wave[w] : 0;
    all += s.wave[w];
  }
  return v + before;
}
__device__ __forceinline__ u64 GroupMax(Shared &s, u64 v) {
  for (int o = 32; o > 0; o >>= 1) {
    const u64 w = __shfl_xor(v, o);
    v = w > v ? w : v;
  }
  __syncthreads();
  if (threadIdx.x % 64 == 0) s.wave[threadIdx.x / 64] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = s.wave[w] > v ? s.wave[w] : v;
  return v;
}

// ---- a row ----------------------------------------------------------------------

template <int DT> struct Row {
  static constexpr int N = DT == kFloat ? 4 : 8;  // logits of a load
  const void *x;
  int64_t base;
  int vocab;
  int shift;              // log2 of a chunk's tokens
  bool infinite;          // the largest logit is: it counts as 0, and all others as -inf
  // what weights go by
  float top, per_bin;     // the largest logit
  float floor, least;     // logits below weigh nothing: 2^-500; less than min_p
  double octaves, none;   // log2(e) / T; a difference of 500 octaves
  const double *power;
  // bfloat16: weights of the numbers, without their sign, from `low` on
  const u64 *code;
  int low;

  __device__ __forceinline__ void Weigh(unsigned largest, float T, float min_p) {
    infinite = LogitOf(largest) > kMaxFloat;
    top = infinite ? 0.f : LogitOf(largest);
    octaves = fmax(1.4426950408889634074 / (double)T, 1e-300);
    none = 500.0 / octaves;
    // any positive number keeps the order of the bins
    per_bin = fminf(fmaxf((float)(octaves * (kBins / kOctaves)), kMinFloat), kMaxFloat);
    floor = fmaxf((float)((double)top - none), -kMaxFloat);  // rounded: at most 1000 octaves down
    least = floor;
    if (min_p > 0.f) {
      const double m = fmin((double)min_p, 1.0);
      least = fmaxf(floor, FirstLogit([&](float v) { return Weight(v, floor) >= m; }));
    }
  }
  // The smallest logit that `is` holds for, as it does for the largest and from some
  // logit on; 64 places at a time, the same for every wave.
  template <typename F> __device__ __forceinline__ float FirstLogit(F &&is) const {
    unsigned lo = KeyOf(-kMaxFloat), hi = KeyOf(top);  // in lo .. hi
    while (lo < hi) {
      const unsigned step = (hi - lo) / 64 + 1, at = lo + min((threadIdx.x % 64) * step, hi - lo);
      const u64 yes = __ballot(is(LogitOf(at)));
      if (!yes) {
        lo = lo + min(63 * step, hi - lo) + 1;  // hi is one
        if (lo > hi) lo = hi;
      } else {
        const unsigned first = (unsigned)__builtin_ctzll(yes);
        hi = lo + min(first * step, hi - lo);
        if (first) lo = min(lo + (first - 1) * step + 1, hi);
      }
    }
    return LogitOf(hi);
  }
  __device__ __forceinline__ void Get(int i, float (&v)[N]) const {
    if constexpr (DT == kFloat) {
      __builtin_memcpy(v, static_cast<const float *>(x) + base + i, 16);
    } else {
      uint16_t u[N];
      __builtin_memcpy(u, static_cast<const uint16_t *>(x) + base + i, 16);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = DT == kFloat16 ? F16ToF32(u[j]) : Bf16ToF32(u[j]);
    }
  }
  __device__ __forceinline__ float As(float v) const {
    return !infinite ? v : v > kMaxFloat ? 0.f : -__builtin_huge_valf();
  }
  __device__ __forceinline__ float Raw(int i) const {
    if constexpr (DT == kFloat) return static_cast<const float *>(x)[base + i];
    const uint16_t u = static_cast<const uint16_t *>(x)[base + i];
    return DT == kFloat16 ? F16ToF32(u) : Bf16ToF32(u);
  }
  __device__ __forceinline__ float At(int i) const { return As(Raw(i)); }
  // 2^-t of t = (top - v) log2(e) / T by a table of the 64ths, whose number stands in the
  // low bits of a sum with 1.5 2^46, and the series of the rest, at most 1/128, to 2^-44;
  // of what is not from `from` on 2^-500.
  __device__ __forceinline__ double Weight(float v, float from) const {
    const double d = v >= from ? (double)top - (double)v : none;
    const double sum = fma(d, octaves, 0x1.8p46), r = fma(-d, octaves, sum - 0x1.8p46);
    double p = fma(r, 0x1.3b2ab6fba4e77p-7, 0x1.c6b08d704a0bfp-5);
    p = fma(p, r, 0x1.ebfbdff82c58ep-3);
    p = fma(p, r, 0x1.62e42fefa39efp-1);
    p = fma(p, r, 1.0);
    const unsigned k = (unsigned)__builtin_bit_cast(u64, sum);
    const u64 w = __builtin_bit_cast(u64, power[k & 63] * p);
    return __builtin_bit_cast(double, w - ((u64)(k >> 6) << 52));
  }
  // in units of 2^-42, the last place of numbers from 1024 to 2048
  __device__ __forceinline__ u64 Whole(float v) const { return Units(Weight(v, floor)); }
  // and what min_p leaves of it
  __device__ __forceinline__ u64 Kept(float v) const { return Units(Weight(v, least)); }
  __device__ static __forceinline__ u64 Units(double w) {
    return __builtin_bit_cast(u64, w + 1024.0) - __builtin_bit_cast(u64, 1024.0);
  }
  // Makes the weights of a bfloat16 row's numbers from 4 octaves above the largest logit's
  // size to 28 below: one read in LDS for a logit, where the exponential takes 24
  // instructions, 11 of them in 64 bits.
  __device__ __forceinline__ void MakeCodes(u64 (&table)[2][kCodes]) {
    if constexpr (DT == kBfloat16) {
      code = table[0];
      low = min(max((int)(__builtin_bit_cast(unsigned, top) >> 16 & 0x7fff) + 512 - kCodes, 0), 0x7f80 - kCodes);
#pragma unroll 1
      for (int i = threadIdx.x; i < kCodes; i += kThreads) {
        const float v = __builtin_bit_cast(float, (unsigned)(low + i) << 16);
        table[0][i] = v <= top ? Whole(v) : 0;
        table[1][i] = -v <= top ? Whole(-v) : 0;
      }
      __syncthreads();
    }
  }
  // Whole weights of logits that are at least `from`, 0 of others.
  __device__ __forceinline__ void Weights(const float (&v)[N], float from, u64 (&w)[N]) const {
    if constexpr (DT == kBfloat16) {
      bool other = false;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const unsigned u = __builtin_bit_cast(unsigned, v[j]);
        const unsigned i = (u >> 16 & 0x7fff) - (unsigned)low;
        const bool has = v[j] >= from;
        w[j] = code[(u >> 31) * kCodes + (i & (kCodes - 1))];
        if (!has) w[j] = 0;
        other |= has && i >= (unsigned)kCodes;
      }
      if (!__ballot(other)) return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = Units(Weight(v[j], from));
  }
  // Adds the 16 bytes' weights from token i on to their chunk, of a row of 16 lanes at once
  // where that is in one.
  __device__ __forceinline__ void AddToChunk(u64 *chunk, int i, u64 sum) const {
    if (16 * N <= 1 << shift) {
      sum = RowSum(sum);
      if (threadIdx.x % 16 != 15) sum = 0;
    }
    if (sum) atomicAdd(&chunk[i >> shift], sum);
  }
  // falls with v, as every rounding in it does; anything for a NaN
  __device__ __forceinline__ int Bin(float v) const {
    return (int)__builtin_amdgcn_fmed3f((top - v) * per_bin, 0.f, (float)(kBins - 1)) & (kBins - 1);
  }
  // f(logits, the first one's index, i) for N at a time of the tokens from..to - 1, four to
  // eight loads of a thread on their way; i is the index of the first of them that is new:
  // those before it, and past the end, are -inf
  template <typename F> __device__ __forceinline__ void Each(int from, int to, F &&f) const {
    constexpr int step = N * kThreads, U = 4;
    const bool whole = to - from >= N;
    auto get = [&](int i) __attribute__((always_inline)) {
      v4u r = {};
      if (whole) {
        __builtin_memcpy(&r, static_cast<const char *>(x) + (base + min(i, to - N)) * (16 / N), 16);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int at = min(from + j, to - 1);
          if constexpr (DT == kFloat)
            r[j] = static_cast<const unsigned *>(x)[base + at];
          else
            r[j / 2] |= (unsigned)static_cast<const uint16_t *>(x)[base + at] << (j % 2 * 16);
        }
      }
      return r;
    };
    int i = from + (int)threadIdx.x * N;
    int left = (to - (from + (int)(threadIdx.x & ~63u) * N) + step - 1) / step;  // of the wave
    if (to <= from || left <= 0) return;
    v4u now[U], next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = get(i + u * step);
#pragma unroll 1
    for (; left > 0; left -= U) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = get(i + (U + u) * step);
#pragma unroll
      for (int u = 0; u < U; ++u, i += step) {
        if (u < left) {
          float v[N];
#pragma unroll
          for (int j = 0; j < N; ++j) {
            if constexpr (DT == kFloat)
              v[j] = __builtin_bit_cast(float, (unsigned)now[u][j]);
            else
              v[j] = DT == kFloat16 ? F16ToF32((uint16_t)(now[u][j / 2] >> (j % 2 * 16))) : Bf16ToF32((uint16_t)(now[u][j / 2] >> (j % 2 * 16)));
          }
          const int at = whole ? min(i, to - N) : from;
          if (at != i || !whole || infinite) {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = at + j >= i && at + j < to ? As(v[j]) : -__builtin_huge_valf();
          }
          f(v, at, i);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = next[u];
    }
  }
};

// What a row asks for, and which token that is where nothing has to be weighed: the first
// in order, -1 of none.
struct Wish {
  float T, top_p, min_p;
  int64_t k;
  bool cuts;  // top_p does
};
__device__ __forceinline__ Wish WishOf(const SampleParams &p, int64_t row) {
  Wish w;
  w.T = p.temperature ? p.temperature[row] : 1.f;
  w.top_p = p.top_p ? p.top_p[row] : 1.f;
  w.min_p = p.min_p ? p.min_p[row] : 0.f;
  w.k = 0;
  if (p.top_k) w.k = p.k64 ? static_cast<const int64_t *>(p.top_k)[row] : (int64_t) static_cast<const int32_t *>(p.top_k)[row];
  if (w.k < 0 || w.k >= p.vocab) w.k = 0;
  w.cuts = w.top_p < 1.f;
  return w;
}
__device__ __forceinline__ void Answer(const SampleParams &p, int64_t row, int64_t token, float probability) {
  if (p.token64)
    static_cast<int64_t *>(p.token)[row] = token;
  else
    static_cast<int32_t *>(p.token)[row] = (int32_t)token;
  if (p.probability) p.probability[row] = probability;
}
// `best`: the largest key, and the complement of the lowest index that has it
__device__ __forceinline__ bool Plain(const Wish &w, u64 best) { return best >> 32 == 0 || !(w.T > 0.f) || w.k == 1; }
__device__ __forceinline__ void AnswerPlain(const SampleParams &p, int64_t row, u64 best) {
  const bool none = best >> 32 == 0;
  Answer(p, row, none ? -1 : (int64_t)(0xffffffffu - (unsigned)best), none ? 0.f : 1.f);
}
// floor(f n) of f from 0 to 1, which is m 2^-shift with m of 24 bits, and a sum n below 2^63;
// `rest`: whether that leaves anything.  In whole numbers: the product has 87 bits.
__device__ __forceinline__ u64 ShareOf(float f, u64 n, bool &rest) {
  const unsigned u = __builtin_bit_cast(unsigned, f), e = max(u >> 23, 1u);
  const u64 m = u < 0x800000u ? u : (u & 0x7fffffu) | 0x800000u;
  const u64 hi = __umul64hi(m, n), lo = m * n;
  const unsigned shift = 150 - e;  // 23 and more
  if (shift < 64) {
    rest = lo << (64 - shift) != 0;
    return hi << (64 - shift) | lo >> shift;
  }
  const unsigned s = min(shift - 64, 63u);  // hi has 23 bits
  rest = lo != 0 || (hi & ((u64(1) << s) - 1)) != 0;
  return hi >> s;
}
// The token at which the weights up to it reach this is the last that top_p keeps.
__device__ __forceinline__ u64 WantOf(float top_p, u64 total) {
  bool rest;
  const u64 w = ShareOf(fmaxf(top_p, 0.f), total, rest) + rest;
  return w ? w : 1;
}

// ---- the steps -------------------------------------------------------------------

// The values are made where they stand, not where they are used: one after the other,
// behind a branch each, they wait for themselves.
template <int N> __device__ __forceinline__ void Made(u64 (&w)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+v"(w[j]));
}

__device__ __forceinline__ void MakePowers(Shared &s) {
  if (threadIdx.x < 64) s.power[threadIdx.x] = exp2((int)threadIdx.x / -64.0);
}

// Of the workgroup; `own` of the thread.
template <int DT> __device__ __forceinline__ u64 Best(Shared &s, const Row<DT> &r, int from, int to, u64 &own) {
  float top = -__builtin_huge_valf();
  int at = 0;
  r.Each(from, to, [&](const auto &v, int first, int) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < r.N; ++j) {
      at = v[j] > top ? first + j : at;
      top = fmaxf(top, v[j]);
    }
  });
  own = IsLogit(top) ? (u64)KeyOf(top) << 32 | (0xffffffffu - (unsigned)at) : 0;
  return GroupMax(s, own);
}

__device__ __forceinline__ void Clear(Shared &s) {
  const int tid = threadIdx.x;
  s.bin[2 * tid] = s.bin[2 * tid + 1] = 0;
  s.chunk[tid] = 0;
  if (tid == 0) s.n = 0;
  __syncthreads();
}

// The largest number of 16 bits that at least `want` of the threads' are not below, 0 if there
// are not so many.
__device__ __forceinline__ unsigned KthOf(Shared &s, unsigned mine, unsigned want) {
  unsigned found = 0;
#pragma unroll 1
  for (int bit = 15; bit >= 0; --bit) {
    const unsigned at = found | 1u << bit;
    const u64 vote = __ballot(mine >= at);
    if (threadIdx.x % 64 == 0) s.votes[bit & 1][threadIdx.x / 64] = (unsigned)__popcll(vote);
    __syncthreads();
    unsigned sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += s.votes[bit & 1][w];
    if (sum >= want) found = at;
  }
  return found;
}

// Where the border is.  The tokens from `sure` on are kept for certain; those below it from
// `listed` on are listed, and the border is among them (NaN: there are none).
struct Place {
  float sure, listed;
  bool by_bits;     // the border is not known but to be somewhere
  unsigned k;       // of top_k, 0 where it leaves nothing out
  u64 above, want;  // top_p's: weights of what is kept for certain, and up to the border
};
constexpr float kNever = __builtin_nanf("");
__device__ __forceinline__ Place KeepAll() { return Place{-kMaxFloat, kNever, false, 0, 0, 0}; }
__device__ __forceinline__ Place ListFrom(float v, unsigned k) { return Place{kNever, v, false, k, 0, 0}; }

// The bin up to which bins add up to `want`; `above` what is in those before, `in` in it.
__device__ __forceinline__ int BinOf(Shared &s, u64 upto, u64 a, u64 b, u64 want, u64 &above, u64 &in) {
  const int tid = threadIdx.x;
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
}
template <int DT> __device__ __forceinline__ float FirstOfBin(const Row<DT> &r, int bin) {
  return bin < 0 ? kNever : r.FirstLogit([&](float v) { return r.Bin(v) <= bin; });
}

// From the largest keys of groups of tokens, one a thread: where the k-th of those stands,
// at least k tokens do, and hardly more while k is well below the number of groups.
constexpr int kFew = 512;
__device__ __forceinline__ Place PlaceOfLargest(Shared &s, const Wish &w, u64 own) {
  const unsigned key = KthOf(s, (unsigned)(own >> 48), (unsigned)w.k) << 16;
  if (key == 0) return ListFrom(kNever, 0);
  return ListFrom(LogitOf(max(key, KeyOf(-kMaxFloat))), (unsigned)w.k);  // smaller keys are no logits
}

// The border of top_k by counts in bins; KeepAll where it leaves nothing out, so that top_p
// has to find its border by itself.
template <int DT> __device__ __forceinline__ Place PlaceOfCounts(Shared &s, const Row<DT> &r, const Wish &w) {
  r.Each(0, r.vocab, [&](const auto &v, int, int) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < r.N; ++j)
      if (IsLogit(v[j])) atomicAdd(&s.bin[r.Bin(v[j])], 1ull);
  });
  __syncthreads();
  const u64 a = s.bin[2 * threadIdx.x], b = s.bin[2 * threadIdx.x + 1];
  u64 all, above, in;
  const u64 upto = GroupScan(s, a + b, all);
  if (all <= (u64)w.k) return KeepAll();
  const int bin = BinOf(s, upto, a, b, (u64)w.k, above, in);
  Place q = ListFrom(kNever, (unsigned)w.k);
  if (above + in > kList)
    q.by_bits = true;
  else
    q.listed = FirstOfBin(r, bin);
  return q;
}

// N logits of each thread from all over the row say how far down the border of top_p may
// be: half of what it leaves out goes without bins.  The first logit of the rest; bins are
// clear before.
template <int DT> __device__ __forceinline__ float BinsFrom(Shared &s, const Row<DT> &r, const Wish &w) {
  const int tid = threadIdx.x;
  float v[Row<DT>::N];
  r.Get((int)((int64_t)tid * (r.vocab - r.N) / (kThreads - 1)), v);
#pragma unroll
  for (int j = 0; j < r.N; ++j) {
    const float x = r.As(v[j]);
    // the first tokens may have most of the weight, and chance whether they are in the
    // sample: without them the border is no higher
    if (IsLogit(x) && r.Bin(x) >= kBins / 8) atomicAdd(&s.bin[r.Bin(x)], r.Whole(x));
  }
  __syncthreads();
  u64 all, above, in;
  const u64 a = s.bin[2 * tid], b = s.bin[2 * tid + 1], upto = GroupScan(s, a + b, all);
  if (!all) return -kMaxFloat;
  const float from = FirstOfBin(r, BinOf(s, upto, a, b, WantOf(0.5f + 0.5f * fmaxf(w.top_p, 0.f), all), above, in));
  __syncthreads();
  return from;
}
// Weights of the tokens from..to - 1 in bins, of those that are at least `least`, there for
// every thread when it returns; the sum of this thread's, all of them.
template <int DT> __device__ __forceinline__ u64 FillBins(Shared &s, const Row<DT> &r, float least, int from, int to) {
  u64 sum = 0;
  r.Each(from, to, [&](const auto &x, int, int) __attribute__((always_inline)) {
    u64 e[Row<DT>::N];
    r.Weights(x, r.floor, e);
    Made(e);
#pragma unroll
    for (int j = 0; j < r.N; ++j) {
      sum += e[j];
      if (x[j] >= least) atomicAdd(&s.bin[r.Bin(x[j])], e[j]);
    }
  });
  __syncthreads();
  return sum;
}
// The border of top_p from bins, or from sums of `width` of them that stand in the last; by_bits
// where they do not reach it.
template <int DT> __device__ __forceinline__ Place PlaceOfWeights(Shared &s, const Row<DT> &r, const Wish &w, u64 total, int width) {
  const u64 a = s.bin[2 * threadIdx.x], b = s.bin[2 * threadIdx.x + 1];
  u64 all, in;
  const u64 upto = GroupScan(s, a + b, all);
  Place q{kNever, kNever, false, 0, 0, WantOf(w.top_p, total)};
  if (all < q.want) {
    q.by_bits = true;
    return q;
  }
  const int bin = BinOf(s, upto, a, b, q.want, q.above, in);
  q.sure = FirstOfBin(r, bin - width);
  q.listed = FirstOfBin(r, bin);
  return q;
}

// Voting lanes before this one.
__device__ __forceinline__ int Before(u64 vote) {
  return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(vote >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)vote, 0));
}

// Lists what is to be listed, and adds what is kept for certain to its chunks.
template <int DT> __device__ __forceinline__ void Take(Shared &s, const Row<DT> &r, const Place &q, int from, int to) {
  const int lane = threadIdx.x % 64;
  if (!(q.listed == q.listed)) {  // nothing is listed
    if (q.sure == q.sure)
      r.Each(from, to, [&](const auto &v, int, int i) __attribute__((always_inline)) {
        u64 w[Row<DT>::N], sum = 0;
        r.Weights(v, r.least, w);
#pragma unroll
        for (int j = 0; j < r.N; ++j) sum += w[j];
        r.AddToChunk(s.chunk, i, sum);
      });
    __syncthreads();
    return;
  }
  // Few of a wave's tokens are kept: they wait in a queue until there is one for each lane.
  u64 *queue = s.queue[threadIdx.x / 64];
  int queued = 0;
  auto weigh = [&](int count) __attribute__((always_inline)) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const u64 e = queue[lane], more = queue[64 + lane];
    if (lane < count) {
      const u64 kept = r.Kept(__builtin_bit_cast(float, (unsigned)(e >> 32)));
      if (kept) atomicAdd(&s.chunk[(unsigned)e >> r.shift], kept);
    }
    queue[lane] = more;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  // (with a table of weights there is nothing to wait for)
  constexpr bool kTable = DT == kBfloat16;
  const float first_sure = fmaxf(q.sure, r.least);
  r.Each(from, to, [&](const auto &v, int first, int i) __attribute__((always_inline)) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < r.N; ++j) any |= v[j] >= q.listed;
    if (!__ballot(any)) return;
    if (kTable && q.sure == q.sure) {
      u64 w[Row<DT>::N], sum = 0;
      r.Weights(v, first_sure, w);
#pragma unroll
      for (int j = 0; j < r.N; ++j) sum += w[j];
      r.AddToChunk(s.chunk, i, sum);
    }
#pragma unroll
    for (int j = 0; j < r.N; ++j) {
      const bool sure = v[j] >= q.sure, mine = !sure && v[j] >= q.listed;
      const u64 vote = __ballot(mine), kept = kTable ? 0 : __ballot(sure);
      if (vote) {
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(&s.n, (unsigned)__popcll(vote));
        at = __builtin_amdgcn_readfirstlane(at) + Before(vote);
        if (mine && at < kList) s.list[at] = (u64)KeyOf(v[j]) << 32 | (unsigned)(first + j);
      }
      if (kept) {
        const int at = queued + Before(kept);
        if (sure) queue[at] = (u64)__builtin_bit_cast(unsigned, v[j]) << 32 | (unsigned)(first + j);
        queued += __popcll(kept);
        if (queued >= 64) {
          weigh(64);
          queued -= 64;
        }
      }
    }
  });
  if (queued) weigh(queued);
  __syncthreads();
}

// The number at which units, counted from the largest numbers down, reach `want` (the
// smallest number, where they do not); `above` and `in`: the units of larger ones and of
// it.  visit(f) calls f(number, unit) for the workgroup's numbers, from lo to hi.
template <typename V>
__device__ __forceinline__ unsigned Border(Shared &s, unsigned lo, unsigned hi, u64 want, u64 &above, u64 &in, V &&visit) {
  const int bits = hi > lo ? 32 - __builtin_clz(hi - lo) : 0;
  unsigned prefix = 0;  // of the number less lo
  above = in = 0;
#pragma unroll 1
  for (int shift = bits > 8 ? (bits - 1) / 8 * 8 : 0; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) s.digit[threadIdx.x] = 0;
    __syncthreads();
    visit([&](unsigned number, u64 unit) __attribute__((always_inline)) {
      number -= lo;
      if (shift == 24 || number >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s.digit[number >> shift & 255], unit);
    });
    __syncthreads();
    if (threadIdx.x < 64) {
      // four digits a lane, the largest first
      const int lane = threadIdx.x;
      u64 d[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += d[j] = s.digit[255 - 4 * lane - j];
      const u64 upto = WaveScan(sum), reach = __ballot(above + upto >= want);
      if (lane == (reach ? __builtin_ctzll(reach) : 63)) {
        u64 a = above + upto - sum, one = d[0];
        int j = 0;
#pragma unroll
        for (int t = 0; t < 3; ++t)
          if (j == t && a + one < want) a += one, one = d[t + 1], j = t + 1;
        s.out[0] = a;
        s.out[1] = one;
        s.at = 255 - 4 * lane - j;
      }
    }
    __syncthreads();
    above = s.out[0];
    in = s.out[1];
    prefix |= s.at << shift;
  }
  return lo + prefix;
}

// Kept are the tokens with a larger key, and of those with this key the ones up to an
// index.
struct Edge {
  unsigned key, last;
};

// Sorts x of the threads, number E tid + e, the largest first: bitonic, by registers, lanes
// and LDS as the distance grows.
template <int E> __device__ __forceinline__ void SortDown(Shared &s, u64 (&x)[E], int n) {
  const int tid = threadIdx.x;
  u64 *buffer = s.list;
#pragma unroll 1
  for (int k = 2; k <= n; k <<= 1) {
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      // waves without numbers only come to the barriers
      if (j < 64 * E && (int)(threadIdx.x & ~63u) * E >= n) continue;
      u64 y[E];
      if (j >= 64 * E) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) buffer[e * kThreads + tid] = x[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = buffer[e * kThreads + (tid ^ (j / E))];
      } else if (j >= E) {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = __shfl_xor(x[e], j / E);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = j == 1 ? x[e ^ (E > 1 ? 1 : 0)] : x[e ^ (E > 2 ? 2 : 0)];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = E * tid + e;
        const bool larger = ((i & k) == 0) == ((i & j) == 0);  // this one keeps the larger
        x[e] = (x[e] > y[e]) == larger ? x[e] : y[e];
      }
    }
  }
}

// The border among what is listed, of top_k, then of top_p; adds what of it is kept to its
// chunks.
template <int DT, int E> __device__ __forceinline__ Edge ByOrder(Shared &s, const Row<DT> &r, const Wish &w, const Place &q, unsigned n) {
  int size = 64;
  while (size < (int)n) size *= 2;
  u64 x[E], weight[E], sum = 0, all;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    // the lower index is the larger number
    const unsigned i = E * threadIdx.x + e;
    x[e] = i < n ? s.list[i] ^ 0xffffffffull : 0;
  }
  SortDown<E>(s, x, size);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned i = E * threadIdx.x + e;
    weight[e] = x[e] && (q.k == 0 || i < q.k) ? r.Whole(LogitOf((unsigned)(x[e] >> 32))) : 0;
    sum += weight[e];
  }
  u64 before = GroupScan(s, sum, all) - sum;
  const u64 want = !w.cuts ? ~u64(0) : q.want ? q.want - q.above : WantOf(w.top_p, all);
  if (threadIdx.x == 0) s.out[0] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned i = E * threadIdx.x + e;
    if (x[e] && (q.k == 0 || i < q.k) && before < want) {
      const float v = LogitOf((unsigned)(x[e] >> 32));
      const u64 kept = r.Kept(v);
      const unsigned at = ~(unsigned)x[e];
      if (kept) atomicAdd(&s.chunk[at >> r.shift], kept);
      // the last of those kept: the next one, if any, is not
      const u64 next = before + weight[e];
      if (i + 1 == n || (q.k && i + 1 == q.k) || next >= want) s.out[0] = x[e];
    }
    before += weight[e];
  }
  __syncthreads();
  return Edge{(unsigned)(s.out[0] >> 32), ~(unsigned)s.out[0]};
}

// The same by the bits of all the row's logits, with all that is kept.
template <int DT> __device__ __forceinline__ Edge ByBits(Shared &s, const Row<DT> &r, const Wish &w, const Place &q) {
  Edge e{0, ~0u};
  auto visit = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int i = threadIdx.x; i < r.vocab; i += kThreads) {
      const unsigned key = KeyOf(r.At(i));
      if (key) f(key, (unsigned)i);
    }
  };
  unsigned lo = 1;
  u64 over, in, ties = 0, equal = 0;
  if (q.k) {
    e.key = Border(s, lo, ~0u, q.k, over, in, [&](auto &&f) { visit([&](unsigned key, unsigned) { f(key, 1ull); }); });
    ties = q.k - over < in ? q.k - over : in;
    equal = in;
    lo = e.key;
  }
  if (w.cuts) {
    u64 want = q.want;
    if (!want) {
      // the sum of what top_k leaves
      u64 mine = 0, total;
      visit([&](unsigned key, unsigned) { mine += key > e.key ? r.Whole(LogitOf(key)) : 0; });
      GroupScan(s, mine, total);
      want = WantOf(w.top_p, total + ties * r.Whole(LogitOf(e.key)));
    }
    const unsigned b = Border(s, lo, ~0u, want, over, in, [&](auto &&f) {
      visit([&](unsigned key, unsigned) {
        if (key >= lo) f(key, r.Whole(LogitOf(key)));
      });
    });
    const u64 one = r.Whole(LogitOf(b)), left = want > over ? want - over : 0;
    const u64 m = one ? (left + one - 1) / one : 1;
    if (!q.k || b != e.key || m < ties) ties = m;
    equal = one ? in / one : ~u64(0);
    e.key = b;
  }
  if (ties < equal)
    e.last = ~Border(s, ~(unsigned)(r.vocab - 1), ~0u, ties, over, in, [&](auto &&f) {
      visit([&](unsigned key, unsigned i) {
        if (key == e.key) f(~i, 1ull);
      });
    });
  __syncthreads();
  s.chunk[threadIdx.x] = 0;
  __syncthreads();
  visit([&](unsigned key, unsigned i) {
    if (key > e.key || (key == e.key && i <= e.last)) {
      const u64 kept = r.Kept(LogitOf(key));
      if (kept) atomicAdd(&s.chunk[i >> r.shift], kept);
    }
  });
  __syncthreads();
  return e;
}

template <int DT> __device__ __forceinline__ Edge Resolve(Shared &s, const Row<DT> &r, const Wish &w, const Place &q) {
  if (q.listed != q.listed && !q.by_bits) return Edge{0, ~0u};  // all is kept
  const unsigned n = s.n;
  if (q.by_bits || n > kList) return ByBits(s, r, w, q);
  return n <= kThreads ? ByOrder<DT, 1>(s, r, w, q, n) : n <= 2 * kThreads ? ByOrder<DT, 2>(s, r, w, q, n) : ByOrder<DT, 4>(s, r, w, q, n);
}

// The chunk, then the token, at which the kept weights pass the share.
template <int DT> __device__ __forceinline__ void Choose(Shared &s, const Row<DT> &r, const SampleParams &p, int64_t row, const Edge &edge, float u) {
  u64 total;
  const u64 mine = s.chunk[threadIdx.x], upto = GroupScan(s, mine, total);
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  bool rest;
  const u64 share = ShareOf(u, total, rest);
  if (upto > share && upto - mine <= share) {
    s.at = threadIdx.x;
    s.out[0] = share - (upto - mine);
  }
  __syncthreads();
  const int size = 1 << r.shift, from = (int)s.at << r.shift;
  u64 left = s.out[0];
#pragma unroll 1
  for (int i0 = 0; i0 < size; i0 += kThreads) {
    const int i = from + i0 + (int)threadIdx.x;
    u64 kept = 0, sum;
    float v = 0.f;
    if (i0 + (int)threadIdx.x < size && i < r.vocab) {
      v = r.At(i);
      const unsigned key = KeyOf(v);
      if (key > edge.key || (key != 0 && key == edge.key && (unsigned)i <= edge.last)) kept = r.Kept(v);
    }
    const u64 incl = GroupScan(s, kept, sum);
    if (incl > left && incl - kept <= left) Answer(p, row, i, (float)(r.Weight(v, r.floor) / ((double)total * 0x1p-42)));
    if (sum > left) return;
    left -= sum;
  }
}

// ---- a workgroup a row --------------------------------------------------------------

template <int DT> __device__ __forceinline__ Row<DT> RowOf(const SampleParams &p, int64_t row, const Shared &s) {
  Row<DT> r{};
  r.x = p.x;
  r.base = row * p.vocab;
  r.vocab = p.vocab;
  // chunks of at least the tokens of a load
  r.shift = 3;
  while ((p.vocab - 1) >> r.shift >= kChunks) ++r.shift;
  r.power = s.power;
  return r;
}

template <int DT> __global__ __launch_bounds__(kThreads) void SampleRowKernel(const SampleParams p) {
  __shared__ Shared s;
  const int64_t row = p.first + blockIdx.x;
  const Wish w = WishOf(p, row);
  const float u = p.uniform[row];
  Row<DT> r = RowOf<DT>(p, row, s);
  MakePowers(s);
  Clear(s);
  u64 own;
  const u64 best = Best(s, r, 0, p.vocab, own);
  if (Plain(w, best)) {
    if (threadIdx.x == 0) AnswerPlain(p, row, best);
    return;
  }
  r.Weigh((unsigned)(best >> 32), w.T, w.min_p);
  Place q = KeepAll();
  bool taken = false, weights = w.k == 0 && w.cuts;
  if (w.k > 0) {
    if (w.k <= kFew && !r.infinite) q = PlaceOfLargest(s, w, own);
    if (q.k) {
      Take(s, r, q, 0, p.vocab);
      taken = s.n <= kList;
      __syncthreads();
      if (!taken) Clear(s);
    }
    if (!taken) {
      q = PlaceOfCounts(s, r, w);
      weights = w.cuts && q.k == 0;
      __syncthreads();
      if (weights) Clear(s);
    }
  }
  if (weights || q.sure == q.sure) r.MakeCodes(s.code);
  if (weights) {
    // (a short row's sample would be as much work as its bins)
    float from = p.vocab > 16 * kThreads ? BinsFrom(s, r, w) : -kMaxFloat;
    for (;;) {
      Clear(s);
      u64 total;
      const u64 mine = FillBins(s, r, from, 0, p.vocab);
      GroupScan(s, mine, total);
      q = PlaceOfWeights(s, r, w, total, 1);
      if (!q.by_bits || from == -kMaxFloat) break;
      from = -kMaxFloat;  // all of it
      __syncthreads();
    }
  }
  if (!taken) Take(s, r, q, 0, p.vocab);
  const Edge e = Resolve(s, r, w, q);
  Choose(s, r, p, row, e, u);
}

// ---- several workgroups a row ---------------------------------------------------------

// What the launches of a row leave for each other.
constexpr int kSlices = 16, kWidth = 2, kJoined = kBins / kWidth;  // most workgroups; bins in one between them
struct RowState {
  u64 best;
  float from;    // bins start here
  int weights;   // top_p's border is to be found from bins
  Place q;
  float least;   // min_p's first logit
  u64 group[kThreads];  // largest keys of the waves' tokens
  u64 chunk[kChunks];
  u64 list[kList];
  u64 total[kSlices];         // weights
  u64 bin[kSlices][kJoined];
};
// Zero between calls: workgroups of a step that are done, and what is listed.
struct RowCounters {
  unsigned done[3], n;
};
constexpr int kWords = (int)(sizeof(RowCounters) / sizeof(unsigned));

// Past this XCD's caches, for a workgroup of the same launch on another one.
template <typename T> __device__ __forceinline__ void Leave(T *at, T v) {
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T> __device__ __forceinline__ T Fetch(const T *at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of its row's in this launch; what the others left is
// there then.
__device__ __forceinline__ bool Last(Shared &s, unsigned *done, int slices) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) s.last = atomicAdd(done, 1u) == (unsigned)slices - 1;
  __syncthreads();
  if (s.last && threadIdx.x == 0) *done = 0;
  return s.last;
}

struct SplitArgs {
  SampleParams p;
  RowState *state;
  RowCounters *counters;
  int slices, slice;  // workgroups of a row, tokens of each: whole chunks
};
template <int DT> struct Split {
  int64_t row;
  int number, from, to;
  RowState *state;
  RowCounters *count;
  __device__ __forceinline__ explicit Split(const SplitArgs &a) {
    const int i = blockIdx.x / a.slices;
    number = blockIdx.x % a.slices;
    row = a.p.first + i;
    from = number * a.slice;
    to = min(from + a.slice, a.p.vocab);
    state = a.state + i;
    count = a.counters + i;
  }
};
// The largest logit, and where to begin.
template <int DT> __global__ __launch_bounds__(kThreads) void SampleTopKernel(const SplitArgs a) {
  __shared__ Shared s;
  const Split<DT> t(a);
  const SampleParams &p = a.p;
  const Wish w = WishOf(p, t.row);
  Row<DT> r = RowOf<DT>(p, t.row, s);
  u64 own;
  Best(s, r, t.from, t.to, own);
  for (int o = 32; o > 0; o >>= 1) {
    const u64 v = __shfl_xor(own, o);
    own = v > own ? v : own;
  }
  if (threadIdx.x % 64 == 0) Leave(&t.state->group[t.number * kWaves + threadIdx.x / 64], own);
  if (!Last(s, &t.count->done[0], a.slices)) return;
  MakePowers(s);
  Clear(s);
  own = (int)threadIdx.x < a.slices * kWaves ? Fetch(&t.state->group[threadIdx.x]) : 0;
  const u64 best = GroupMax(s, own);
  Place q = KeepAll();
  int weights = 0;
  float from = -kMaxFloat;
  if (!Plain(w, best)) {
    r.Weigh((unsigned)(best >> 32), w.T, w.min_p);
    weights = w.k == 0 && w.cuts;
    if (w.k > 0) {
      if (w.k <= kFew && !r.infinite) q = PlaceOfLargest(s, w, own);
      if (!q.k) {
        q = PlaceOfCounts(s, r, w);
        weights = w.cuts && q.k == 0;
        __syncthreads();
        if (weights) Clear(s);
      }
    }
    if (weights) from = BinsFrom(s, r, w);
  }
  if (threadIdx.x == 0) {
    t.state->best = best;
    t.state->from = from;
    t.state->weights = weights;
    t.state->q = q;
    t.state->least = r.least;
  }
}

template <int DT> __device__ __forceinline__ Row<DT> RowAgain(const SplitArgs &a, const Split<DT> &t, const Wish &w, Shared &s, bool codes) {
  Row<DT> r = RowOf<DT>(a.p, t.row, s);
  r.Weigh((unsigned)(t.state->best >> 32), w.T, 0.f);
  r.least = t.state->least;
  MakePowers(s);
  Clear(s);
  if (codes) r.MakeCodes(s.code);
  return r;
}

// top_p's border.
template <int DT> __global__ __launch_bounds__(kThreads) void SampleBinsKernel(const SplitArgs a) {
  __shared__ Shared s;
  const Split<DT> t(a);
  if (!t.state->weights) return;
  const Wish w = WishOf(a.p, t.row);
  const Row<DT> r = RowAgain(a, t, w, s, true);
  u64 total;
  const u64 mine = FillBins(s, r, t.state->from, t.from, t.to);
  GroupScan(s, mine, total);
  // (stores and loads: an addition to memory that all XCDs see costs 0.4 ns of the chip)
  static_assert(kJoined == kThreads && kWidth == 2, "a sum a thread");
  Leave(&t.state->bin[t.number][threadIdx.x], s.bin[2 * threadIdx.x] + s.bin[2 * threadIdx.x + 1]);
  if (threadIdx.x == 0) Leave(&t.state->total[t.number], total);
  if (!Last(s, &t.count->done[1], a.slices)) return;
  u64 joined = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSlices; ++i) {
    if (i >= a.slices) break;
    joined += Fetch(&t.state->bin[i][threadIdx.x]);
    total += Fetch(&t.state->total[i]);
  }
  s.bin[2 * threadIdx.x] = 0;
  s.bin[2 * threadIdx.x + 1] = joined;
  __syncthreads();
  Place q = PlaceOfWeights(s, r, w, total, kWidth);
  if (q.by_bits) {  // the sample was none for this row: bins of all of it
    __syncthreads();
    Clear(s);
    FillBins(s, r, -kMaxFloat, 0, a.p.vocab);
    q = PlaceOfWeights(s, r, w, total, 1);
  }
  if (threadIdx.x == 0) t.state->q = q;
}

// The list, the chunks, and the token.
template <int DT> __global__ __launch_bounds__(kThreads) void SampleTakeKernel(const SplitArgs a) {
  __shared__ Shared s;
  const Split<DT> t(a);
  const SampleParams &p = a.p;
  const Wish w = WishOf(p, t.row);
  if (Plain(w, t.state->best)) {
    if (t.number == 0 && threadIdx.x == 0) AnswerPlain(p, t.row, t.state->best);
    return;
  }
  const Place q = t.state->q;
  const Row<DT> r = RowAgain(a, t, w, s, q.sure == q.sure);
  Take(s, r, q, t.from, t.to);
  // whole chunks are this slice's alone
  const int first = t.from >> r.shift, chunks = (t.to - t.from + (1 << r.shift) - 1) >> r.shift;
  if ((int)threadIdx.x < chunks) Leave(&t.state->chunk[first + threadIdx.x], s.chunk[first + threadIdx.x]);
  const unsigned n = s.n;
  if (threadIdx.x == 0) s.at = n ? atomicAdd(&t.count->n, n) : 0;
  __syncthreads();
  for (unsigned i = threadIdx.x; i < n && i < kList && s.at + i < kList; i += kThreads) Leave(&t.state->list[s.at + i], s.list[i]);
  if (!Last(s, &t.count->done[2], a.slices)) return;
  const unsigned all = Fetch(&t.count->n);
  s.chunk[threadIdx.x] = (int64_t)threadIdx.x << r.shift < p.vocab ? Fetch(&t.state->chunk[threadIdx.x]) : 0;
  for (unsigned i = threadIdx.x; i < all && i < kList; i += kThreads) s.list[i] = Fetch(&t.state->list[i]);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.n = all;
    t.count->n = 0;
  }
  __syncthreads();
  const Edge e = Resolve(s, r, w, q);
  Choose(s, r, p, t.row, e, p.uniform[t.row]);
}

// Workgroups of a row.  us, one | several, bfloat16, by vocabulary and rows:
//                       40000         131072        200000
//   top_p     1 row     41 | 44       78 | 52       108 | 56
//            16 rows    45 | 48       85 | 59       116 | 67
//            32 rows    45 | 69       84 | 101      117 | 115
//   top_k 50  1 row     22 | 26       31 | 27       39 | 27   (fp32)
//            16 rows    24 | 28       33 | 29       42 | 31
//  and by 66000, 131072, 200000:
//   top_k 300 1 row     35 | 41       44 | 47       51 | 54
//            16 rows    36 | 44       45 | 50       55 | 58
//   top_k 513 1 row     44 | 39       60 | 46       75 | 53
//            16 rows    46 | 42       61 | 49       79 | 57
// (Shared rows have 256 groups, so a top_k of more is counted over the row by its last workgroup, where one
// workgroup has 1024: from 257 to 512 sharing loses up to 20 %.  top_k is on the device, and the rule cannot
// look at it.)
int SlicesOf(const SampleParams &p) { return p.vocab >= 65536 && p.rows <= 16 ? kSlices : 1; }

template <int DT> void LaunchSample(SampleParams p, void *scratch, hipStream_t stream) {
  const int slices = SlicesOf(p);
  if (slices == 1) {
    LaunchInPieces(p.rows, kThreads, [&](int64_t first, unsigned count) {
      p.first = first;
      SampleRowKernel<DT><<<count, kThreads, 0, stream>>>(p);
    });
    return;
  }
  int shift = 3;
  while ((p.vocab - 1) >> shift >= kChunks) ++shift;
  SplitArgs a{p, static_cast<RowState *>(scratch), reinterpret_cast<RowCounters *>(Ctx().ws.Counters((size_t)p.rows * kWords)), 0, 0};
  a.slice = ((p.vocab + slices - 1) / slices + (1 << shift) - 1) >> shift << shift;
  a.slices = (p.vocab + a.slice - 1) / a.slice;
  const unsigned grid = (unsigned)(p.rows * a.slices);
  SampleTopKernel<DT><<<grid, kThreads, 0, stream>>>(a);
  if (p.top_p) SampleBinsKernel<DT><<<grid, kThreads, 0, stream>>>(a);
  SampleTakeKernel<DT><<<grid, kThreads, 0, stream>>>(a);
}

}  // namespace

size_t SampleScratchBytes(const SampleParams &p) { return SlicesOf(p) > 1 ? (size_t)p.rows * sizeof(RowState) : 0; }

void LaunchSampleTokens(const SampleParams &p, void *scratch, hipStream_t stream) {
  if (p.dtype == kFloat)
    LaunchSample<kFloat>(p, scratch, stream);
  else if (p.dtype == kFloat16)
    LaunchSample<kFloat16>(p, scratch, stream);
  else
    LaunchSample<kBfloat16>(p, scratch, stream);
}

}  // namespace onnxl_amd
