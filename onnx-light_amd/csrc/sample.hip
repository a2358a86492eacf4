// A token from each row of logits and a given random number: temperature, top-k,
// top-p and min-p, then the first token, in order of index, at which the kept
// weights add up to more than the random number's share of their sum.
//
// A weight exp((x - max) / T) is a whole number of 2^-42: sums of them have no
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
#include <type_traits>

#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"

namespace onnxl_amd {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048, kList = 4096, kChunks = 1024;
constexpr float kOctaves = 44.f;  // of weights that the bins span; the last bin has the rest
constexpr float kMaxFloat = 0x1.fffffep127f, kMinFloat = 0x1p-126f;
typedef unsigned long long u64;

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
  double power[32];  // 2^(-j / 32)
  u64 wave[kWaves];
  u64 digit[256];
  u64 chunk[kChunks];
  u64 bin[kBins];
  u64 list[kList];         // key << 32 | index
  u64 queue[kWaves][128];  // of a wave: logit << 32 | index, kept for certain
  u64 out[2];
  unsigned n, at;
};

// ---- sums over lanes and threads ----------------------------------------------

template <int CTRL, int ROWS> __device__ __forceinline__ u64 AddFrom(u64 v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((u64)hi << 32 | lo);
}
// Sums of the lanes up to and with this one: inside rows of 16, then the last lane of a
// row to the next row, of the second to the third and fourth.
__device__ __forceinline__ u64 WaveScan(u64 v) {
  v = AddFrom<0x111, 0xf>(v);
  v = AddFrom<0x112, 0xf>(v);
  v = AddFrom<0x114, 0xf>(v);
  v = AddFrom<0x118, 0xf>(v);
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
  const void *x;
  int64_t base;
  int vocab;
  int shift;       // log2 of a chunk's tokens
  // what weights go by, from the largest logit on
  float top, per_bin;
  double high, octaves;  // the largest logit (past all others where it is infinite); log2(e) / T
  double least;          // min_p, 0: none
  const double *power;

  __device__ __forceinline__ void Weigh(float largest, float T, float min_p) {
    top = fminf(largest, kMaxFloat);
    high = largest > kMaxFloat ? 0x1p1000 : (double)largest;
    octaves = largest > kMaxFloat ? 1.0 : 1.4426950408889634074 / (double)T;
    // any positive number keeps the order of the bins
    per_bin = fminf(fmaxf((float)(octaves * (kBins / kOctaves)), kMinFloat), kMaxFloat);
    least = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
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
  __device__ __forceinline__ float At(int i) const {
    float v[1];
    Load<1>(i, v);
    return v[0];
  }
  // 2^-t by a table of the 32nds, whose number stands in the low bits of a sum with 1.5
  // 2^47, and the series of the rest, at most 1/64, to about 2^-48.  A difference past
  // 1000 octaves counts as that, one of infinities as the largest logit itself.
  __device__ __forceinline__ double Weight(float v) const {
    const double t = fmax(fmin((high - (double)v) * octaves, 1000.0), 0.0);
    const double sum = t + 0x1.8p47, r = (sum - 0x1.8p47) - t;
    double p = fma(r, 0x1.5d87fe78a6731p-10, 0x1.3b2ab6fba4e77p-7);
    p = fma(p, r, 0x1.c6b08d704a0c0p-5);
    p = fma(p, r, 0x1.ebfbdff82c58fp-3);
    p = fma(p, r, 0x1.62e42fefa39efp-1);
    p = fma(p, r, 1.0);
    const unsigned k = (unsigned)__builtin_bit_cast(u64, sum);
    const u64 w = __builtin_bit_cast(u64, power[k & 31] * p);
    return __builtin_bit_cast(double, w - ((u64)(k >> 5) << 52));
  }
  // in units of 2^-42, the last place of numbers from 1024 to 2048
  __device__ static __forceinline__ u64 Whole(double w) {
    return __builtin_bit_cast(u64, w + 1024.0) - __builtin_bit_cast(u64, 1024.0);
  }
  // what min_p leaves of a token's weight
  __device__ __forceinline__ u64 Kept(float v) const {
    const double w = Weight(v);
    return Whole(w >= least ? w : 0.0);
  }
  // falls with v, as every rounding in it does; anything for a NaN
  __device__ __forceinline__ int Bin(float v) const {
    return (int)__builtin_amdgcn_fmed3f((top - v) * per_bin, 0.f, (float)(kBins - 1)) & (kBins - 1);
  }
  // f(logits, first index) for 16 bytes at a time of the tokens from..to - 1, four of them
  // on their way; what is past the end is -inf
  template <typename F> __device__ __forceinline__ void Each(int from, int to, F &&f) const {
    constexpr int N = DT == kFloat ? 4 : 8, U = 4;
    for (int i0 = from; i0 < to; i0 += U * N * kThreads) {
      float v[U][N];
      const int wave = i0 + (int)(threadIdx.x & ~63u) * N;  // the wave's first
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + (u * kThreads + (int)threadIdx.x) * N;
        if (i + N <= to) {
          Load<N>(i, v[u]);
        } else if (wave + u * kThreads * N < to) {
#pragma unroll
          for (int j = 0; j < N; ++j) v[u][j] = i + j < to ? At(i + j) : -__builtin_huge_valf();
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (wave + u * kThreads * N < to) f(v[u], i0 + (u * kThreads + (int)threadIdx.x) * N);
    }
  }
  // f(logit, index) for each that can be chosen, one after the other
  template <typename F> __device__ __forceinline__ void EachLogit(int from, int to, F &&f) const {
    Each(from, to, [&](const auto &v, int i) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < (int)(sizeof(v) / 4); ++j)
        if (IsLogit(v[j])) f(v[j], i + j);
    });
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
// The token at which the weights up to it reach this is the last that top_p keeps.
__device__ __forceinline__ u64 WantOf(float top_p, u64 total) {
  const u64 w = (u64)ceil((double)fmaxf(top_p, 0.f) * (double)total);
  return w ? w : 1;
}

// ---- the steps -------------------------------------------------------------------

// The values are made where they stand, not where they are used: one after the other,
// behind a branch each, they wait for themselves (a row of 131072 42 us in place of 16).
template <int N> __device__ __forceinline__ void Made(u64 (&w)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+v"(w[j]));
}

// Of the workgroup; `own` of the thread.
template <int DT> __device__ __forceinline__ u64 Best(Shared &s, const Row<DT> &r, int from, int to, u64 &own) {
  u64 best = 0;
  r.Each(from, to, [&](const auto &v, int i) __attribute__((always_inline)) {
    // the largest of the 16 bytes, and where it stands first
    constexpr int N = sizeof(v) / 4;
    float top = v[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < N; ++j)
      if (!(top >= v[j]) && v[j] == v[j]) top = v[j], at = j;
    const u64 k = (u64)KeyOf(top) << 32 | (0xffffffffu - (unsigned)(i + at));
    best = k > best ? k : best;
  });
  own = best;
  return GroupMax(s, best);
}

__device__ __forceinline__ void Clear(Shared &s) {
  const int tid = threadIdx.x;
  s.bin[2 * tid] = s.bin[2 * tid + 1] = 0;
  s.chunk[tid] = 0;
  if (tid < 32) s.power[tid] = exp2(-tid / 32.0);
  if (tid == 0) s.n = 0;
  __syncthreads();
}

// Counts, or weights, of the tokens in bins.
template <int DT, bool WEIGHTS> __device__ __forceinline__ void FillBins(Shared &s, const Row<DT> &r, int from, int to) {
  r.Each(from, to, [&](const auto &v, int) __attribute__((always_inline)) {
    constexpr int N = sizeof(v) / 4;
    u64 w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = WEIGHTS ? r.Whole(r.Weight(v[j])) : IsLogit(v[j]);
    Made(w);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (w[j]) atomicAdd(&s.bin[r.Bin(v[j])], w[j]);
  });
  __syncthreads();
}

// Where the border is.  If `sure`, the tokens in bins above the border's are kept for
// certain, and those of its bin are listed, if `listed`; else it is among the tokens of
// bins up to `bin` that are at least `least`, and those are listed.
struct Place {
  int bin;
  int sure, listed, by_bits;
  unsigned k;       // of top_k, 0 where it leaves nothing out
  u64 above, want;  // top_p's: weights of the bins above, and up to the border
  float least;
};

__device__ __forceinline__ Place KeepAll() { return Place{kBins, 1, 0, 0, 0, 0, 0, -__builtin_huge_valf()}; }
__device__ __forceinline__ Place ListAll(unsigned k) { return Place{kBins - 1, 0, 1, 0, k, 0, 0, -__builtin_huge_valf()}; }

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
// From bins of counts; `again`: top_k leaves nothing out and the list would not hold
// all, so that top_p needs bins of weights.
__device__ __forceinline__ Place PlaceOfCounts(Shared &s, const Wish &w, bool &again) {
  const u64 a = s.bin[2 * threadIdx.x], b = s.bin[2 * threadIdx.x + 1];
  u64 all, above, in;
  const u64 upto = GroupScan(s, a + b, all);
  again = false;
  if (all <= kList) return ListAll(all <= (u64)w.k ? 0 : (unsigned)w.k);
  if (all <= (u64)w.k) {
    again = w.cuts;
    return KeepAll();
  }
  const int bin = BinOf(s, upto, a, b, (u64)w.k, above, in);
  if (above + in > kList) return Place{0, 0, 0, 1, (unsigned)w.k, 0, 0, 0.f};
  return Place{bin, 0, 1, 0, (unsigned)w.k, 0, 0, -__builtin_huge_valf()};
}
__device__ __forceinline__ Place PlaceOfWeights(Shared &s, const Wish &w) {
  const u64 a = s.bin[2 * threadIdx.x], b = s.bin[2 * threadIdx.x + 1];
  u64 all, in;
  const u64 upto = GroupScan(s, a + b, all);
  Place q{0, 1, 1, 0, 0, 0, 0, 0.f};
  q.want = WantOf(w.top_p, all);
  q.bin = BinOf(s, upto, a, b, q.want, q.above, in);
  return q;
}

// Voting lanes before this one.
__device__ __forceinline__ int Before(u64 vote) {
  return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(vote >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)vote, 0));
}
__device__ __forceinline__ void List(Shared &s, u64 vote, bool mine, float v, int i) {
  unsigned at = 0;
  if (threadIdx.x % 64 == 0) at = atomicAdd(&s.n, (unsigned)__popcll(vote));
  at = __builtin_amdgcn_readfirstlane(at) + Before(vote);
  if (mine && at < kList) s.list[at] = (u64)KeyOf(v) << 32 | (unsigned)i;
}

// Lists what is to be listed, and adds what is kept for certain to its chunks.
template <int DT> __device__ __forceinline__ void Take(Shared &s, const Row<DT> &r, const Place &q, int from, int to) {
  const int lane = threadIdx.x % 64;
  if (!q.listed) {  // all of it is kept, or nothing known
    if (q.sure)
      r.Each(from, to, [&](const auto &v, int i) __attribute__((always_inline)) {
        // -inf and NaN weigh 2^-1000, which is 0 in whole units
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < (int)(sizeof(v) / 4); ++j) sum += r.Kept(v[j]);
        if (sum) atomicAdd(&s.chunk[i >> r.shift], sum);
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
  r.Each(from, to, [&](const auto &v, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(v) / 4); ++j) {
      const int b = r.Bin(v[j]);
      const bool is = IsLogit(v[j]);
      const bool mine = is && (q.sure ? b == q.bin : b <= q.bin && v[j] >= q.least), sure = is && q.sure && b < q.bin;
      const u64 vote = __ballot(mine), kept = __ballot(sure);
      if (vote) List(s, vote, mine, v[j], i + j);
      if (kept) {
        const int at = queued + Before(kept);
        if (sure) queue[at] = (u64)__builtin_bit_cast(unsigned, v[j]) << 32 | (unsigned)(i + j);
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
// LAST: the shift of the last digit looked at; with more than 0 the result is the
// smallest number with the digits before.
template <int LAST = 0, typename V>
__device__ unsigned Border(Shared &s, unsigned lo, unsigned hi, u64 want, u64 &above, u64 &in, V &&visit) {
  const int bits = hi > lo ? 32 - __builtin_clz(hi - lo) : 0;
  unsigned prefix = 0;  // of the number less lo
  above = in = 0;
  for (int shift = (bits + 7) / 8 * 8 - 8 < 0 ? 0 : (bits + 7) / 8 * 8 - 8; shift >= LAST; shift -= 8) {
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
        u64 a = above + upto - sum;
        int j = 0;
        for (; j < 3 && a + d[j] < want; ++j) a += d[j];
        s.out[0] = a;
        s.out[1] = d[j];
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

// From every thread's largest key: where the k-th of those stands, at least k tokens do,
// and hardly more while k is well below the number of threads.
constexpr int kFew = 512;
__device__ __forceinline__ bool PlaceOfLargest(Shared &s, const Wish &w, u64 best, u64 own, Place &q) {
  u64 above, in;
  const unsigned key = Border<16>(s, 1, (unsigned)(best >> 32), (u64)w.k, above, in, [&](auto &&f) {
    if (own >> 32) f((unsigned)(own >> 32), 1ull);
  });
  if (above + in < (u64)w.k) return false;
  q = ListAll((unsigned)w.k);
  q.least = LogitOf(max(key, KeyOf(-kMaxFloat)));  // smaller keys are no logits
  return true;
}

// Kept are the tokens with a larger key, and of those with this key the ones up to an
// index.
struct Edge {
  unsigned key, last;
};

// The border among tokens that visit(f) gives as f(key, weight, index), their keys from lo to
// hi: of top_k, then of top_p.
template <int DT, typename V>
__device__ __forceinline__ Edge EdgeOf(Shared &s, const Row<DT> &r, const Wish &w, const Place &q, unsigned lo, unsigned hi, V &&visit) {
  Edge e{0, 0};
  u64 over, in, ties = 0, equal = 0, want = q.want - q.above;
  if (q.k) {
    e.key = Border(s, lo, hi, q.k, over, in, [&](auto &&f) { visit([&](unsigned key, float, int) { f(key, 1ull); }); });
    ties = q.k - over < in ? q.k - over : in;  // fewer tokens than k may be there
    equal = in;
    lo = e.key;
  }
  if (w.cuts) {
    auto weights = [&](auto &&f) {
      visit([&](unsigned key, float v, int) {
        if (key >= e.key) f(key, r.Whole(r.Weight(v)));
      });
    };
    if (!q.want) {
      // the sum of what top_k leaves
      u64 mine = 0, total;
      weights([&](unsigned key, u64 one) { mine += key > e.key ? one : 0; });
      GroupScan(s, mine, total);
      want = WantOf(w.top_p, total + (e.key ? ties * r.Whole(r.Weight(LogitOf(e.key))) : 0));
    }
    const unsigned b = Border(s, lo, hi, want, over, in, weights);
    const u64 one = r.Whole(r.Weight(LogitOf(b))), left = want > over ? want - over : 0;
    const u64 n = one ? (left + one - 1) / one : 1;
    if (!q.k || b != e.key || n < ties) ties = n;
    equal = one ? in / one : ~u64(0);
    e.key = b;
  }
  e.last = ~0u;
  if (ties < equal)
    e.last = ~Border(s, ~(unsigned)(r.vocab - 1), ~0u, ties, over, in, [&](auto &&f) {
      visit([&](unsigned key, float, int i) {
        if (key == e.key) f(~(unsigned)i, 1ull);
      });
    });
  return e;
}

// The border, and the chunks' weights with what was listed.
template <int DT> __device__ __forceinline__ Edge Resolve(Shared &s, const Row<DT> &r, const Wish &w, const Place &q) {
  Edge edge{0, ~0u};
  const unsigned n = s.n;
  if (q.listed && n <= kList) {
    constexpr int E = kList / kThreads;
    u64 e[E];
    unsigned lo = ~0u, hi = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const unsigned i = j * kThreads + threadIdx.x;
      e[j] = i < n ? s.list[i] : 0;
      if (!e[j]) continue;
      lo = min(lo, (unsigned)(e[j] >> 32));
      hi = max(hi, (unsigned)(e[j] >> 32));
    }
    auto listed = [&](auto &&f) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (e[j]) f((unsigned)(e[j] >> 32), LogitOf((unsigned)(e[j] >> 32)), (int)(unsigned)e[j]);
    };
    if (q.k || w.cuts) {
      // the largest and the complement of the smallest, at once: neither is 0
      hi = (unsigned)(GroupMax(s, hi));
      lo = ~(unsigned)GroupMax(s, ~lo);
      edge = EdgeOf(s, r, w, q, lo, hi, listed);
    }
    listed([&](unsigned key, float v, int i) {
      if (key > edge.key || (key == edge.key && (unsigned)i <= edge.last)) {
        const u64 kept = r.Kept(v);
        if (kept) atomicAdd(&s.chunk[i >> r.shift], kept);
      }
    });
    __syncthreads();
  } else if (q.listed || q.by_bits) {
    auto logits = [&](auto &&f) { r.EachLogit(0, r.vocab, [&](float v, int i) { f(KeyOf(v), v, i); }); };
    Place whole = q;  // among all tokens
    whole.above = 0;
    edge = EdgeOf(s, r, w, whole, 1, ~0u, logits);
    __syncthreads();
    s.chunk[threadIdx.x] = 0;
    __syncthreads();
    logits([&](unsigned key, float v, int i) {
      if (key > edge.key || (key == edge.key && (unsigned)i <= edge.last)) {
        const u64 kept = r.Kept(v);
        if (kept) atomicAdd(&s.chunk[i >> r.shift], kept);
      }
    });
    __syncthreads();
  }
  return edge;
}

// The chunk, then the token, at which the kept weights pass the share.
template <int DT> __device__ __forceinline__ void Choose(Shared &s, const Row<DT> &r, const SampleParams &p, int64_t row, const Edge &edge) {
  u64 total;
  const u64 mine = s.chunk[threadIdx.x], upto = GroupScan(s, mine, total);
  float u = p.uniform[row];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  u64 share = (u64)((double)u * (double)total);
  if (share >= total) share = total - 1;
  if (upto > share && upto - mine <= share) {
    s.at = threadIdx.x;
    s.out[0] = share - (upto - mine);
  }
  __syncthreads();
  const int size = 1 << r.shift, from = (int)s.at << r.shift;
  u64 left = s.out[0];
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
    if (incl > left && incl - kept <= left) Answer(p, row, i, (float)(r.Weight(v) / ((double)total * 0x1p-42)));
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
  // chunks of at least the 8 tokens of a load
  r.shift = 3;
  while ((p.vocab - 1) >> r.shift >= kChunks) ++r.shift;
  r.power = s.power;
  return r;
}

template <int DT> __global__ __launch_bounds__(kThreads) void SampleRowKernel(const SampleParams p) {
  __shared__ Shared s;
  const int64_t row = p.first + blockIdx.x;
  const Wish w = WishOf(p, row);
  Row<DT> r = RowOf<DT>(p, row, s);
  Clear(s);
  u64 own;
  const u64 best = Best(s, r, 0, p.vocab, own);
  if (Plain(w, best)) {
    if (threadIdx.x == 0) AnswerPlain(p, row, best);
    return;
  }
  r.Weigh(LogitOf((unsigned)(best >> 32)), w.T, w.min_p);
  Place q = KeepAll();
  bool taken = false, weights = w.k == 0 && w.cuts;
  if (p.vocab <= kList && (w.k > 0 || w.cuts)) {
    q = ListAll((unsigned)w.k);
    weights = false;
  } else if (w.k > 0) {
    if (w.k <= kFew && PlaceOfLargest(s, w, best, own, q)) {
      Take(s, r, q, 0, p.vocab);
      taken = s.n <= kList;
      __syncthreads();
      if (!taken) Clear(s);
    }
    if (!taken) {
      FillBins<DT, false>(s, r, 0, p.vocab);
      q = PlaceOfCounts(s, w, weights);
      __syncthreads();
      if (weights) Clear(s);
    }
  }
  if (weights) {
    FillBins<DT, true>(s, r, 0, p.vocab);
    q = PlaceOfWeights(s, w);
  }
  if (!taken) Take(s, r, q, 0, p.vocab);
  Choose(s, r, p, row, Resolve(s, r, w, q));
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
