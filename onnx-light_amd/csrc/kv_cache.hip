// New keys and values into the paged 8-bit cache, one scale for each block of
// tokens and head.
//
// Bound by memory: the new tokens are read once (kept in registers between the
// block's maximum and its codes) and their codes written once.  A workgroup has
// one block of one sequence, one head, and k or v:
//   s' = max(scale of the tokens kept in the block, max|new| / qmax),
// the kept codes rounded again by s / s' where the scale grew, the new codes.
// Nothing else touches that block and head, so there are no atomics.  Values go
// through LDS, which turns 16 tokens of a dimension into one 16-byte store.
//
// The append of a joint projection's rows is the same kernel on the rows' keys, turned
// on the way and kept in fp32, and values; workgroups of their own before those turn the
// queries.  us, 32 + 2 x 8 heads of 128 in bfloat16: 64 sequences with a token each 4.9,
// as good as a launch; four prompts of 1500 to 4096 tokens, 256 MB read and written, 62
// (4.1 TB/s), against 66 with the queries last and 73 with a block's own queries in its
// workgroup.
#include <type_traits>

#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "quant8.hpp"
#include "rotary.hpp"

namespace onnxl_amd {
namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

// Four codes rounded again: code * ratio.
__device__ __forceinline__ unsigned Again4(unsigned w, float ratio, bool fp8) {
  if (fp8) {
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return Fp8Codes4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
  }
  return Int8Codes4((float)(int8_t)w * ratio, (float)(int8_t)(w >> 8) * ratio, (float)(int8_t)(w >> 16) * ratio,
                    (float)(int8_t)(w >> 24) * ratio);
}

// Blocks of sequence b with new tokens.
__device__ __forceinline__ int NewBlocks(const KvCacheParams &c, int b) {
  const int n = KvNewTokens(c, b);
  if (n <= 0) return 0;
  const int len = c.lengths[b];
  return ((len - 1) >> c.block_shift) - ((len - n) >> c.block_shift) + 1;
}

// The sequence and the block of it that ordinal `w` of the batch's new blocks is:
// every wave looks through 64 sequences at a time.
__device__ __forceinline__ bool FindBlock(const KvCacheParams &c, int64_t w, int &b, int &j) {
  const int lane = threadIdx.x % 64;
  for (int base = 0; base < c.batch; base += 64) {
    const int mine = base + lane < c.batch ? NewBlocks(c, base + lane) : 0;
    int64_t upto = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(upto, o);
      if (lane >= o) upto += v;
    }
    const uint64_t past = __ballot(w < upto);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = __builtin_amdgcn_readfirstlane(base + l);
      j = __builtin_amdgcn_readfirstlane((int)(w - __shfl(upto - mine, l)));
      return true;
    }
    w -= __shfl(upto, 63);
  }
  return false;
}

// Eight values of a row of the joint projection: of a key, turned to the row's
// position, or as they are.
struct Wide8 {
  float v[8];
};
template <int DT>
__device__ __forceinline__ Wide8 JointValues(const RotaryTable &t, const uint16_t *row, int d, bool turn, int64_t pos) {
  Wide8 r;
  Widen<DT, 8>(row, d, r.v);
  if (!turn || d >= 2 * t.half) return r;
  if (t.interleaved) {
    float c[4], s[4];
    TableValues<DT, 4>(t, pos, d / 2, c, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = r.v[2 * i], b = r.v[2 * i + 1];
      r.v[2 * i] = a * c[i] - b * s[i];
      r.v[2 * i + 1] = a * s[i] + b * c[i];
    }
    return r;
  }
  const bool upper = d >= t.half;
  float o[8], c[8], s[8];
  Widen<DT, 8>(row, upper ? d - t.half : d + t.half, o);
  TableValues<DT, 8>(t, pos, upper ? d - t.half : d, c, s);
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = upper ? o[i] * s[i] + r.v[i] * c[i] : r.v[i] * c[i] - o[i] * s[i];
  return r;
}

// Queries of the joint rows, by waves: a lane has 16 dimensions of a head, the wave as many
// heads at once as that makes.
template <int DT> __device__ __forceinline__ void RotateQueries(const RotaryAppendParams &p, int64_t wave, int64_t waves) {
  const KvCacheParams &c = p.a.c;
  const int lane = threadIdx.x % 64, D = c.head_dim, parts = D / 16, at_once = 64 / parts;
  const int units = (p.heads + at_once - 1) / at_once;  // of a token
  for (int64_t u = wave; u < c.tokens * units; u += waves) {
    const int64_t t = u / units;
    int b = -1;  // the first sequence that ends past the row
    for (int base = 0; base < c.batch && b < 0; base += 64) {
      const bool ends = base + lane < c.batch && c.start[base + lane + 1] > t;
      const uint64_t past = __ballot(ends);
      if (past) b = base + __builtin_ctzll(past);
    }
    if (b < 0 || c.start[b] > t || KvNewTokens(c, b) < 0) continue;
    const int first = (int)(u % units) * at_once + lane / parts;
    if (lane >= at_once * parts || first >= p.heads) continue;
    const int64_t pos = RotaryRow(p.t, t, (int64_t)c.lengths[b] - (c.start[b + 1] - t));
    const int64_t from = t * (p.heads + 2 * c.kv_heads) * (int64_t)D, to = t * p.heads * (int64_t)D;
    if (p.t.interleaved)
      RotateHeads<DT, 1, true>(p.t, p.a.k, from, D, p.q, to, D, first, 1, p.heads, D, lane % parts, pos, p.stream);
    else
      RotateHeads<DT, 1, false>(p.t, p.a.k, from, D, p.q, to, D, first, 1, p.heads, D, lane % parts, pos, p.stream);
  }
}

__device__ __forceinline__ const KvAppendParams &Append(const KvAppendParams &p) { return p; }
__device__ __forceinline__ const KvAppendParams &Append(const RotaryAppendParams &p) { return p.a; }

// NG groups of 8 values per thread are kept; KEPT: they are all there can be.
// JOINT: the rows of a joint projection, p.k, whose keys are rotated on the way.
template <int THREADS, int NG, bool KEPT, int JOINT = 0>
__global__ __launch_bounds__(THREADS) void KvAppendKernel(
    const std::conditional_t<JOINT != 0, RotaryAppendParams, KvAppendParams> all) {
  extern __shared__ __align__(16) uint8_t codes[];  // [token][dimension] of the new values
  __shared__ unsigned s_top[THREADS / 64];
  const KvAppendParams &p = Append(all);
  const KvCacheParams &c = p.c;
  const int tid = threadIdx.x, bt = c.block_tokens, D = c.head_dim, gd = D / 8;
  int head = blockIdx.y;
  bool is_v = blockIdx.z != 0;
  int64_t block = p.first + blockIdx.x;
  if constexpr (JOINT != 0) {
    // the queries' workgroups first: they are the most, and what the others wait for, their
    // block's maximum, is then waited for beside the last of them
    if (block < all.groups) {
      constexpr int W = THREADS / 64;
      RotateQueries<JOINT>(all, block * W + __builtin_amdgcn_readfirstlane(tid / 64), all.groups * W);
      return;
    }
    // (fewer than 2^32: the call checks it)
    const unsigned rest = (unsigned)(block - all.groups), blocks = (unsigned)all.blocks;
    block = rest % blocks;
    head = (int)(rest / blocks % (unsigned)c.kv_heads);
    is_v = rest / blocks >= (unsigned)c.kv_heads;
  }
  const bool fp8 = c.fp8;
  int b, w;
  if (!FindBlock(c, block, b, w)) return;
  const int len = c.lengths[b], start = c.start[b], first = len - (c.start[b + 1] - start);
  const int j = (first >> c.block_shift) + w;
  const int64_t blk = c.table[(int64_t)b * c.max_blocks + j];
  if (blk < 0 || blk >= c.num_blocks) return;
  const int lo = max(first - j * bt, 0), hi = min(len - j * bt, bt);  // tokens kept before lo, new from lo on
  const int groups = (hi - lo) * gd;
  int64_t pitch = (int64_t)c.kv_heads * D;
  const uint16_t *src = static_cast<const uint16_t *>(JOINT == 0 && is_v ? p.v : p.k);
  const int row0 = start + j * bt + lo - first;  // row of the block's first new token
  if constexpr (JOINT != 0) {
    pitch = (all.heads + 2 * (int64_t)c.kv_heads) * D;
    src += row0 * pitch + (all.heads + (is_v ? c.kv_heads : 0) + (int64_t)head) * D;
  } else {
    src += row0 * pitch + (int64_t)head * D;
  }
  uint8_t *dst = (is_v ? c.v_cache : c.k_cache) + (blk * c.kv_heads + head) * (int64_t)bt * D;
  float *scale = (is_v ? c.v_scale : c.k_scale) + blk * c.kv_heads + head;
  const float was = lo ? *scale : 0.f;

  typedef std::conditional_t<JOINT != 0, Wide8, v4u> Group;
  Group raw[NG];
  auto load = [&](int q) __attribute__((always_inline)) {
    if constexpr (JOINT != 0) {
      const int64_t pos = is_v ? 0 : RotaryRow(all.t, row0 + q / gd, j * bt + lo + q / gd);
      return JointValues<JOINT>(all.t, src + q / gd * pitch, q % gd * 8, !is_v, pos);
    } else {
      v4u r;
      __builtin_memcpy(&r, src + q / gd * pitch + q % gd * 8, 16);
      return r;
    }
  };
  // the largest magnitude as bits (both 16-bit types, and 32-bit ones, order like
  // whole numbers; a NaN is above every number)
  unsigned top = 0;
  auto look = [&](const Group &r) __attribute__((always_inline)) {
    if constexpr (JOINT != 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(unsigned, r.v[i]) & 0x7fffffffu);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, max(r[i] & 0x7fffu, r[i] >> 16 & 0x7fffu));
    }
  };
  if constexpr (KEPT) {
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (k * THREADS + tid < groups) raw[k] = load(k * THREADS + tid);
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (k * THREADS + tid < groups) look(raw[k]);
  } else {
    for (int q = tid; q < groups; q += THREADS) look(load(q));
  }
  for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
  if constexpr (THREADS > 64) {
    if (tid % 64 == 0) s_top[tid / 64] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) top = max(top, s_top[i]);
  }
  auto widen = [&](unsigned u) { return p.bf16 ? __builtin_bit_cast(float, u << 16) : F16ToF32((uint16_t)u); };
  BlockScale s = ScaleOf(JOINT != 0 ? __builtin_bit_cast(float, top) : widen(top), fp8 ? kFp8Max : kInt8Max);
  // a larger or NaN scale of the kept tokens stays; a NaN of the new ones too
  if (s.scale == s.scale && !(was <= s.scale)) s = BlockScale{was, was == was ? 1.f / was : 0.f, 0};
  const bool nan = s.scale != s.scale;
  if (lo && (nan || s.scale != was)) {
    // kept codes, 16 at a time: whole rows of keys; of values a piece of 16 tokens
    // may hold new ones and later ones, whose bytes stay
    const float ratio = was * s.inv;
    const int pieces = is_v ? D * ((lo + 15) / 16) : lo * D / 16;
    for (int q = tid; q < pieces; q += THREADS) {
      const int t = is_v ? q / D * 16 : 0;
      v4u *at = reinterpret_cast<v4u *>(dst + (is_v ? q % D * bt + t : 16 * q));
      v4u v = *at;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned n = nan ? 0u : Again4(v[i], ratio, fp8);
        const int kept = is_v ? lo - t - 4 * i : 4;  // of these four tokens
        const unsigned mask = kept >= 4 ? ~0u : kept <= 0 ? 0u : (1u << 8 * kept) - 1u;
        v[i] = (n & mask) | (v[i] & ~mask);
      }
      *at = v;
    }
    // before new bytes go into those pieces
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (THREADS > 64) __syncthreads();
  }
  if (tid == 0) *scale = s.scale;
  auto encode = [&](int q, const Group &r) __attribute__((always_inline)) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (JOINT != 0)
        v[i] = r.v[i] * s.inv;
      else
        v[i] = widen(r[i / 2] >> (16 * (i % 2)) & 0xffffu) * s.inv;
    }
    uint2 w = fp8 ? make_uint2(Fp8Codes4(v[0], v[1], v[2], v[3]), Fp8Codes4(v[4], v[5], v[6], v[7]))
                  : make_uint2(Int8Codes4(v[0], v[1], v[2], v[3]), Int8Codes4(v[4], v[5], v[6], v[7]));
    if (nan) w = make_uint2(0, 0);
    *reinterpret_cast<uint2 *>(is_v ? codes + q * 8 : dst + lo * D + q * 8) = w;
  };
  if constexpr (KEPT) {
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (k * THREADS + tid < groups) encode(k * THREADS + tid, raw[k]);
  } else {
    for (int q = tid; q < groups; q += THREADS) encode(q, load(q));
  }
  if (!is_v) return;
  __syncthreads();
  // 4 dimensions by 16 tokens per thread
  const int c0 = lo / 16, pieces = ((hi + 15) / 16 - c0) * (D / 4);
  for (int q = tid; q < pieces; q += THREADS) {
    const int t = (c0 + q / (D / 4)) * 16, d = q % (D / 4) * 4;
    if (t >= lo && t + 16 <= hi) {
      v4u out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = *reinterpret_cast<const unsigned *>(codes + (t - lo + 4 * i + e) * D + d);
        // bytes of 4 tokens x 4 dimensions change places
        const unsigned a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), a2 = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
        const unsigned b2 = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), b3 = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
        out[0][i] = __builtin_amdgcn_perm(b2, a, 0x05040100u);
        out[1][i] = __builtin_amdgcn_perm(b2, a, 0x07060302u);
        out[2][i] = __builtin_amdgcn_perm(b3, a2, 0x05040100u);
        out[3][i] = __builtin_amdgcn_perm(b3, a2, 0x07060302u);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<v4u *>(dst + (d + e) * bt + t) = out[e];
    } else {
      for (int u = max(t, lo); u < min(t + 16, hi); ++u) {
        const unsigned r = *reinterpret_cast<const unsigned *>(codes + (u - lo) * D + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[(d + e) * bt + u] = (uint8_t)(r >> (8 * e));
      }
    }
  }
}

template <int THREADS, int NG, bool KEPT> void LaunchBlocks(KvAppendParams p, int64_t blocks, hipStream_t s) {
  LaunchInPieces(blocks, THREADS, [&](int64_t first, unsigned count) {
    p.first = first;
    const dim3 grid(count, (unsigned)p.c.kv_heads, 2);
    KvAppendKernel<THREADS, NG, KEPT><<<grid, THREADS, p.c.block_tokens * p.c.head_dim, s>>>(p);
  });
}

template <int THREADS, int NG, bool KEPT> void LaunchBlocks(RotaryAppendParams p, int64_t blocks, hipStream_t s) {
  const KvCacheParams &c = p.a.c;
  const int D = c.head_dim, half = p.t.half, at_once = 64 / (D / 16);
  // whole lines of an aligned q: its stores go past the caches (rotary.hip); not those of a few
  // tokens, which the attention reads at once
  p.stream = (p.t.interleaved ? D % 128 == 0 : half % 64 == 0 && (D / 2 - half) % 64 == 0) &&
             reinterpret_cast<uintptr_t>(p.q) % 128 == 0 && THREADS > 64;
  p.blocks = blocks;
  // a piece a wave, and rounds past what the chip holds at once
  p.groups = std::min<int64_t>((c.tokens * ((p.heads + at_once - 1) / at_once) + THREADS / 64 - 1) / (THREADS / 64), 1280);
  LaunchInPieces(p.groups + 2 * blocks * c.kv_heads, THREADS, [&](int64_t first, unsigned count) {
    p.a.first = first;
    const int lds = c.block_tokens * D;
    if (p.a.bf16)
      KvAppendKernel<THREADS, NG, KEPT, kBfloat16><<<count, THREADS, lds, s>>>(p);
    else
      KvAppendKernel<THREADS, NG, KEPT, kFloat16><<<count, THREADS, lds, s>>>(p);
  });
}

template <typename P> void LaunchAppend(const KvCacheParams &c, const P &p, hipStream_t stream) {
  if (c.tokens == 0 || c.batch == 0) return;
  const int64_t most = MostNewBlocks(c);  // workgroups past the last block find none
  const int values = c.block_tokens * c.head_dim;
  // A wave per block where a sequence has a token or two on average: there is
  // little to share, and no barrier.  64 sequences with a token each, 8 heads of
  // 128: at least 4.4 us, with 256 threads 5.0 (5.1 in the middle for both).  Else 256 threads, which keep a block in
  // registers while it fits: four times 2048 tokens, blocks of 16 tokens one
  // group a thread 19.7 us, four 22.1; of 64 tokens kept 16.1 us (3.1 TB/s), read
  // twice 15.8, no difference between runs.
  if (c.tokens <= 2 * (int64_t)c.batch) {
    LaunchBlocks<64, 1, false>(p, most, stream);
  } else if (values <= 256 * 8) {
    LaunchBlocks<256, 1, true>(p, most, stream);
  } else if (values <= 4 * 256 * 8) {
    LaunchBlocks<256, 4, true>(p, most, stream);
  } else {
    LaunchBlocks<256, 1, false>(p, most, stream);
  }
}

}  // namespace

void LaunchKvCacheAppend(const KvAppendParams &p, hipStream_t stream) { LaunchAppend(p.c, p, stream); }
void LaunchRotaryKvCacheAppend(const RotaryAppendParams &p, hipStream_t stream) { LaunchAppend(p.a.c, p, stream); }

}  // namespace onnxl_amd
