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
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "quant8.hpp"

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

// NG groups of 8 values per thread are kept; KEPT: they are all there can be.
template <int THREADS, int NG, bool KEPT>
__global__ __launch_bounds__(THREADS) void KvAppendKernel(const KvAppendParams p) {
  extern __shared__ __align__(16) uint8_t codes[];  // [token][dimension] of the new values
  __shared__ unsigned s_top[THREADS / 64];
  const KvCacheParams &c = p.c;
  const int head = blockIdx.y, tid = threadIdx.x, bt = c.block_tokens, D = c.head_dim, gd = D / 8;
  const bool is_v = blockIdx.z != 0, fp8 = c.fp8;
  int b, w;
  if (!FindBlock(c, p.first + blockIdx.x, b, w)) return;
  const int len = c.lengths[b], start = c.start[b], first = len - (c.start[b + 1] - start);
  const int j = (first >> c.block_shift) + w;
  const int64_t blk = c.table[(int64_t)b * c.max_blocks + j];
  if (blk < 0 || blk >= c.num_blocks) return;
  const int lo = max(first - j * bt, 0), hi = min(len - j * bt, bt);  // tokens kept before lo, new from lo on
  const int groups = (hi - lo) * gd;
  const uint16_t *src = static_cast<const uint16_t *>(is_v ? p.v : p.k) +
                        ((int64_t)start + j * bt + lo - first) * c.kv_heads * D + (int64_t)head * D;
  uint8_t *dst = (is_v ? c.v_cache : c.k_cache) + (blk * c.kv_heads + head) * (int64_t)bt * D;
  float *scale = (is_v ? c.v_scale : c.k_scale) + blk * c.kv_heads + head;
  const float was = lo ? *scale : 0.f;

  v4u raw[NG];
  auto load = [&](int q) __attribute__((always_inline)) {
    v4u r;
    __builtin_memcpy(&r, src + (int64_t)(q / gd) * c.kv_heads * D + q % gd * 8, 16);
    return r;
  };
  // the largest magnitude as bits (both 16-bit types order like whole numbers; a
  // NaN is above every number)
  unsigned top = 0;
  auto look = [&](const v4u &r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max(r[i] & 0x7fffu, r[i] >> 16 & 0x7fffu));
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
  BlockScale s = ScaleOf(widen(top), fp8 ? kFp8Max : kInt8Max);
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
  auto encode = [&](int q, const v4u &r) __attribute__((always_inline)) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = widen(r[i / 2] >> (16 * (i % 2)) & 0xffffu) * s.inv;
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

}  // namespace

void LaunchKvCacheAppend(const KvAppendParams &p, hipStream_t stream) {
  const KvCacheParams &c = p.c;
  if (c.tokens == 0 || c.batch == 0) return;
  // n new tokens of a sequence lie in at most (n - 1) / block_tokens + 2 blocks,
  // and in n; workgroups past the last block find none
  const int64_t most = std::min<int64_t>(c.tokens, c.tokens / c.block_tokens + 2 * (int64_t)c.batch);
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

}  // namespace onnxl_amd
