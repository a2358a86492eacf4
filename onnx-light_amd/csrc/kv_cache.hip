// New keys and values into the paged 8-bit cache, one scale for each block of
// tokens and head.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"
#include "quant8.hpp"

namespace onnxl_amd {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float BlockMax(float v, float *s) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

__device__ __forceinline__ float CodeValue(uint8_t c, int fp8) { return fp8 ? Fp8E4M3ToF32(c) : (float)(int8_t)c; }

// One workgroup per (cache block with new tokens, head, k or v): its new scale
//   s' = max(scale of the tokens kept in the block, max|new| / qmax),
// the kept codes rounded again by s / s' where the scale grew, the new codes.
// grid.x runs over more blocks than there can be: every sequence's own and one
// more each.
__global__ __launch_bounds__(kThreads) void KvAppendKernel(const KvAppendParams p) {
  __shared__ float red[4];
  const KvCacheParams &c = p.c;
  const int head = blockIdx.y, tid = threadIdx.x, bt = c.block_tokens, D = c.head_dim;
  const bool is_v = blockIdx.z != 0;
  // the sequence and the block of it that this workgroup has
  int64_t w = blockIdx.x;
  int b = 0, n = 0;
  for (; b < c.batch; ++b) {
    n = KvNewTokens(c, b);
    if (n <= 0) continue;
    const int64_t first = c.lengths[b] - n, blocks = (c.lengths[b] + bt - 1) / bt - first / bt;
    if (w < blocks) break;
    w -= blocks;
  }
  if (b == c.batch) return;
  const int len = c.lengths[b], first = len - n;
  const int64_t j = first / bt + w;
  const int64_t blk = c.table[(int64_t)b * c.max_blocks + j];
  if (blk < 0 || blk >= c.num_blocks) return;
  const int lo = first > j * bt ? (int)(first - j * bt) : 0;             // tokens kept
  const int hi = len - j * bt < bt ? (int)(len - j * bt) : bt;
  const uint16_t *src = static_cast<const uint16_t *>(is_v ? p.v : p.k) +
                        ((int64_t)c.start[b] + j * bt + lo - first) * c.kv_heads * D + (int64_t)head * D;
  uint8_t *dst = (is_v ? c.v_cache : c.k_cache) + (blk * c.kv_heads + head) * (int64_t)bt * D;
  float *scale = (is_v ? c.v_scale : c.k_scale) + blk * c.kv_heads + head;
  auto at = [&](int t, int d) { return is_v ? d * bt + t : t * D + d; };
  auto value = [&](int i) {
    const uint16_t u = src[(int64_t)(i / D) * c.kv_heads * D + i % D];
    return p.bf16 ? Bf16ToF32(u) : F16ToF32(u);
  };
  float top = 0.f;
  bool finite = true;
  for (int i = tid; i < (hi - lo) * D; i += kThreads) {
    const float v = fabsf(value(i));
    finite = finite && v < __builtin_huge_valf();
    top = fmaxf(top, v);
  }
  top = BlockMax(finite ? top : __builtin_huge_valf(), red);
  const float qmax = c.fp8 ? kFp8Max : kInt8Max;
  BlockScale s = ScaleOf(top, qmax);
  const float was = lo ? *scale : 0.f;
  if (!(was <= s.scale)) {  // a larger or NaN scale stays; a NaN of the new tokens stays too
    if (s.scale == s.scale) s = BlockScale{was, was == was ? 1.f / was : 0.f, 0};
  }
  __syncthreads();
  if (tid == 0) *scale = s.scale;
  if (lo && s.scale != was) {
    const float ratio = was * s.inv;
    for (int i = tid; i < lo * D; i += kThreads) {
      uint8_t *q = dst + at(i / D, i % D);
      const float v = CodeValue(*q, c.fp8) * ratio;
      *q = c.fp8 ? Fp8Code(v) : Int8Code(v);
    }
  }
  for (int i = tid; i < (hi - lo) * D; i += kThreads) {
    const float v = value(i) * s.inv;
    dst[at(lo + i / D, i % D)] = c.fp8 ? Fp8Code(v) : Int8Code(v);
  }
}

}  // namespace

void LaunchKvCacheAppend(const KvAppendParams &p, hipStream_t stream) {
  const KvCacheParams &c = p.c;
  if (c.tokens == 0 || c.batch == 0) return;
  // n new tokens lie in at most (n - 1) / bt + 2 blocks, and in n
  const int64_t most = std::min<int64_t>(c.tokens, c.tokens / c.block_tokens + 2 * (int64_t)c.batch);
  KvAppendKernel<<<dim3((unsigned)most, (unsigned)c.kv_heads, 2), kThreads, 0, stream>>>(p);
}

}  // namespace onnxl_amd
