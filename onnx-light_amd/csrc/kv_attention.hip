// Causal attention of the newest tokens of every sequence over the paged 8-bit
// cache.
#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"

namespace onnxl_amd {
namespace {

__device__ __forceinline__ float CodeValue(uint8_t c, int fp8) { return fp8 ? Fp8E4M3ToF32(c) : (float)(int8_t)c; }

// One wave per (token, head): lane l holds dimensions l, l + 64, ..; one pass
// over the tokens with the running maximum m and sum s of the softmax.
__global__ __launch_bounds__(64) void KvAttentionKernel(const KvAttentionParams p) {
  const KvCacheParams &c = p.c;
  const int64_t row = blockIdx.x;
  const int head = blockIdx.y, lane = threadIdx.x, D = c.head_dim, bt = c.block_tokens;
  const int kvh = head / (p.heads / c.kv_heads);
  int b = 0;
  while (b < c.batch && !(c.start[b] <= row && row < c.start[b + 1])) ++b;
  const int n = b < c.batch ? KvNewTokens(c, b) : -1;
  const int64_t at = (row * p.heads + head) * D;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -__builtin_huge_valf(), s = 0.f;
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    const uint16_t u = d < D ? static_cast<const uint16_t *>(p.q)[at + d] : 0;
    q[i] = p.bf16 ? Bf16ToF32(u) : F16ToF32(u);
  }
  bool good = n > 0;
  const int64_t last = good ? (int64_t)c.lengths[b] - n + (row - c.start[b]) : -1;
  for (int64_t t = 0; t <= last && good; ++t) {
    const int64_t blk = c.table[(int64_t)b * c.max_blocks + t / bt];
    if (blk < 0 || blk >= c.num_blocks) {
      good = false;
      break;
    }
    const int64_t base = (blk * c.kv_heads + kvh) * (int64_t)bt * D;
    const int u = (int)(t % bt);
    float dot = 0.f;
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < D) dot += q[i] * CodeValue(c.k_cache[base + (int64_t)u * D + d], c.fp8);
    }
    for (int w = 32; w > 0; w >>= 1) dot += __shfl_xor(dot, w);
    const float z = dot * c.k_scale[blk * c.kv_heads + kvh] * p.scale, mn = fmaxf(m, z);
    const float keep = __expf(m - mn), e = __expf(z - mn), ev = e * c.v_scale[blk * c.kv_heads + kvh];
    s = s * keep + e;
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < D) o[i] = o[i] * keep + ev * CodeValue(c.v_cache[base + (int64_t)d * bt + u], c.fp8);
    }
    m = mn;
  }
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    const float v = good ? o[i] / s : __builtin_nanf("");
    if (d < D) static_cast<uint16_t *>(p.out)[at + d] = p.bf16 ? F32ToBf16(v) : F32ToF16(v);
  }
}

}  // namespace

size_t KvAttentionScratchBytes(const KvAttentionParams &) { return 0; }

void LaunchKvCacheAttention(const KvAttentionParams &p, void *, hipStream_t stream) {
  if (p.c.tokens == 0) return;
  KvAttentionKernel<<<dim3((unsigned)p.c.tokens, (unsigned)p.heads), 64, 0, stream>>>(p);
}

}  // namespace onnxl_amd
