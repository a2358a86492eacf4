// Launch parameters and launcher declarations of the decoder-layer operators
// that stand between the quantized products: RMS norm with 8-bit output,
// microscaled (MX) quantization, product and gated feed-forward, rotary
// positions, the paged 8-bit key / value cache and its attention, and sampling.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "mx_plan.hpp"

namespace onnxl_amd {

// A launch has fewer than 2^32 threads along x: a larger grid runs in part, and
// nothing reports it.  launch(first, count) gets the workgroups piece by piece.
template <typename F> void LaunchInPieces(int64_t groups, int threads, F launch) {
  const int64_t most = (int64_t(1) << 31) / threads;
  for (int64_t first = 0; first < groups; first += most)
    launch(first, (unsigned)(groups - first < most ? groups - first : most));
}

// ---------------------------------------------------------------------------
// RMS norm with the residual's addition and 8-bit output.
//   h = round16(x + residual)  (x without a residual),  written to sum
//   y = h * (1 / sqrt(mean(h^2) + eps)) * weight, in fp32
//   per block of `block` values: scale = max|y| / qmax, code = round(y / scale)
// A block with a value that is not finite gets a NaN scale and zero codes.

enum RmsNormScale : int { kRnsFloat = 0, kRnsE8M0 = 1 };

struct RmsNormParams {
  const void *x;
  const void *residual;  // or nullptr
  const void *weight;
  void *y;
  void *scale;           // FLOAT or E8M0 [rows, D / block]
  void *sum;             // or nullptr; may be x's or the residual's own memory
  int64_t rows, D, block;
  float eps;
  int x_dtype;           // kFloat, kFloat16, kBfloat16 (x, residual and sum)
  int weight_f32;        // weight is FLOAT, else x's type
  int y_fp8;             // FLOAT8E4M3FN codes, else INT8
  int scale_kind;        // RmsNormScale
  int64_t first;         // row of the launch's first workgroup
};
void LaunchRmsNormQuantize(const RmsNormParams &p, hipStream_t stream);

// ---------------------------------------------------------------------------
// Microscaled (MX) types: blocks of 32 values along K with an E8M0 scale,
// 2^(e - 127), e = 255 NaN.  Codes E4M3 (one byte) or E2M1 (two in a byte, the
// even element in the low nibble).

struct MxQuantParams {
  const void *x;     // [rows, K], K % 32 == 0
  uint8_t *y;        // codes
  uint8_t *scale;    // [rows, K / 32]
  int64_t rows, K;
  int x_dtype;       // kFloat, kFloat16, kBfloat16
  int fp4;           // E2M1 codes, else E4M3
  int64_t first;     // the launch's first workgroup of 2048 values
};
void LaunchMxQuantize(const MxQuantParams &p, hipStream_t stream);

// y[m, n] = sum over blocks of 2^(sa + sb) * sum of a[m, k] b[n, k]; M, N > 0.
// Gated: y = act(a . b^T) * (a . up^T), both weights [N, K], in 16 bits or as MXFP8
// (codes y and E8M0 scales y_scale [M, N / 32], N % 32 == 0).
enum Activation : int { kSilu = 0, kGelu = 1, kGeluTanh = 2, kRelu = 3 };
struct MxMatMulParams {
  const void *x;           // [M, K] FLOAT16 or BFLOAT16, quantized by the call; or nullptr and
  const uint8_t *a;        // [M, K] E4M3 or E2M1 codes with
  const uint8_t *a_scale;  // [M, K / 32]
  const uint8_t *b;        // [N, K] E2M1 codes
  const uint8_t *b_scale;  // [N, K / 32]
  void *y;                 // [M, N] FLOAT16 or BFLOAT16
  int64_t M, N, K;
  int x_dtype;             // of x
  int a_fp4;               // a's codes are (or x's become) E2M1, else E4M3
  int y_bf16;
  int output;              // MxOutput
  const uint8_t *up, *up_scale;  // the second weight of a gated product
  int activation;
  uint8_t *y_scale;
};
size_t MxMatMulScratchBytes(const MxMatMulParams &p);
void LaunchMxMatMul(const MxMatMulParams &p, void *scratch, hipStream_t stream);

// ---------------------------------------------------------------------------
// Paged 8-bit cache.
//   k_cache [blocks, kv_heads, block_tokens, head_dim]
//   v_cache [blocks, kv_heads, head_dim, block_tokens]  (token-contiguous: the
//           layout of the second product's matrix operand)
//   k_scale, v_scale FLOAT [blocks, kv_heads]
//   block_table INT32 [batch, max_blocks], query_start INT32 [batch + 1] (first
//   new token of every sequence), lengths INT32 [batch] (tokens in the cache
//   with the new ones).
// A sequence whose numbers do not fit its tensors (new tokens < 0 or beyond
// its length, a length beyond the table, rows past the last token) is not
// appended and its attention is NaN; new tokens of a block outside the cache
// are dropped, and rows that see one are NaN.
// Each sequence is judged by its own numbers, so where query_start falls several
// may claim the same rows: the last to write them wins, their NaN among it, and an
// append, whose launch counts on no more new tokens than rows, may leave some out.

struct KvCacheParams {
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  const int32_t *table, *start, *lengths;
  int64_t num_blocks;
  int kv_heads, block_tokens, block_shift, head_dim;
  int batch, max_blocks;
  int64_t tokens;  // new tokens: rows of k, v and q
  int fp8;         // FLOAT8E4M3FN codes, else INT8
};

struct KvAppendParams {
  KvCacheParams c;
  const void *k, *v;  // [tokens, kv_heads, head_dim]
  int bf16;           // BFLOAT16, else FLOAT16
  int64_t first;      // new block of the launch's first workgroup
};
void LaunchKvCacheAppend(const KvAppendParams &p, hipStream_t stream);
// n new tokens of a sequence lie in at most (n - 1) / block_tokens + 2 blocks, and in n.
inline int64_t MostNewBlocks(const KvCacheParams &c) {
  return std::min<int64_t>(c.tokens, c.tokens / c.block_tokens + 2 * (int64_t)c.batch);
}

// ---------------------------------------------------------------------------
// Rotary positions: pairs (a, b) of a head's first 2 half dimensions, (i, half + i)
// or (2 i, 2 i + 1), become (a c - b s, a s + b c) with row `position` of the
// tables cos and sin [positions, half]; the other dimensions stay.

enum RotaryScaling : int { kRotaryNone = 0, kRotaryLinear = 1, kRotaryNtk = 2, kRotaryByParts = 3, kRotaryYarn = 4 };

struct RotaryTablesParams {
  void *cos, *sin;      // [positions, half]
  int64_t positions;
  int half;
  int dtype;            // kFloat, kFloat16, kBfloat16
  int scaling;          // RotaryScaling
  double log_base;      // of the base, ntk's growth included
  double factor, original, turns_fast, turns_slow;
  double low, high;     // yarn: pairs up to low keep their frequency, from high on 1 / factor of it
  float magnitude;
};
void LaunchRotaryTables(const RotaryTablesParams &p, hipStream_t stream);

struct RotaryTable {
  const void *cos, *sin;  // [positions, half], FLOAT or the rotated tensor's type
  int64_t positions;
  int half, f32, interleaved;
  const void *ids;        // INT32 or INT64 position of every token, or nullptr
  int ids64;
};

struct RotaryParams {
  RotaryTable t;          // ids nullptr: row `token` of the tables
  const void *x;
  void *y;                // the same layout; may be x
  int64_t tokens, seq;    // tokens: batch * seq
  int heads, D;
  int by_head;            // [batch, heads, seq, D], else [tokens, heads, D]
  int dtype;              // kFloat, kFloat16, kBfloat16
  int64_t first;          // the launch's first workgroup
};
void LaunchRotaryEmbedding(const RotaryParams &p, hipStream_t stream);

// The append of a joint projection's rows [tokens, heads + 2 kv_heads, head_dim]:
// queries rotated into q, keys rotated and values as they are into the cache.
struct RotaryAppendParams {
  KvAppendParams a;       // k: the joint rows; v is not looked at
  RotaryTable t;          // ids nullptr: a token's place in its sequence
  void *q;                // [tokens, heads, head_dim]
  int heads;
  int64_t groups, blocks; // the launcher's: workgroups for queries, and for keys of a head,
  bool stream;            // and whether q is written past the caches
};
void LaunchRotaryKvCacheAppend(const RotaryAppendParams &p, hipStream_t stream);

struct KvAttentionParams {
  KvCacheParams c;
  const void *q;      // [tokens, heads, head_dim]
  void *out;          // the same
  int heads, bf16;
  float scale;
  int64_t max_query;  // most new tokens of a sequence where known, else 0
};
size_t KvAttentionScratchBytes(const KvAttentionParams &p);
void LaunchKvCacheAttention(const KvAttentionParams &p, void *scratch, hipStream_t stream);

// ---------------------------------------------------------------------------
// A token from each row of logits and a given random number.

struct SampleParams {
  const void *x;             // [rows, vocab]
  const float *uniform;      // [rows]
  const float *temperature;  // [rows], or nullptr: 1
  const void *top_k;         // INT32 or INT64 [rows], or nullptr: all
  const float *top_p;        // [rows], or nullptr: 1
  const float *min_p;        // [rows], or nullptr: 0
  void *token;               // INT32 or INT64 [rows]
  float *probability;        // [rows], or nullptr
  int64_t rows;
  int vocab;
  int dtype;                 // kFloat, kFloat16, kBfloat16
  int k64, token64;
  int64_t first;             // row of the launch's first workgroup
};
size_t SampleScratchBytes(const SampleParams &p);
void LaunchSampleTokens(const SampleParams &p, void *scratch, hipStream_t stream);

#ifdef __HIPCC__
// New tokens of sequence b, or -1 where its numbers do not fit.
__device__ __forceinline__ int KvNewTokens(const KvCacheParams &c, int b) {
  const int64_t lo = c.start[b], hi = c.start[b + 1], len = c.lengths[b];
  const bool fits = lo >= 0 && hi >= lo && hi <= c.tokens && hi - lo <= len &&
                    len <= (int64_t)c.max_blocks * c.block_tokens;
  return fits ? (int)(hi - lo) : -1;
}
#endif

}  // namespace onnxl_amd
