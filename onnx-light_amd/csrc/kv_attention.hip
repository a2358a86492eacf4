// Causal attention of the newest tokens of every sequence over the paged 8-bit
// cache.
//
// For one sequence and kv head the rows of a matrix product are the (new
// token, head of the group) pairs, row = token * group + head, so that the
// heads that share keys and values share every byte read.  A tile is 64 tokens
// of the cache:
//   S^T = K Q^T   (16 x 16 x 32 MFMA, A = 16 tokens of K, B = 16 rows of Q)
//   P   = 2^(S - m)
//   O^T += V^T P  (A = 16 dimensions of V^T, B = P)
// Result lane 16 g + c of the first product holds 4 tokens of row c.  The token
// in A's row r of the 16-token operand t is 16 (r / 4) + 4 t + r % 4, so over
// the four operands lane group g gets the 16 consecutive tokens from 16 g, which
// is what the second product's B operand wants of it (P never leaves the
// registers) and, in the token-contiguous V cache, one 16-byte load per
// dimension (no transposition).  Those 16 tokens lie in one cache block, so
// both scales are one number per lane and tile.
//
// Codes become fp16 exactly (|int8| <= 128, E4M3 is a subset).  Q becomes fp16
// after a power of two per row has brought its largest value to [1, 2): exact
// but for what is below 2^-14 of that largest.  Sums, statistics and O are
// fp32; P is rounded to fp16.  The weight of a token in O is its softmax weight
// times its block's v scale, so P is taken relative to mo, the running maximum
// of S + log2(v scale): P = 2^(S + log2 vs - mo + kTop) fills the fp16 range whatever
// the scales are.  The softmax sum takes the unrounded P / vs (one
// multiplication per 16 tokens), and O / sum needs no other reference.
#include <type_traits>

#include "common.hpp"
#include "decoder.hpp"
#include "device_codecs.hpp"

namespace onnxl_amd {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256, kWaves = 4, kTile = 64;
constexpr float kNone = -0x1.fffffep127f;  // the maximum of no token: no finite score is below it
constexpr float kLog2e = 1.44269504088896340736f;

// Eight codes (two dwords) as fp16, exact.
template <bool FP8> __device__ __forceinline__ v8h Widen(int lo, int hi) {
  v8h r;
  v2h *h = reinterpret_cast<v2h *>(&r);
  if constexpr (FP8) {
    h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
    h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
    h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
    h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  } else {
    // the byte c + 128 under the exponent of 1024 is 1024 + 128 + c
    const v2h off = {(_Float16)-1152.f, (_Float16)-1152.f};
    const unsigned a = (unsigned)lo ^ 0x80808080u, b = (unsigned)hi ^ 0x80808080u, e = 0x64646464u;
    h[0] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(a, e, 0x00050004u)) + off;
    h[1] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(a, e, 0x00070006u)) + off;
    h[2] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(b, e, 0x00050004u)) + off;
    h[3] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(b, e, 0x00070006u)) + off;
  }
  return r;
}

__device__ __forceinline__ uint2 Pack4(v4f v, int bf16) {
  typedef _Float16 v4h __attribute__((ext_vector_type(4)));
  uint2 b;  // pairs by the instruction itself: one for two values, to nearest even
  asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(b.x) : "v"(v[0]), "v"(v[1]));
  asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(b.y) : "v"(v[2]), "v"(v[3]));
  const uint2 h = __builtin_bit_cast(uint2, __builtin_convertvector(v, v4h));
  return make_uint2(bf16 ? b.x : h.x, bf16 ? b.y : h.y);
}

// P is up to 2^kTop, near the largest fp16: its smallest is 2^-24, so a weight
// keeps 11 bits down to 2^-29 of the row's largest (of weight times v scale), and
// is lost below 2^-40 (2^kLag times these in the prompt kernel).  O carries that
// power of two, the sum does not.
constexpr float kTop = 15.f;

// log2 of a token's weight in O: score (s * cs) plus log2 of its v scale, two
// roundings, never fused, so that it is the same wherever it is computed.
__device__ __forceinline__ float Weight(float s, float cs, float lv) {
#pragma clang fp contract(off)
  const float z = s * cs;
  return z + lv;
}

// log2 of a v scale and its inverse.  A scale below 2^-100 (zero: a block of
// zeros) counts as 2^-100; NaN stays.
__device__ __forceinline__ float LogScale(float vs) { return vs > 0x1p-100f ? __builtin_amdgcn_logf(vs) : vs == vs ? -100.f : vs; }
__device__ __forceinline__ float InvScale(float vs) { return vs > 0x1p-100f ? __builtin_amdgcn_rcpf(vs) : 0x1p100f; }

// What the G lane groups hold (lanes l, l ^ 32 and, of four, l ^ 16, l ^ 48),
// joined: swaps of register halves, no trip through LDS.
template <int G, typename F> __device__ __forceinline__ float OverGroups(float v, F join) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const float w = join(__builtin_bit_cast(float, (unsigned)a[0]), __builtin_bit_cast(float, (unsigned)a[1]));
  if (G == 2) return w;
  const unsigned x = __builtin_bit_cast(unsigned, w);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return join(__builtin_bit_cast(float, (unsigned)b[0]), __builtin_bit_cast(float, (unsigned)b[1]));
}
template <int G = 4> __device__ __forceinline__ float GroupMax(float v) {
  return OverGroups<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G = 4> __device__ __forceinline__ float GroupSum(float v) {
  return OverGroups<G>(v, [](float a, float b) { return a + b; });
}

// ---------------------------------------------------------------------------
// Few rows (decoding): the reading of the cache is the cost.  The tiles of all
// (sequence, kv head, 16-row tile) jobs form one line of units, and every
// workgroup takes an equal piece of it, whatever the lengths are; its waves
// take the tiles of a job in turn and join in LDS.  A job inside the piece is
// written out; the parts of a job that crosses pieces go to the workspace, at
// most two per workgroup (the first and the last of its piece), and the
// workgroup that writes the last of them joins them, in the order of the pieces
// whoever that is.
//
// 64 sequences of 500 to 16384 tokens, 64 heads over 8 of 128 dimensions: 1.1 GB in
// 206 us, 5.4 TB/s (a copy of 1 GB reaches 5.1).  One sequence of 8191 tokens: 17 MB
// in 13.2 us, a chain of latencies (lengths, table, tile, parts, their join).

struct Line {        // units before every thread's share of the sequences
  int64_t upto[kThreads];
};

struct Job {
  int b, n, len, head, row0;  // sequence, its new tokens and length, kv head, first row
  int start;                  // its first new token
  int tiles;                  // units of the job
  int64_t first;              // its first unit on the line
};

struct Plan {
  KvAttentionParams a;
  int group;
  int rows_max;     // sequences with more rows (new tokens * group) are the prompt kernel's
  int fill;         // NaN for the rows of sequences that do not fit
  float *part;      // parts: [workgroup][2][HD / 16][64] float4
  float *stat;      // [workgroup][2][2][16]: mo, the sum
  unsigned *done;   // [workgroup] parts written of the job that starts last in its piece; zero between launches
};

// New tokens of sequence b that this kernel has (0: none).
__device__ __forceinline__ int RowsOf(const Plan &p, int b) {
  const int n = KvNewTokens(p.a.c, b);
  return n > 0 && (int64_t)n * p.group <= p.rows_max ? n : 0;
}
__device__ __forceinline__ int64_t UnitsOf(const Plan &p, int b) {
  const int n = RowsOf(p, b);
  if (n == 0) return 0;
  return (int64_t)p.a.c.kv_heads * ((n * p.group + 15) / 16) * ((p.a.c.lengths[b] + kTile - 1) / kTile);
}

__device__ __forceinline__ int Uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int Lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ int64_t Lane(int64_t v, int lane) {
  return (int64_t)((uint64_t)(uint32_t)Lane((int)(v >> 32), lane) << 32 | (uint32_t)Lane((int)v, lane));
}
__device__ __forceinline__ int64_t Uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)Uniform((int)(v >> 32)) << 32 | (uint32_t)Uniform((int)v));
}

// Fills `line` and returns the number of units.
__device__ __forceinline__ int64_t MakeLine(const Plan &p, Line &line) {
  const int B = p.a.c.batch, share = (B + kThreads - 1) / kThreads, tid = threadIdx.x;
  int64_t mine = 0;
  for (int b = tid * share; b < min(B, (tid + 1) * share); ++b) mine += UnitsOf(p, b);
  int64_t sum = mine;
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t v = __shfl_up(sum, o);
    if (tid % 64 >= o) sum += v;
  }
  line.upto[tid] = sum;
  __syncthreads();
  int64_t before = 0;
  for (int w = 0; w < tid / 64; ++w) before += line.upto[64 * w + 63];
  __syncthreads();
  line.upto[tid] = sum + before;
  __syncthreads();
  return Uniform(line.upto[kThreads - 1]);
}

// NaN for the rows of sequences whose numbers do not fit.
__device__ __forceinline__ void FillInvalid(const Plan &p) {
  const KvCacheParams &c = p.a.c;
  for (int b = blockIdx.x; b < c.batch; b += gridDim.x) {
    if (KvNewTokens(c, b) >= 0) continue;
    const int64_t lo = c.start[b] < 0 ? 0 : c.start[b], hi = c.start[b + 1] < c.tokens ? c.start[b + 1] : c.tokens;
    const int64_t wide = (int64_t)p.a.heads * c.head_dim;
    for (int64_t i = lo * wide + threadIdx.x; i < hi * wide; i += blockDim.x)
      static_cast<uint16_t *>(p.a.out)[i] = p.a.bf16 ? 0x7fc0 : 0x7e00;
  }
}

// The 64 bits' quotient; most are short, and a long division takes four times as
// many instructions.
__device__ __forceinline__ int64_t Over(int64_t a, int b) {
  return (uint64_t)a >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// The job of unit u of sequence b, whose units start at `at`; the same in every lane.
__device__ __forceinline__ Job JobOf(const Plan &p, int64_t u, int64_t at, int b, int n, int len, int start) {
  Job j;
  j.b = b;
  j.n = n;
  j.len = len;
  j.start = start;
  j.tiles = (len + kTile - 1) / kTile;
  const int row_tiles = (n * p.group + 15) / 16;
  const int64_t k = Uniform(Over(u - at, j.tiles));
  j.head = (int)Over(k, row_tiles);
  j.row0 = (int)(k - (int64_t)j.head * row_tiles) * 16;
  j.first = at + k * j.tiles;
  return j;
}

__device__ __forceinline__ Job FindJob(const Plan &p, const Line &line, int64_t u) {
  const int share = (p.a.c.batch + kThreads - 1) / kThreads;
  int lo = 0, hi = kThreads - 1;
  while (lo < hi) {  // the first thread whose share ends past u
    const int mid = (lo + hi) / 2;
    if (line.upto[mid] > u) hi = mid; else lo = mid + 1;
  }
  int64_t at = lo ? line.upto[lo - 1] : 0;
  int b = lo * share;
  for (;; ++b) {
    const int64_t n = UnitsOf(p, b);
    if (u < at + n) break;
    at += n;
  }
  b = Uniform(b);
  return JobOf(p, u, Uniform(at), b, Uniform(RowsOf(p, b)), Uniform(p.a.c.lengths[b]), Uniform(p.a.c.start[b]));
}

// Up to 64 sequences: lane b of every wave keeps what there is to know of sequence
// b, and nobody searches LDS or waits for another wave: one sequence of 8191
// tokens 16.0 -> 15.2 us (with the join of parts below 13.2).
struct Lanes {
  int64_t upto;       // units up to the end of the sequence
  int n, len, start;  // its rows' new tokens, length, first new token
};
__device__ __forceinline__ int64_t MakeLanes(const Plan &p, Lanes &l) {
  const int B = p.a.c.batch, b = threadIdx.x % 64;
  const int at = b < B ? b : 0, n = KvNewTokens(p.a.c, at);
  l.start = p.a.c.start[at];
  l.len = p.a.c.lengths[at];
  l.n = b < B && n > 0 && (int64_t)n * p.group <= p.rows_max ? n : 0;
  l.upto = l.n ? (int64_t)p.a.c.kv_heads * ((l.n * p.group + 15) / 16) * ((l.len + kTile - 1) / kTile) : 0;
  for (int o = 1; o < B; o <<= 1) {
    const int64_t v = __shfl_up(l.upto, o);
    if (b >= o) l.upto += v;
  }
  if (p.fill && __any(b < B && n < 0)) FillInvalid(p);
  return Lane(l.upto, B - 1);
}
__device__ __forceinline__ Job FindJob(const Plan &p, const Lanes &l, int64_t u) {
  const int b = __builtin_ctzll(__ballot(l.upto > u));
  const int64_t at = b ? Lane(l.upto, b - 1) : 0;
  return JobOf(p, u, at, b, Lane(l.n, b), Lane(l.len, b), Lane(l.start, b));
}

// Units of one workgroup: equal pieces, of at least one tile per wave.
__device__ __forceinline__ int64_t PieceOf(int64_t units) {
  const int64_t piece = (units + gridDim.x - 1) / gridDim.x;
  return piece < kWaves ? kWaves : piece;
}

// Where a row's output goes, and the dimensions from d on of it.
__device__ __forceinline__ uint16_t *OutRow(const Plan &p, const Job &j, int row) {
  const int64_t token = j.start + (int64_t)(row / p.group);
  return static_cast<uint16_t *>(p.a.out) + (token * p.a.heads + j.head * p.group + row % p.group) * p.a.c.head_dim;
}
__device__ __forceinline__ void StoreDims(const Plan &p, uint16_t *out, int d, v4f o) {
  if (d >= p.a.c.head_dim) return;
  const uint2 h = Pack4(o, p.a.bf16);
  __builtin_memcpy(out + d, &h, 8);
}
// O / sum of the rows that there are: 16 dimensions of 16 rows.
__device__ __forceinline__ void StoreRows(const Plan &p, const Job &j, int t, v4f o, float sum) {
  const int row = j.row0 + threadIdx.x % 16;
  if (row < j.n * p.group) StoreDims(p, OutRow(p, j, row), 16 * t + threadIdx.x % 64 / 16 * 4, o * (0x1p-15f / sum));
}

// 16 bytes from any address.
__device__ __forceinline__ v4i Load16(const void *p) {
  v4i v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// Q of one row as the first product's operand: lane group g holds the
// dimensions 64 h + 16 g + 8 s + (0..7) at q[h][s], scaled by 2^-exponent and
// with the sign of the softmax scale.
template <int CH, bool EXACT> struct QRow {
  v4i raw[CH][2];
  v8h q[CH][2];
  int exponent;

  __device__ __forceinline__ void Load(const KvAttentionParams &p, int64_t at, bool live, int g) {
    for (int h = 0; h < CH; ++h)
      for (int s = 0; s < 2; ++s) {
        const int d = 64 * h + 16 * g + 8 * s;
        raw[h][s] = live && (EXACT || d < p.c.head_dim) ? Load16(static_cast<const uint16_t *>(p.q) + at + d) : v4i{0, 0, 0, 0};
      }
  }
  __device__ __forceinline__ void Scale(const KvAttentionParams &p) {
    float v[CH][2][8], top = 0.f;
    for (int h = 0; h < CH; ++h)
      for (int s = 0; s < 2; ++s)
        for (int i = 0; i < 8; ++i) {
          const int w = raw[h][s][i / 2];
          const uint16_t u = (uint16_t)((unsigned)w >> (16 * (i % 2)));
          v[h][s][i] = p.bf16 ? Bf16ToF32(u) : F16ToF32(u);
          top = fmaxf(top, fabsf(v[h][s][i]));
        }
    top = GroupMax(top);
    exponent = top > 0.f && top < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
    for (int h = 0; h < CH; ++h)
      for (int s = 0; s < 2; ++s)
        for (int i = 0; i < 8; ++i) {
          const float x = __builtin_amdgcn_ldexpf(v[h][s][i], -exponent);
          q[h][s][i] = (_Float16)(p.scale < 0.f ? -x : x);
        }
  }
};

// One tile's codes and scales of a wave, loaded ahead of their use, and the
// cache blocks of the tile after it.
template <int HD, bool EXACT> struct TileLoad {
  static constexpr int DT = HD / 16, CH = HD / 64;
  int kb, vb;  // blocks of the tile to load next
  const uint8_t *vp;
  v4i k[4][CH], v[DT];
  float ks, vs;

  // Tokens past the end are looked up as the last there is.
  __device__ __forceinline__ void Lookup(const KvCacheParams &p, const Job &j, int t, int c, int g) {
    const int32_t *table = p.table + (int64_t)j.b * p.max_blocks;
    kb = table[min(t * kTile + 16 * (c / 4), j.len - 1) >> p.block_shift];
    vb = table[min(t * kTile + 16 * g, j.len - 1) >> p.block_shift];
  }
  // Keys and scales of tile t.  A block outside the cache reads block 0 and gets
  // a NaN k scale, so NaN scores; its values become zeros before they are used.
  __device__ __forceinline__ void LoadK(const KvCacheParams &p, const Job &j, int t, int c, int g) {
    const int kt = t * kTile + 16 * (c / 4), vt = t * kTile + 16 * g, D = EXACT ? HD : p.head_dim, bt = p.block_tokens;
    const bool bad = vb < 0 || vb >= p.num_blocks;
    const int64_t k_at = (int64_t)(kb >= 0 && kb < p.num_blocks ? kb : 0) * p.kv_heads + j.head;
    const int64_t v_at = (int64_t)(bad ? 0 : vb) * p.kv_heads + j.head;
    const uint8_t *kp = p.k_cache + (k_at * bt + (kt & (bt - 1)) + c % 4) * D + 16 * g;
    vp = p.v_cache + (v_at * D + c) * bt + (vt & (bt - 1));
    for (int s = 0; s < 4; ++s)
      for (int h = 0; h < CH; ++h)
        k[s][h] = EXACT || 64 * h + 16 * g < D ? *reinterpret_cast<const v4i *>(kp + 4 * s * D + 64 * h) : v4i{0, 0, 0, 0};
    ks = p.k_scale[v_at];
    ks = bad ? __builtin_nanf("") : ks;
    vs = p.v_scale[v_at];
  }
  __device__ __forceinline__ void LoadV(const KvCacheParams &p) {
    const int D = EXACT ? HD : p.head_dim;
    for (int d = 0; d < DT; ++d)
      v[d] = EXACT || 16 * d < D ? *reinterpret_cast<const v4i *>(vp + (int64_t)16 * d * p.block_tokens) : v4i{0, 0, 0, 0};
  }
};

// Parts are written and read past the XCDs' own L2 caches (sc1), so that no
// fence has to write those back or drop them.
constexpr int kDeviceScope = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t Rsrc(void *p) {
  return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, 0x7fffffff, 0x00020000);
}
__device__ __forceinline__ void PutStat(const Plan &p, int slot, int i, int c, float v) {
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), Rsrc(p.stat), ((slot * 2 + i) * 16 + c) * 4, 0,
                                        kDeviceScope);
}
__device__ __forceinline__ float GetStat(const Plan &p, int slot, int i, int c) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_raw_buffer_load_b32(Rsrc(p.stat), ((slot * 2 + i) * 16 + c) * 4, 0, kDeviceScope));
}

// The waves' results in LDS, so with the statistics sm, as one: their factors, the
// sum and, returned, the maximum of row c.
template <typename SM> __device__ __forceinline__ float JoinWaves(const SM &sm, int c, float (&f)[kWaves], float &sum) {
  float mo = kNone;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mo = fmaxf(mo, sm[w][0][c]);
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = __builtin_amdgcn_exp2f(sm[w][0][c] - mo);
    sum += sm[w][1][c] * f[w];
  }
  return mo;
}
template <typename SO> __device__ __forceinline__ v4f WaveSum(const SO &so, const float (&f)[kWaves], int d, int lane) {
  v4f a = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) a += so[w][d][lane] * f[w];
  return a;
}

// Joins the parts of a job: slot `first` of piece w0, slots 2 w of the others.
// Every wave has its share of the dimensions, so that nothing is joined between
// waves, and kFly parts' loads on their way at once.
template <int HD> __device__ __forceinline__ void JoinParts(const Plan &p, const Job &j, int w0, int w1, int first) {
  constexpr int DT = HD / 16, kMine = DT / kWaves, kFly = kMine == 4 ? 4 : 8;
  const int lane = threadIdx.x % 64, c = lane % 16, wave = threadIdx.x / 64;
  const int parts = w1 - w0 + 1;
  float mo = kNone, sum = 0.f;
  v4f a[kMine];
#pragma unroll
  for (int d = 0; d < kMine; ++d) a[d] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < parts; i += kFly) {
    float m[kFly], l[kFly];
    v4u x[kFly][kMine];
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      const int part = min(i + k, parts - 1), from = part ? (w0 + part) * 2 : first;
      m[k] = GetStat(p, from, 0, c);
      l[k] = GetStat(p, from, 1, c);
#pragma unroll
      for (int d = 0; d < kMine; ++d)
        x[k][d] = __builtin_amdgcn_raw_buffer_load_b128(Rsrc(p.part), ((from * DT + d * kWaves + wave) * 64 + lane) * 16, 0,
                                                        kDeviceScope);
    }
    __builtin_amdgcn_sched_barrier(0);
    float now = mo;
#pragma unroll
    for (int k = 0; k < kFly; ++k) now = fmaxf(now, m[k]);
    const float keep = __builtin_amdgcn_exp2f(mo - now);
    mo = now;
    sum *= keep;
#pragma unroll
    for (int d = 0; d < kMine; ++d) a[d] *= keep;
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (i + k >= parts) break;
      const float by = __builtin_amdgcn_exp2f(m[k] - now);
      sum += l[k] * by;
#pragma unroll
      for (int d = 0; d < kMine; ++d) a[d] += __builtin_bit_cast(v4f, x[k][d]) * by;
    }
  }
#pragma unroll
  for (int d = 0; d < kMine; ++d) StoreRows(p, j, d * kWaves + wave, a[d], sum);
}

template <int HD, bool FP8, bool EXACT>
__global__ __launch_bounds__(kThreads, HD == 256 ? 1 : 2) void KvDecodeKernel(const Plan p) {
  constexpr int DT = HD / 16, CH = HD / 64;  // dimension tiles, 64-byte chunks of a key
  __shared__ Line line;
  __shared__ v4f so[kWaves][DT][64];
  __shared__ float sm[kWaves][2][16];
  __shared__ unsigned before;
  const KvCacheParams &cp = p.a.c;
  const int tid = threadIdx.x, lane = tid % 64, c = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const bool small = cp.batch <= 64;
  Lanes lanes;
  if (!small && p.fill) FillInvalid(p);
  const int64_t units = small ? MakeLanes(p, lanes) : MakeLine(p, line), piece = PieceOf(units);
  int64_t u = (int64_t)blockIdx.x * piece;
  const int64_t end = u + piece < units ? u + piece : units;
  for (int part = 0; u < end; part = 1) {
    const Job j = small ? FindJob(p, lanes, u) : FindJob(p, line, u);
    const int t0 = (int)(u - j.first), t1 = (int)(end - j.first < j.tiles ? end - j.first : j.tiles);
    const int row = j.row0 + c;
    const bool live = row < j.n * p.group;
    const int64_t token = j.start + (live ? row / p.group : 0);
    const int last = j.len - j.n + (live ? row / p.group : 0);  // the last token the row sees
    QRow<CH, EXACT> q;
    TileLoad<HD, EXACT> ld;
    q.Load(p.a, (token * p.a.heads + j.head * p.group + (live ? row % p.group : 0)) * cp.head_dim, live, g);
    // the first tile's loads start before Q is looked at
    int t = t0 + wave;
    if (t < t1) {
      ld.Lookup(cp, j, t, c, g);
      ld.LoadK(cp, j, t, c, g);
      ld.LoadV(cp);
      ld.Lookup(cp, j, t + kWaves, c, g);
    }
    q.Scale(p.a);
    const float qf = __builtin_amdgcn_ldexpf(fabsf(p.a.scale) * kLog2e, q.exponent);

    v4f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = v4f{0.f, 0.f, 0.f, 0.f};
    float mo = kNone, sum = 0.f;
    // One tile; with `more` the next one's keys load under its softmax and the
    // values under the next scores.  The last tile is a copy of its own: behind
    // a branch inside the loop every use would wait for all loads.
    auto tile = [&](auto more) __attribute__((always_inline)) {
      const int base = t * kTile, vt = base + 16 * g;
      v4f s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < CH; ++h) {
          s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Widen<FP8>(ld.k[i][h][0], ld.k[i][h][1]), q.q[h][0], s[i], 0, 0, 0);
          s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Widen<FP8>(ld.k[i][h][2], ld.k[i][h][3]), q.q[h][1], s[i], 0, 0, 0);
        }
      }
      const float cs = ld.ks * qf, lv = LogScale(ld.vs), inv = InvScale(ld.vs) * 0x1p-15f;
      const bool none = ld.ks != ld.ks;  // a row has a NaN score of these tokens, or does not see them
      if constexpr (more) ld.LoadK(cp, j, t + kWaves, c, g);
      // tokens that the row does not see, in the tiles that have any
      const bool edge = base + kTile > j.len - j.n + 1;
      float top = -__builtin_huge_valf();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = edge && vt + i > last ? -__builtin_huge_valf() : Weight(s[i / 4][i % 4], cs, lv);
        s[i / 4][i % 4] = x;
        top = fmaxf(top, x);
      }
      const float now = fmaxf(mo, GroupMax(top)), keep = __builtin_amdgcn_exp2f(mo - now);
      mo = now;
      float ps = 0.f;
      v8h pr[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float w = __builtin_amdgcn_exp2f((s[i / 4][i % 4] - now) + kTop);
        ps += w;
        pr[i / 8][i % 8] = (_Float16)w;
      }
      sum = __builtin_fmaf(ps, inv, sum * keep);
      if (edge || __any(none)) {
        // what the cache holds past the end, or in the block that stands for one
        // outside, may be any code, NaN among them, which a weight of 0 keeps
        const int left = none ? 0 : j.len - vt;  // tokens of this lane that are there
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int n = left - 4 * w;
          const unsigned mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
#pragma unroll
          for (int d = 0; d < DT; ++d) ld.v[d][w] &= (int)mask;
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        o[d] *= keep;
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Widen<FP8>(ld.v[d][0], ld.v[d][1]), pr[0], o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Widen<FP8>(ld.v[d][2], ld.v[d][3]), pr[1], o[d], 0, 0, 0);
      }
      if constexpr (more) {
        ld.LoadV(cp);
        ld.Lookup(cp, j, t + 2 * kWaves, c, g);
      }
      t += kWaves;
    };
    while (t + kWaves < t1) tile(std::true_type{});
    if (t < t1) tile(std::false_type{});
    sum = GroupSum(sum);

    // the waves' parts become one
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) so[wave][d][lane] = o[d];
    if (g == 0) {
      sm[wave][0][c] = mo;
      sm[wave][1][c] = sum;
    }
    __syncthreads();
    float f[kWaves];
    mo = JoinWaves(sm, c, f, sum);
    const bool whole = t0 == 0 && t1 == j.tiles;
    const int slot = (int)blockIdx.x * 2 + part;
    for (int d = wave; d < DT; d += kWaves) {
      const v4f a = WaveSum(so, f, d, lane);
      if (whole)
        StoreRows(p, j, d, a, sum);
      else if (live)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, a), Rsrc(p.part), ((slot * DT + d) * 64 + lane) * 16,
                                               0, kDeviceScope);
    }
    if (!whole) {
      if (wave == 0 && g == 0) {
        PutStat(p, slot, 0, c, mo);
        PutStat(p, slot, 1, c, sum);
      }
      const int w0 = Uniform((int)(j.first / piece)), w1 = Uniform((int)((j.first + j.tiles - 1) / piece));
      // this part is in memory for every XCD before it is counted
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0) before = atomicAdd(p.done + w0, 1u);
      __syncthreads();
      if (before == (unsigned)(w1 - w0)) {
        if (tid == 0) p.done[w0] = 0;
        // a job that starts inside a piece is the last in it
        JoinParts<HD>(p, j, w0, w1, w0 * 2 + (j.first > w0 * piece ? 1 : 0));
      }
    }
    u = j.first + t1;
  }
}

// ---------------------------------------------------------------------------
// Many rows (prompts): the products are the cost.  A job is one kv head and a
// tile of 8 waves * W rows of a sequence, over the tokens that its last row sees;
// each wave owns its W rows, so nothing is joined between waves.  The products
// are W x W (Mfma below), W = 32; 16 for head dimensions above 128, whose O would
// not fit the registers otherwise.  A lane then holds a quarter or half of the
// tile's tokens of one row, in a row: 16 or 32 of them, one or two scales.
//
// The codes of a 64-token tile become fp16 once, in LDS (two buffers), where
// every wave reads them.  A SIMD has two waves; what a wave does for a tile takes
// about as long on the vector unit (softmax, widening, addresses) as on the
// matrix unit, and a wave alone cannot overlap the two, so one half of the waves
// multiplies while the other is at its softmax (the slots below).  The waves that
// multiply go first (s_setprio): without it the older half's softmax delays the
// younger half's products, and 32 heads of 128 over two prompts of 4096 new
// tokens, 8192 in all, take 649 us, not 617.
//
// Jobs form a line of tiles as above (kv heads outermost), cut into equal pieces,
// so the causal triangle, ragged lengths and few rows over long caches all keep
// every CU busy; parts are joined the same way.  Workgroups of one XCD take
// neighbouring pieces: the keys and values that they share stay in its L2, 617 ->
// 586 us (930 TFLOP/s; a wave's part of a tile 5400 -> 4300 clocks, and the clock
// gave way to power from 2.4 to 2.05 GHz).  With the 16 x 16 products for 128
// dimensions the issue slots that MFMAs take from the vector unit double.  Registers
// are full: head dimensions above 64 other than 128 and 256, which look at every
// dimension's end, keep up to 10 of them in memory.
//
// The reference mo moves only when it is exceeded by 2^kLag or more, which is left
// free below kTop.

// Q of one row for the prompt kernel: lane group g of G holds the dimensions
// 8 (G k + g) + (0..7) at q[k], scaled to [1, 2); qf gives the scores in powers of two,
// and is not negative (the sign of the softmax scale goes to Q).
template <int G, int KS, bool EXACT>
__device__ __forceinline__ void LoadQ(const KvAttentionParams &p, int64_t at, bool live, int g, v8h (&q)[KS], float &qf) {
  float v[KS][8], top = 0.f;
  v4i raw[KS];  // all loads first; `at` is a row that is there also where live is not set
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int d = 8 * (G * k + g);
    raw[k] = Load16(static_cast<const uint16_t *>(p.q) + at + (EXACT || d < p.c.head_dim ? d : 0));
  }
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const bool here = live && (EXACT || 8 * (G * k + g) < p.c.head_dim);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int w = here ? raw[k][i / 2] : 0;
      const uint16_t u = (uint16_t)((unsigned)w >> (16 * (i % 2)));
      v[k][i] = p.bf16 ? Bf16ToF32(u) : F16ToF32(u);
      top = fmaxf(top, fabsf(v[k][i]));
    }
  }
  top = GroupMax<G>(top);
  const int e = top > 0.f && top < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __builtin_amdgcn_ldexpf(v[k][i], -e);
      q[k][i] = (_Float16)(p.scale < 0.f ? -x : x);
    }
  qf = __builtin_amdgcn_ldexpf(fabsf(p.scale) * kLog2e, e);
}

constexpr int kRowWaves = 8, kRowThreads = 64 * kRowWaves;
constexpr float kLag = 2.f;  // 4 and 8 measure the same and leave less of fp16 to the small weights

struct RowLine {                // over the row tiles of all sequences
  int64_t upto[kRowThreads];    // units before the end of every thread's share
  int tiles_upto[kRowThreads];  // row tiles before the end of every thread's share of the sequences
  int row_tiles;
};

__device__ __forceinline__ int64_t BlockScan(int64_t v, int64_t *s) {
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t w = __shfl_up(v, o);
    if ((int)threadIdx.x % 64 >= o) v += w;
  }
  s[threadIdx.x] = v;
  __syncthreads();
  int64_t before = 0;
  for (int w = 0; w < (int)threadIdx.x / 64; ++w) before += s[64 * w + 63];
  __syncthreads();
  return v + before;
}

struct RowTile {
  int b, n, len, row0, tiles, start;
};

// Row tiles of sequence b (0 where its rows are the decoding kernel's).
__device__ __forceinline__ int RowTilesOf(const Plan &p, int b, int rows) {
  const int n = KvNewTokens(p.a.c, b);
  return n > 0 && (int64_t)n * p.group > p.rows_max ? (n * p.group + rows - 1) / rows : 0;
}

// Tiles of the cache that some row from row0 on sees.
__device__ __forceinline__ int TilesOf(const Plan &p, int len, int n, int row0, int rows) {
  const int last_row = min(row0 + rows, n * p.group) - 1;
  return (len - n + last_row / p.group) / kTile + 1;
}

// Row tile i of the batch; the longest of a sequence come first.
__device__ __forceinline__ RowTile FindRowTile(const Plan &p, const RowLine &l, int i, int rows) {
  const int share = (p.a.c.batch + kRowThreads - 1) / kRowThreads;
  int lo = 0, hi = kRowThreads - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (l.tiles_upto[mid] > i) hi = mid; else lo = mid + 1;
  }
  int at = lo ? l.tiles_upto[lo - 1] : 0, b = lo * share, n = RowTilesOf(p, b, rows);
  while (i >= at + n) {
    at += n;
    n = RowTilesOf(p, ++b, rows);
  }
  RowTile r;
  r.b = b;
  r.n = KvNewTokens(p.a.c, b);
  r.len = p.a.c.lengths[b];
  r.start = p.a.c.start[b];
  r.row0 = (n - 1 - (i - at)) * rows;
  r.tiles = TilesOf(p, r.len, r.n, r.row0, rows);
  return r;
}

__device__ __forceinline__ int64_t MakeRowLine(const Plan &p, RowLine &l, int rows) {
  const int B = p.a.c.batch, tid = threadIdx.x, share = (B + kRowThreads - 1) / kRowThreads;
  int64_t mine = 0;
  for (int b = tid * share; b < min(B, (tid + 1) * share); ++b) mine += RowTilesOf(p, b, rows);
  l.tiles_upto[tid] = (int)BlockScan(mine, l.upto);
  __syncthreads();
  const int all = l.tiles_upto[kRowThreads - 1], per = (all + kRowThreads - 1) / kRowThreads;
  mine = 0;
  for (int i = tid * per; i < min(all, (tid + 1) * per); ++i)
    mine += FindRowTile(p, l, i, rows).tiles;
  const int64_t sum = BlockScan(mine, l.upto);
  l.upto[tid] = sum;
  if (tid == 0) l.row_tiles = all;
  __syncthreads();
  return Uniform(l.upto[kRowThreads - 1]);
}

struct RowJob : Job {
  int i;  // its row tile
};
__device__ __forceinline__ void Take(RowJob &j, const RowTile &r) {
  j.b = Uniform(r.b);
  j.n = Uniform(r.n);
  j.len = Uniform(r.len);
  j.row0 = Uniform(r.row0);
  j.tiles = Uniform(r.tiles);
  j.start = Uniform(r.start);
}

// The job of unit u; `head` units are the row tiles of one kv head.
__device__ __forceinline__ RowJob FindRowJob(const Plan &p, const RowLine &l, int64_t u, int64_t head, int rows) {
  const int per = (l.row_tiles + kRowThreads - 1) / kRowThreads;
  RowJob j;
  j.head = Uniform((int)(u / head));
  const int64_t in_head = u - j.head * head;
  int lo = 0, hi = kRowThreads - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (l.upto[mid] > in_head) hi = mid; else lo = mid + 1;
  }
  int64_t at = lo ? l.upto[lo - 1] : 0;
  int i = lo * per;
  RowTile r = FindRowTile(p, l, i, rows);
  while (in_head >= at + r.tiles) {
    at += r.tiles;
    r = FindRowTile(p, l, ++i, rows);
  }
  Take(j, r);
  j.i = Uniform(i);
  j.first = j.head * head + Uniform(at);
  return j;
}
// The job after j.
__device__ __forceinline__ void NextRowJob(const Plan &p, const RowLine &l, RowJob &j, int rows) {
  j.first += j.tiles;
  ++j.i;
  if (j.row0 > 0) {
    j.row0 -= rows;
    j.tiles = TilesOf(p, j.len, j.n, j.row0, rows);
    return;
  }
  if (j.i == l.row_tiles) {
    j.i = 0;
    ++j.head;
  }
  Take(j, FindRowTile(p, l, j.i, rows));
}

// The 16-byte chunk of a row in LDS: keys have HD / 8 chunks per token, values
// 8 per dimension.
// They are exchanged so that the lanes that read at one time, any 16 in a row or
// the quads 0, 3, 5, 6 and 1, 2, 4, 7 of 32 (operands of W rows), take all banks.
template <int HD, int W> __device__ __forceinline__ int KeyChunk(int token, int chunk) {
  const int high = W == 32 ? (token >> 5 & 1) | (token >> 1 & 2) : token >> 4;
  const int key = HD == 64 ? (token >> 1 & 1) | high << 1 : (token & 3) | high << 2;
  return token * (HD / 8) + (chunk ^ key);
}
template <int W> __device__ __forceinline__ int ValueChunk(int dim, int chunk) {
  const int key = W == 32 ? dim >> 1 & 7 : (dim >> 1 & 1) | (dim >> 2 & 2) | ((dim >> 1 ^ dim) & 4);
  return dim * 8 + (chunk ^ key);
}

// The loads of a tile's codes by a workgroup, every thread 16 bytes (HD 256: two
// times).  A block of the cache has fewer than 2^32 bytes.  With `at` the place
// of the tile's first token in its block (zero for blocks of less than a tile),
// a thread's place is that plus a constant.

// Keys: the tokens of a wave's load lie in one block, so that its address is
// scalar and the thread's part is 32 bits.
template <int HD, int W, bool FP8, bool EXACT> struct KeyStage {
  static constexpr int kChunks = HD / 16, kEach = (kChunks * kTile + kRowThreads - 1) / kRowThreads;
  int blk[kEach];
  v4i r[kEach];
  unsigned off;  // from the tile's first token to this thread's bytes, in the block
  bool live;     // this thread's dimensions are there

  __device__ __forceinline__ static int Token(int e) { return (int)(threadIdx.x + e * kRowThreads) / kChunks % kTile; }
  __device__ __forceinline__ void Start(const KvCacheParams &p) {
    const int dim = (int)threadIdx.x % kChunks * 16;
    live = EXACT || dim < p.head_dim;
    off = (unsigned)((Token(0) & (p.block_tokens - 1)) * p.head_dim + (live ? dim : 0));
  }
  __device__ __forceinline__ void Lookup(const KvCacheParams &p, const int32_t *table, int last, int t) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) blk[e] = table[min(t * kTile + Uniform(Token(e)), last) >> p.block_shift];
  }
  __device__ __forceinline__ void Load(const KvCacheParams &p, const uint8_t *head, unsigned stride, unsigned blocks, int t) {
    const int bt = p.block_tokens;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const unsigned u = (unsigned)Uniform(blk[e]);
      const int at = ((t * kTile) & (bt - 1)) + ((e * kRowThreads / kChunks) & (bt - 1));
      const uint8_t *base = head + (uint64_t)(u < blocks ? u : 0) * stride + at * p.head_dim;
      r[e] = *reinterpret_cast<const v4i *>(base + off);
      if (!EXACT && !live) r[e] = v4i{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void Store(char *lds) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (kChunks * kTile < kRowThreads && threadIdx.x >= kChunks * kTile) continue;
      const unsigned at = KeyChunk<HD, W>(Token(e), (int)threadIdx.x % kChunks * 2) * 16;
      *reinterpret_cast<v8h *>(lds + at) = Widen<FP8>(r[e][0], r[e][1]);
      *reinterpret_cast<v8h *>(lds + (at ^ 16)) = Widen<FP8>(r[e][2], r[e][3]);
    }
  }
};

// Values: four lanes take the 64 tokens of a dimension.
template <int HD, int W, bool FP8, bool EXACT> struct ValueStage {
  static constexpr int kEach = (HD * 4 + kRowThreads - 1) / kRowThreads;
  int blk;
  v4i r[kEach];
  const uint8_t *base;  // this thread's bytes of the tile's first tokens in block 0
  bool live[kEach];
  bool bad;  // the codes in r stand for those of a block outside the cache

  __device__ __forceinline__ static int Token() { return 16 * (threadIdx.x % 4); }
  __device__ __forceinline__ static int Dim(int e) { return (int)(threadIdx.x + e * kRowThreads) / 4 % HD; }
  __device__ __forceinline__ void Start(const KvCacheParams &p, const uint8_t *head) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) live[e] = EXACT || Dim(e) < p.head_dim;
    base = head + (live[0] ? Dim(0) * p.block_tokens : 0) + (Token() & (p.block_tokens - 1));
  }
  __device__ __forceinline__ void Lookup(const KvCacheParams &p, const int32_t *table, int last, int t) {
    blk = table[(unsigned)min(t * kTile + Token(), last) >> p.block_shift];
  }
  __device__ __forceinline__ void Load(const KvCacheParams &p, unsigned stride, unsigned blocks, int t) {
    bad = (unsigned)blk >= blocks;
    const unsigned u = bad ? 0u : (unsigned)blk;
    const uint8_t *at = base + ((t * kTile) & (p.block_tokens - 1)) + (uint64_t)u * stride;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const bool here = EXACT || live[e];
      r[e] = here ? *reinterpret_cast<const v4i *>(at + e * kRowThreads / 4 * p.block_tokens) : v4i{0, 0, 0, 0};
    }
  }
  // Codes past the sequence's end (`left` tokens of the tile are there) or of a
  // block outside the cache may be any, NaN among them: as the second product
  // multiplies them by zero in rows that do not see them, they become zero.
  __device__ __forceinline__ void Store(char *lds, int left) {
    if (left < kTile || __any(bad)) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = (bad ? 0 : left) - Token() - 4 * w;
        const int mask = (int)(n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u);
#pragma unroll
        for (int e = 0; e < kEach; ++e) r[e][w] &= mask;
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (HD * 4 < kRowThreads && threadIdx.x >= HD * 4) continue;
      const unsigned at = ValueChunk<W>(Dim(e), (int)threadIdx.x % 4 * 2) * 16;
      *reinterpret_cast<v8h *>(lds + at) = Widen<FP8>(r[e][0], r[e][1]);
      *reinterpret_cast<v8h *>(lds + (at ^ 16)) = Widen<FP8>(r[e][2], r[e][3]);
    }
  }
};

// Both scales of a lane group's tokens, 16 at a time, a tile ahead, and their
// block two ahead.  A block outside the cache gives a NaN score.
template <int G> struct ScaleStage {
  static constexpr int kEach = 4 / G;
  int blk[kEach];
  bool bad[kEach];
  float ks[kEach], vs[kEach];
  __device__ __forceinline__ void Lookup(const KvCacheParams &p, const int32_t *table, int last, int t, int g) {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      blk[e] = table[(unsigned)min(t * kTile + 16 * (kEach * g + e), last) >> p.block_shift];
  }
  __device__ __forceinline__ void Load(const KvCacheParams &p, int head, unsigned blocks) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      bad[e] = (unsigned)blk[e] >= blocks;
      const uint64_t at = (uint64_t)(bad[e] ? 0u : (unsigned)blk[e]) * (unsigned)p.kv_heads + (unsigned)head;
      ks[e] = p.k_scale[at];
      vs[e] = p.v_scale[at];
    }
  }
};

// The products of W x W results: lane W h + r of G = 64 / W groups has operand
// row r at 8 h of the 8 G long sum, and of the results column r, rows
// 4 G (e / 4) + 4 h + e % 4.
template <int W> struct Mfma;
template <> struct Mfma<16> {
  typedef v4f Acc;
  static __device__ __forceinline__ Acc Do(v8h a, v8h b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma<32> {
  typedef float Acc __attribute__((ext_vector_type(16)));
  static __device__ __forceinline__ Acc Do(v8h a, v8h b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

constexpr int kAhead = 4;  // 6 and 8 want registers that are not there

// Tiles that a workgroup takes at least.  Pieces of 4 | 8 | 16 tiles, us, 8 kv heads
// of 128, rows over tokens: one sequence 256 over 8192 69 | 56 | 63, 512 over 8192
// 65 | 65 | 71, 256 over 2048 38 | 41 | 50; two 256 over 4096 49 | 48 | 58.  From
// 1024 rows on pieces are longer by themselves.  The parts of a job, 128 KB each,
// are joined by one CU, at about 75 GB/s.
constexpr int kLeastPiece = 8;

// LDS writes and reads of this wave are done; so for all waves.  Loads stay in
// flight.
__device__ __forceinline__ void SlotBarrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int HD, int W, bool FP8, bool EXACT>
__global__ __launch_bounds__(kRowThreads, 1) void KvPromptKernel(const Plan p) {
  typedef Mfma<W> M;
  typedef typename M::Acc Acc;
  constexpr int G = 64 / W, E = W * W / 64, kRows = kRowWaves * W;
  constexpr int DT = HD / W, KS = HD / (8 * G);       // results of O^T, steps of S^T
  constexpr int NI = kTile / W, KK = kTile / (8 * G); // results of S^T, steps of O^T
  constexpr int kOwn = kTile / G;                     // a lane's consecutive tokens of a tile
  constexpr unsigned kBuffer = kTile * HD * 2, kValues = 2 * kBuffer;  // two buffers of keys, two of values
  __shared__ __align__(16) char lds[4 * kBuffer];
  __shared__ RowLine line;
  __shared__ unsigned before;
  const KvCacheParams &cp = p.a.c;
  const int tid = threadIdx.x, lane = tid % 64, c = lane % W, g = lane / W;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const bool late = wave >= kRowWaves / 2;  // the half of the waves that runs a slot behind
  if (p.fill) FillInvalid(p);
  const int64_t head_units = MakeRowLine(p, line, kRows), units = head_units * cp.kv_heads;
  const int64_t piece = max((units + gridDim.x - 1) / gridDim.x, (int64_t)kLeastPiece);
  // the workgroups of one XCD (every eighth) take pieces in a row, so that they
  // share few heads' keys and values in its L2
  const int me = gridDim.x % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
  int64_t u = (int64_t)me * piece;
  const int64_t end = u + piece < units ? u + piece : units;
  RowJob j;
  for (int part = 0; u < end; part = 1) {
    if (part == 0)
      j = FindRowJob(p, line, u, head_units, kRows);
    else
      NextRowJob(p, line, j, kRows);
    const int t0 = (int)(u - j.first), t1 = (int)(end - j.first < j.tiles ? end - j.first : j.tiles);
    const int wrow = j.row0 + wave * W, rows = j.n * p.group, before_new = j.len - j.n;
    const int32_t *table = cp.table + (int64_t)j.b * cp.max_blocks;
    const unsigned stride = (unsigned)cp.kv_heads * (unsigned)(cp.block_tokens * cp.head_dim);
    const unsigned blocks = (unsigned)(cp.num_blocks < INT64_C(0x80000000) ? cp.num_blocks : INT64_C(0x80000000));
    const uint64_t head = (uint64_t)j.head * (unsigned)(cp.block_tokens * cp.head_dim);
    KeyStage<HD, W, FP8, EXACT> keys;
    ValueStage<HD, W, FP8, EXACT> values;
    ScaleStage<G> scales;
    keys.Start(cp);
    values.Start(cp, cp.v_cache + head);
    keys.Lookup(cp, table, j.len - 1, t0);
    values.Lookup(cp, table, j.len - 1, t0);
    scales.Lookup(cp, table, j.len - 1, t0, g);
    keys.Load(cp, cp.k_cache + head, stride, blocks, t0);
    keys.Lookup(cp, table, j.len - 1, t0 + 1);
    scales.Load(cp, j.head, blocks);
    scales.Lookup(cp, table, j.len - 1, t0 + 1, g);
    v8h q[KS];
    float qf;
    int last;  // the last token that the row sees
    {
      const int row = wrow + c, token = row < rows ? row / p.group : 0;
      const int64_t at = ((j.start + (int64_t)token) * p.a.heads + j.head * p.group + row % p.group) * cp.head_dim;
      last = before_new + token;
      LoadQ<G, KS, EXACT>(p.a, at, row < rows, g, q, qf);
    }
    __syncthreads();  // the buffers of the job before were read
    keys.Store(lds);
    keys.Load(cp, cp.k_cache + head, stride, blocks, t0 + 1);
    keys.Lookup(cp, table, j.len - 1, t0 + 2);
    values.Load(cp, stride, blocks, t0);
    values.Lookup(cp, table, j.len - 1, t0 + 1);
    Acc o[DT], s[NI];
    v8h pr[KK];
    float mo = kNone, sum = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = Acc(0.f);
    // the tokens that every row of the wave sees end here
    const int all_see = before_new + min(wrow, rows - 1) / p.group + 1;
    // this lane's first operands; those of the other steps are an exclusive or away
    const unsigned my_keys = KeyChunk<HD, W>(kOwn * (c / 4 % G) + c / (4 * G) * 4 + c % 4, g) * 16;
    const unsigned my_values = ValueChunk<W>(c, 8 / G * g) * 16;
    // The products of a slot: values of tile t - 1 (V), then keys of tile t (K).  A
    // product is shorter than the read of its operand from LDS takes: kAhead
    // reads are in flight.  With K also the staging of keys t + 1 and values t, and
    // the loads of a tile further; past the job's last tile that writes a buffer
    // that nobody reads again.
    auto multiply = [&](auto V, auto K, int t) __attribute__((always_inline)) {
      constexpr int kV = decltype(V)::value ? DT * KK : 0, kN = kV + (decltype(K)::value ? NI * KS : 0);
      auto read = [&](int n) __attribute__((always_inline)) {
        const int m = n - kV;
        const unsigned at = n < kV ? (my_values ^ (((t - 1 - t0) & 1) * kBuffer | n / DT * 16)) + kValues + W * 128 * (n % DT)
                                   : (my_keys ^ (((t - t0) & 1) * kBuffer | m / NI * (16 * G))) + 2 * HD * E * (m % NI);
        return *reinterpret_cast<const v8h *>(lds + at);
      };
      v8h a[kN];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) a[n] = read(n);
      auto products = [&](auto from, auto to) __attribute__((always_inline)) {
#pragma unroll
        for (int n = decltype(from)::value; n < decltype(to)::value; ++n) {
          if (n + kAhead < kN) a[n + kAhead] = read(n + kAhead);
          const int m = n - kV;
          if (n < kV)
            o[n % DT] = M::Do(a[n], pr[n / DT], o[n % DT]);
          else
            s[m % NI] = M::Do(a[n], q[m / NI], m / NI ? s[m % NI] : Acc(0.f));
          __builtin_amdgcn_sched_barrier(0);  // or all reads go first, into registers that are not there
        }
      };
      const std::integral_constant<int, 0> at0;
      const std::integral_constant<int, kN / 8> at1;
      const std::integral_constant<int, kN / 2> at2;
      const std::integral_constant<int, kN> at3;
      products(at0, at1);
      if (K) {
        keys.Store(lds + ((t + 1 - t0) & 1) * kBuffer);
        keys.Load(cp, cp.k_cache + head, stride, blocks, t + 2);
        keys.Lookup(cp, table, j.len - 1, t + 3);
      }
      products(at1, at2);
      if (K) {
        values.Store(lds + kValues + ((t - t0) & 1) * kBuffer, j.len - t * kTile);
        values.Load(cp, stride, blocks, t + 1);
        values.Lookup(cp, table, j.len - 1, t + 2);
      }
      products(at2, at3);
    };
    // Value n of a lane is token kOwn * g + n of the tile.
    auto softmax = [&](int t) __attribute__((always_inline)) {
      constexpr int NS = kOwn / 16;  // scales
      float lv[NS], inv[NS], cs[NS];
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        lv[e] = LogScale(scales.vs[e]);
        inv[e] = InvScale(scales.vs[e]) * 0x1p-13f;
        cs[e] = (scales.bad[e] ? __builtin_nanf("") : scales.ks[e]) * qf;
      }
      scales.Load(cp, j.head, blocks);
      scales.Lookup(cp, table, j.len - 1, t + 2, g);
      const bool edge = t * kTile + kTile > all_see;
      const int seen = last - t * kTile - kOwn * g;  // the row sees the lane's tokens 0 .. seen
      float top[NS], best = kNone;
      if (edge) {
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          top[e] = -__builtin_huge_valf();
#pragma unroll
          for (int n = 16 * e; n < 16 * e + 16; ++n) top[e] = n <= seen ? fmaxf(top[e], s[n / E][n % E]) : top[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          top[e] = s[16 * e / E][0];
#pragma unroll
          for (int n = 16 * e + 1; n < 16 * e + 16; ++n) top[e] = fmaxf(top[e], s[n / E][n % E]);
        }
      }
#pragma unroll
      for (int e = 0; e < NS; ++e) best = fmaxf(best, Weight(top[e], cs[e], lv[e]));
      best = GroupMax<G>(best);
      if (__any(best > mo + kLag)) {
        const float now = fmaxf(mo, best), keep = __builtin_amdgcn_exp2f(mo - now);
        mo = now;
        sum *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= keep;
      }
      // one fused step rounds otherwise than mo was made, by an ulp of mo: from
      // 2^12 on that is left to the exact difference
      if (edge || __any(fabsf(mo) > 4096.f && mo > kNone)) {
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
          const float z = (Weight(s[n / E][n % E], cs[n / 16], lv[n / 16]) - mo) + (kTop - kLag);
          s[n / E][n % E] = n > seen ? -__builtin_huge_valf() : z;
        }
      } else {
#pragma unroll
        for (int n = 0; n < kOwn; ++n)
          s[n / E][n % E] = __builtin_fmaf(s[n / E][n % E], cs[n / 16], (lv[n / 16] - mo) + (kTop - kLag));
      }
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        float ps = 0.f;
#pragma unroll
        for (int n = 16 * e; n < 16 * e + 16; ++n) {
          const float w = __builtin_amdgcn_exp2f(s[n / E][n % E]);
          ps += w;
          pr[n / 8][n % 8] = (_Float16)w;
        }
        sum = __builtin_fmaf(ps, inv[e], sum);
      }
    };
    // Slots: one half of the waves multiplies and stages while the other is at its
    // softmax; then they change places.  In the two slots that multiply values of
    // tile t - 1 and keys of tile t, keys t + 1 and values t are written, each into
    // the other buffer, which the slots before have read.
    const std::true_type yes;
    const std::false_type no;
    SlotBarrier();
    if (late) SlotBarrier();
    multiply(no, yes, t0);
    SlotBarrier();
    for (int t = t0; t < t1 - 1; ++t) {
      softmax(t);
      SlotBarrier();
      __builtin_amdgcn_s_setprio(1);  // or the older half's softmax holds up the younger's products
      multiply(yes, yes, t + 1);
      __builtin_amdgcn_s_setprio(0);
      SlotBarrier();
    }
    softmax(t1 - 1);
    SlotBarrier();
    multiply(yes, no, t1);
    if (!late) SlotBarrier();
    sum = GroupSum<G>(sum);
    // The wave's results as parts: quads of dimensions, and both statistics of its
    // rows by tiles of 16.
    const bool whole = t0 == 0 && t1 == j.tiles;
    const int slot = me * 2 + part;
    constexpr int kQuads = DT * E / 4;
    const bool alive = wrow < rows;  // the wave has a row
    if (!whole) {
      const int at = slot * kRowWaves + wave;
      if (alive) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            const v4f x{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, x), Rsrc(p.part),
                                                   ((at * kQuads + (d * E + e) / 4) * 64 + lane) * 16, 0, kDeviceScope);
          }
        if (g == 0) {
          PutStat(p, at * (W / 16) + c / 16, 0, c % 16, mo);
          PutStat(p, at * (W / 16) + c / 16, 1, c % 16, sum);
        }
      }
      const int w0 = Uniform((int)(j.first / piece)), w1 = Uniform((int)((j.first + j.tiles - 1) / piece));
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0) before = atomicAdd(p.done + w0, 1u);
      __syncthreads();
      if (before != (unsigned)(w1 - w0)) {
        u = j.first + t1;
        continue;
      }
      if (tid == 0) p.done[w0] = 0;
      const int first = w0 * 2 + (j.first > w0 * piece ? 1 : 0);
      mo = kNone;
      sum = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] = Acc(0.f);
      auto part_of = [&](int w) { return (w == w0 ? first : w * 2) * kRowWaves + wave; };
      for (int w = w0; alive && w <= w1; w += 8) {  // eight loads on their way at once
        float m[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = GetStat(p, part_of(min(w + i, w1)) * (W / 16) + c / 16, 0, c % 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) mo = fmaxf(mo, m[i]);
      }
      for (int w = w0; alive && w <= w1; ++w) {
        const int from = part_of(w);
        const float f = GetStat(p, from * (W / 16) + c / 16, 0, c % 16), l = GetStat(p, from * (W / 16) + c / 16, 1, c % 16);
        v4u x[kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
          x[i] = __builtin_amdgcn_raw_buffer_load_b128(Rsrc(p.part), ((from * kQuads + i) * 64 + lane) * 16, 0, kDeviceScope);
        __builtin_amdgcn_sched_barrier(0);  // all loads are on their way
        const float by = __builtin_amdgcn_exp2f(f - mo);
        sum += l * by;
#pragma unroll
        for (int i = 0; i < 4 * kQuads; ++i) o[i / E][i % E] += __builtin_bit_cast(v4f, x[i / 4])[i % 4] * by;
      }
    }
    if (wrow + c < rows) {
      uint16_t *out = OutRow(p, j, wrow + c);
      const float f = 0x1p-13f / sum;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < E; e += 4)
          StoreDims(p, out, W * d + G * e + 4 * g, v4f{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]} * f);
    }
    u = j.first + t1;
  }
}

int HeadTile(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Two workgroups per CU hold eight waves, enough loads in flight to fill the
// memory (head dimensions above 128 need the registers of both); never more
// than there can be pieces of one tile per wave.
int64_t DecodeGrid(const KvAttentionParams &p) {
  const KvCacheParams &c = p.c;
  const int64_t group = p.heads / c.kv_heads, jobs = (c.tokens * group / 16 + c.batch) * c.kv_heads;
  const int64_t tiles = ((int64_t)c.max_blocks * c.block_tokens + kTile - 1) / kTile;
  const int64_t pieces = (jobs * tiles + kWaves - 1) / kWaves;
  return std::max<int64_t>(1, std::min<int64_t>(pieces, (c.head_dim > 128 ? 1 : 2) * Ctx().num_cus));
}

template <int HD> void LaunchDecode(const Plan &p, int64_t grid, hipStream_t s) {
  const dim3 g((unsigned)grid);
  const bool exact = p.a.c.head_dim == HD;
  if (p.a.c.fp8)
    exact ? KvDecodeKernel<HD, true, true><<<g, kThreads, 0, s>>>(p) : KvDecodeKernel<HD, true, false><<<g, kThreads, 0, s>>>(p);
  else
    exact ? KvDecodeKernel<HD, false, true><<<g, kThreads, 0, s>>>(p) : KvDecodeKernel<HD, false, false><<<g, kThreads, 0, s>>>(p);
}

template <int HD, int W> void LaunchPrompt(const Plan &p, int64_t grid, hipStream_t s) {
  const dim3 g((unsigned)grid);
  const bool exact = p.a.c.head_dim == HD;
  if (p.a.c.fp8)
    exact ? KvPromptKernel<HD, W, true, true><<<g, kRowThreads, 0, s>>>(p)
          : KvPromptKernel<HD, W, true, false><<<g, kRowThreads, 0, s>>>(p);
  else
    exact ? KvPromptKernel<HD, W, false, true><<<g, kRowThreads, 0, s>>>(p)
          : KvPromptKernel<HD, W, false, false><<<g, kRowThreads, 0, s>>>(p);
}

// Sequences with at most so many rows (new tokens * heads of a group) take the
// decoding kernel, the others the prompt kernel; a launch that no sequence can
// need is left out.  Per sequence of 8192 tokens, 8 kv heads of 128 dimensions,
// decoding | prompt kernel: 8 sequences of 32 rows 45 | 73 us, of 64 rows 80 | 75,
// of 128 rows 149 | 81.  Where all rows of the batch are few the parts of a
// sequence are many, and the decoding kernel's are the smaller to join: one
// sequence of 64 rows 17 | 36 us, of 128 rows 21 | 40.  The line could lie higher:
// 256 rows in all are one sequence 31 | 56, two 32 | 41, four 31 | 46, and 512 in
// eight 80 | 75.
//
// Without max_query every sequence may be the long one: 64 sequences of a token
// with groups of 8 heads then pay the prompt kernel's launch, which finds nothing,
// 52 -> 56 us and 118 -> 122, 17 of them 18 -> 21; up to 128 rows in all nothing.
constexpr int kFewRows = 32, kFewInAll = 128;

struct Split {
  bool decode, prompt;
  int few;  // the most rows of a sequence for the decoding kernel
  int64_t decode_grid, prompt_grid;
};

int64_t PromptRows(const KvAttentionParams &p) { return kRowWaves * (p.c.head_dim > 128 ? 16 : 32); }

Split SplitOf(const KvAttentionParams &p) {
  const KvCacheParams &c = p.c;
  const int64_t group = p.heads / c.kv_heads;
  // the most and the least rows that a sequence may have
  const int64_t known = p.max_query > 0 && p.max_query < c.tokens ? p.max_query : c.tokens;
  const int64_t most = known * group;
  const int64_t least = c.tokens - (c.batch - 1) * known;
  Split s;
  s.few = c.tokens * group <= kFewInAll ? kFewInAll : kFewRows;
  s.prompt = c.batch > 0 && most > s.few;
  s.decode = !s.prompt || least * group <= s.few;
  s.decode_grid = DecodeGrid(p);
  const int64_t jobs = (c.tokens * group / PromptRows(p) + c.batch) * c.kv_heads;
  const int64_t tiles = ((int64_t)c.max_blocks * c.block_tokens + kTile - 1) / kTile;
  s.prompt_grid = std::max<int64_t>(1, std::min<int64_t>(jobs * tiles, Ctx().num_cus));
  return s;
}

}  // namespace

size_t KvAttentionScratchBytes(const KvAttentionParams &p) {
  const Split s = SplitOf(p);
  const size_t slots = 2 * std::max<size_t>(s.decode ? s.decode_grid * 16 : 0, s.prompt ? s.prompt_grid * PromptRows(p) : 0);
  return Scratch::Round(slots * HeadTile(p.c.head_dim) * sizeof(float)) + slots * 2 * sizeof(float);
}

void LaunchKvCacheAttention(const KvAttentionParams &a, void *scratch, hipStream_t stream) {
  const Split sp = SplitOf(a);
  const int hd = HeadTile(a.c.head_dim);
  const size_t slots = 2 * std::max<size_t>(sp.decode ? sp.decode_grid * 16 : 0, sp.prompt ? sp.prompt_grid * PromptRows(a) : 0);
  Plan p{};
  p.a = a;
  p.group = a.heads / a.c.kv_heads;
  // a launch that stands alone has every sequence, also where max_query was wrong
  p.rows_max = !sp.prompt ? 0x7fffffff : !sp.decode ? 0 : sp.few;
  p.fill = 1;
  p.done = Ctx().ws.Counters((size_t)std::max(sp.decode_grid, sp.prompt_grid));
  p.part = static_cast<float *>(scratch);
  p.stat = reinterpret_cast<float *>(static_cast<char *>(scratch) + Scratch::Round(slots * hd * sizeof(float)));
  if (sp.prompt) {
    if (hd == 64)
      LaunchPrompt<64, 32>(p, sp.prompt_grid, stream);
    else if (hd == 128)
      LaunchPrompt<128, 32>(p, sp.prompt_grid, stream);
    else
      LaunchPrompt<256, 16>(p, sp.prompt_grid, stream);
    p.fill = 0;
  }
  if (sp.decode) {
    if (hd == 64)
      LaunchDecode<64>(p, sp.decode_grid, stream);
    else if (hd == 128)
      LaunchDecode<128>(p, sp.decode_grid, stream);
    else
      LaunchDecode<256>(p, sp.decode_grid, stream);
  }
}

}  // namespace onnxl_amd
