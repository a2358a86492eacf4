// Block-scaled product for few rows (decoding): y[M, N] = a[M, K] b[N, K]^T with
// the MXFP4 weight read once, straight into the operand registers of
// v_mfma_scale_f32_16x16x128_f8f6f4.
//
// The weight's bytes are the cost, so the k of the instruction is dealt out for
// their sake: of a chunk of 512 values (16 blocks of 32) lane group g = l / 16
// takes the blocks 4 g .. 4 g + 3 of row l % 16, 64 consecutive bytes, and block
// 4 g + j is its operand of the chunk's instruction j.  A chunk's 256 bytes of a
// row are two whole lines, and its 16 scales one dword per lane, whose byte j is
// selected by the instruction.  The activations follow the same order: E2M1
// codes like the weight's; for E4M3 the instruction wants of lane group g the
// half g % 2 of its blocks g / 2 and 2 + g / 2, which are the chunk's blocks
// 4 (g / 2) + j and 4 (2 + g / 2) + j.
//
// A workgroup has 16 NT rows of the weight; its waves take the chunks in turn
// and add up in LDS.  Where rows are few and K is long several workgroups share
// the chunks, so that all of a wave's loads are in flight at once; the last of
// them to finish adds up their sums, in the order of the chunks whoever that is.
// Activations of 16 bits that are few enough are quantized by every workgroup for
// itself, into LDS, while its first weight bytes are on their way: that costs less
// than a launch of its own.
//
// One row of 4096 values by [14336, 4096]: 29.4 MB of codes and 1.8 of scales in
// 9.8 us, 3.2 TB/s with the launch, which is a quarter of it.
//
// What the instruction does with E4M3 products is said at the GEMM (mx_gemm.hpp).
// With four row tiles and three of activations (E2M1, 33 to 48 rows) the registers
// of two waves per SIMD do not hold everything: 4 are kept in memory.
#pragma once

#include <type_traits>

#include "mx_gemm.hpp"
#include "quant8.hpp"

namespace onnxl_amd {
namespace mx {

struct StreamArgs {
  const void *x;                // [M, K] 16 bits, quantized here (QUANT); else
  const uint8_t *a, *as;        // codes [M, K] and scales [M, K / 32]
  const uint8_t *b, *bs;        // weight codes [N, K / 2] and scales [N, K / 32]
  uint16_t *y;
  int M, N, K;
  int x_bf16, bf16;
  int split;                    // workgroups (grid.y) that share the chunks
  float *part;                  // their sums, [row tile][split][NT * MT][64] float4
  unsigned *done;               // [row tile] workgroups that are done, zero between launches
  int first;                    // row tile of the launch's first workgroup
};

// Four block scales from `at` (a multiple of 4) on of the row of `blocks` at
// base + row.  Those
// past the end are scales of other blocks of the row: their activations are
// zeros, and a NaN among them makes the row NaN anyhow.  Nothing is done with
// what is loaded, which would wait for it, but in the last chunk of rows that
// are not whole dwords: there the bytes come one by one, all at once.
__device__ __forceinline__ int Scales4(const uint8_t *base, unsigned row, int at, int blocks, bool tail) {
  int v;
  if (!tail || blocks % 4 == 0) {
    __builtin_memcpy(&v, base + (row + (unsigned)(at < blocks ? at : 0)), 4);
    return v;
  }
  unsigned b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = base[row + (unsigned)min(at + i, blocks - 1)];
  return (int)(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24);
}

// Waves of a workgroup: what the registers of more rows and columns leave.
template <int NT> constexpr int kStreamWaves = NT == 4 ? 4 : 8;

template <bool A4, int NT, int MT, bool QUANT>
__global__ __launch_bounds__((64 * kStreamWaves<NT>), 2) void StreamKernel(const StreamArgs p) {
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int blocks = p.K / 32, chunks = (blocks + 15) / 16;
  const int tile = p.first + (int)blockIdx.x, n0 = tile * 16 * NT;
  const int64_t pitch_b = p.K / 2, pitch_a = A4 ? p.K / 2 : p.K;

  // 32-bit offsets of this lane's rows (those past the last repeat it) from the
  // tile's first
  const uint8_t *tile_b = p.b + n0 * pitch_b, *tile_s = p.bs + (int64_t)n0 * blocks;
  unsigned row_b[NT], row_s[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const unsigned row = (unsigned)(min(n0 + 16 * n + c, p.N - 1) - n0);
    row_b[n] = row * (unsigned)pitch_b;
    row_s[n] = row * (unsigned)blocks;
  }
  typedef std::conditional_t<A4, v4i, v8i> Frag;
  v4i w[NT][4];
  int ws[NT];
  // blocks past the end are read as block 0: the activations there are zeros
  auto load = [&](int ch) __attribute__((always_inline)) {
    const int blk = 16 * ch + 4 * g;
    const bool tail = 16 * ch + 16 > blocks;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[n][j] = *reinterpret_cast<const v4i *>(tile_b + (row_b[n] + 16u * (unsigned)(blk + j < blocks ? blk + j : 0)));
      ws[n] = Scales4(tile_s, row_s[n], blk, blocks, tail);
    }
  };

  // codes in LDS: rows of whole chunks, then their scales
  const int lds_row = chunks * (A4 ? 256 : 512), lds_scale = chunks * 16;
  char *lds_s = lds + (QUANT ? p.M * lds_row : 0);
  const int per = (chunks + p.split - 1) / p.split, ch0 = blockIdx.y * per, ch1 = min(chunks, ch0 + per);
  if (ch0 + wave < ch1) load(ch0 + wave);
  if constexpr (QUANT) {
    // eight values a thread, four neighbours a block; past the row's end zero
    // codes of scale 1
    const int per_row = chunks * 64;
    for (int i = tid; i < p.M * per_row; i += blockDim.x) {
      const int row = i / per_row, k8 = i % per_row;
      float v[8];
      unsigned top = 0;
      const bool in = k8 * 8 < p.K;
      uint16_t u[8] = {};
      if (in) __builtin_memcpy(u, static_cast<const uint16_t *>(p.x) + (int64_t)row * p.K + k8 * 8, 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = p.x_bf16 ? __builtin_bit_cast(float, (unsigned)u[j] << 16) : (float)__builtin_bit_cast(_Float16, u[j]);
        top = max(top, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
      }
      top = max(top, (unsigned)__shfl_xor((int)top, 1));
      top = max(top, (unsigned)__shfl_xor((int)top, 2));
      const BlockScale s = MxScaleOf(__builtin_bit_cast(float, top), A4 ? 2 : 8);
      if constexpr (A4)
        *reinterpret_cast<unsigned *>(lds + row * lds_row + k8 * 4) = MxFp4Codes8(v, s);
      else
        *reinterpret_cast<uint2 *>(lds + row * lds_row + k8 * 8) = MxFp8Codes8(v, s);
      if (k8 % 4 == 0) lds_s[row * lds_scale + k8 / 4] = in ? (char)s.e8m0 : 127;
    }
    __syncthreads();
  }

  v4f acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = v4f{0.f, 0.f, 0.f, 0.f};
  // one chunk; `more` loads the wave's next one as soon as the registers are free
  auto chunk = [&](int ch, auto more) __attribute__((always_inline)) {
    const bool tail = 16 * ch + 16 > blocks;
    // activations of instruction j, a step ahead of their use
    Frag x[2][MT];
    int xs[MT];
    auto get = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Frag &f = x[j % 2][m];
        const int row = min(16 * m + c, p.M - 1);  // rows past the last repeat it
        if constexpr (QUANT && A4) {
          f = *reinterpret_cast<const v4i *>(lds + row * lds_row + (16 * ch + 4 * g + j) * 16);
        } else if constexpr (QUANT) {
          const char *xp = lds + row * lds_row + (16 * ch + 4 * (g >> 1) + j) * 32 + 16 * (g & 1);
          f = __builtin_shufflevector(*reinterpret_cast<const v4i *>(xp), *reinterpret_cast<const v4i *>(xp + 256), 0, 1, 2, 3,
                                      4, 5, 6, 7);
        } else if constexpr (A4) {
          const int blk = 16 * ch + 4 * g + j;
          f = *reinterpret_cast<const v4i *>(p.a + ((unsigned)row * (unsigned)pitch_a + 16u * (unsigned)(blk < blocks ? blk : 0)));
        } else {
          const int lo = 16 * ch + 4 * (g >> 1) + j, hi = lo + 8;
          const unsigned at = (unsigned)row * (unsigned)pitch_a + 16u * (g & 1);
          f = __builtin_shufflevector(*reinterpret_cast<const v4i *>(p.a + (at + 32u * (unsigned)(lo < blocks ? lo : 0))),
                                      *reinterpret_cast<const v4i *>(p.a + (at + 32u * (unsigned)(hi < blocks ? hi : 0))), 0, 1,
                                      2, 3, 4, 5, 6, 7);
        }
      }
    };
    // codes of blocks past the end become zeros
    auto cut = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (A4) {
          if (16 * ch + 4 * g + j >= blocks) x[j % 2][m] = v4i{0, 0, 0, 0};
        } else {
          const int lo = 16 * ch + 4 * (g >> 1) + j;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[j % 2][m][i] = lo + (i < 4 ? 0 : 8) < blocks ? x[j % 2][m][i] : 0;
        }
      }
    };
    auto mma = [&](auto j) __attribute__((always_inline)) {
      if (!QUANT && tail) cut(j);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[n][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(Operand(w[n][j]), Operand(x[j % 2][m]), acc[n][m], 4,
                                                                       A4 ? 4 : 0, j, ws[n], j, xs[m]);
    };
    get(0);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = min(16 * m + c, p.M - 1);
      if constexpr (QUANT)
        xs[m] = *reinterpret_cast<const int *>(lds_s + row * lds_scale + 16 * ch + 4 * g);
      else
        xs[m] = Scales4(p.as, (unsigned)row * (unsigned)blocks, 16 * ch + 4 * g, blocks, tail);
    }
    get(1);
    mma(std::integral_constant<int, 0>{});
    get(2);
    mma(std::integral_constant<int, 1>{});
    get(3);
    mma(std::integral_constant<int, 2>{});
    mma(std::integral_constant<int, 3>{});
    if constexpr (more) load(ch + waves);
  };
  int ch = ch0 + wave;
  for (; ch + waves < ch1; ch += waves) chunk(ch, std::true_type{});
  if (ch < ch1) chunk(ch, std::false_type{});

  // lane (c, g) of a tile has the columns 4 g .. 4 g + 3 of row c of y
  v4f *part = reinterpret_cast<v4f *>(lds);
  __syncthreads();  // the codes were read
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) part[((n * MT + m) * waves + wave) * 64 + lane] = acc[n][m];
  __syncthreads();
  constexpr int kScope = 16;  // sc1: past this XCD's L2, so that no fence is needed
  const __amdgpu_buffer_rsrc_t rs = Rsrc(p.part, 0x7fffffff);
  auto slot = [&](int s, int i) { return (int)(((tile * p.split + s) * (NT * MT) + i) * 64 + lane) * 16; };
  auto store = [&](int i, v4f s) {
    const int row = i % MT * 16 + c, col = n0 + i / MT * 16 + 4 * g;
    if (row >= p.M) return;
    uint16_t *y = p.y + (int64_t)row * p.N + col;
    uint16_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = Half(s[e], p.bf16);
    if (col + 4 <= p.N) {
      __builtin_memcpy(y, v, 8);
    } else {
      for (int e = 0; col + e < p.N; ++e) y[e] = v[e];
    }
  };
  for (int i = wave; i < NT * MT; i += waves) {
    v4f s = part[i * waves * 64 + lane];
    for (int v = 1; v < waves; ++v) s += part[(i * waves + v) * 64 + lane];
    if (p.split == 1)
      store(i, s);
    else
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, s), rs, slot(blockIdx.y, i), 0, kScope);
  }
  if (p.split == 1) return;
  __shared__ unsigned before;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this part is where every XCD sees it before it is counted
  __syncthreads();
  if (tid == 0) before = atomicAdd(p.done + tile, 1u);
  __syncthreads();
  if (before != (unsigned)p.split - 1) return;
  if (tid == 0) p.done[tile] = 0;
  // up to kParts parts of all of a wave's tiles are on their way at once: one
  // after the other the six of 33 x 11008 x 4099 take 5.3 us of the launch's 15
  constexpr int kParts = 6, kMine = (NT * MT + kStreamWaves<NT> - 1) / kStreamWaves<NT>;
  v4f sum[kMine];
#pragma unroll
  for (int t = 0; t < kMine; ++t) sum[t] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int v0 = 0; v0 < p.split; v0 += kParts) {
    v4u x[kMine][kParts];
#pragma unroll
    for (int t = 0; t < kMine; ++t)
#pragma unroll
      for (int v = 0; v < kParts; ++v)
        x[t][v] = __builtin_amdgcn_raw_buffer_load_b128(
            rs, slot(min(v0 + v, p.split - 1), min(wave + t * waves, NT * MT - 1)), 0, kScope);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int v = 0; v < kParts; ++v) {
      if (v0 + v >= p.split) break;
#pragma unroll
      for (int t = 0; t < kMine; ++t) sum[t] += __builtin_bit_cast(v4f, x[t][v]);
    }
  }
#pragma unroll
  for (int t = 0; t < kMine; ++t)
    if (wave + t * waves < NT * MT) store(wave + t * waves, sum[t]);
}

}  // namespace mx
}  // namespace onnxl_amd
