// Block-scaled GEMM for many rows: y[M, N] = a[M, K] b[N, K]^T with a MXFP4 or
// MXFP8 and b MXFP4, on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// Both operands are rows with consecutive k, which is how the instruction wants
// them: lane l holds row l % 32 and, with h = l / 32, for E2M1 the 32 values
// from 32 h (16 bytes), for E4M3 the 16 from 16 h and the 16 from 32 + 16 h; the
// E8M0 scale of k block h comes from the same lane, one byte of a register that
// the instruction selects.
//
// Workgroup: 4 waves (2 x 2), tile 64 MB x 64 NB outputs, each wave MB x NB
// blocks of 32 x 32.  A K step is 256 values: 128 bytes of an E2M1 row, 256 of
// an E4M3 row, two 16-byte chunks (four) per 64-value sub-step and lane.  Two
// stages in LDS, filled by direct loads (16 bytes a lane, nothing held in
// registers) while the other is multiplied; a row's chunks are XOR-swizzled by
// the row, so that a fragment read meets no bank twice.  Scales are read through
// LDS as well, from tiles that a first kernel wrote (ScaleTileAt): the four
// bytes of a lane's register are its blocks of the four sub-steps, so a step
// needs one dword per 32 rows and no byte shuffles.
//
// The fragments of a sub-step are read under the MFMAs of the one before; the
// step's only barrier stands in the middle of its last sub-step, whose
// fragments are in registers by then, so the stage just read is refilled and
// the next one's reads begin under the remaining MFMAs.  The refill goes out in
// thirds, in that sub-step and the next two: all at once it holds the MFMAs up in
// the address unit, later it comes too late (4096 x 8192 x 8192, operands' launch
// and all, MXFP4: at once 174 us, halves 163, thirds 157, quarters 165; MXFP8 256,
// 239, 233, 241).
//
// What bounds it: the matrix cores work half of the time.  A product takes 61 cycles
// of its SIMD where the instruction needs 32 (MXFP4, 4096 rows; with MXFP8 and 1000
// rows 175 and 64), since a step waits for loads that left half a step before, and
// the one wave of a SIMD has nothing else to do meanwhile.
//
// Sums are fp32, but not all of a product enters them: with E4M3 activations the
// instruction aligns 16 products of consecutive k to the largest of them and cuts
// what is below 2^-13 of it (2^-13 itself is kept, 2^-14 lost), so such a group may
// be off by 16 * 2^-13 of its largest product.  Products of E2M1 with E2M1 span
// less than that and lose nothing.  Nothing in the instruction turns this off; the
// alternative is to widen both operands to 16 bits, at half the rate or less.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "decoder.hpp"

namespace onnxl_amd {
namespace mx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

constexpr int kXcds = 8, kGroupM = 4;
constexpr unsigned kOob = 0x80000000u;

// Scale tiles: for 32 rows and 8 blocks (256 values) one dword per lane l of
// the MFMA operand: byte s is the scale of row l % 32, block 2 s + l / 32.
__host__ __device__ inline int64_t ScaleTileAt(int64_t row, int64_t block, int64_t steps) {
  return ((row / 32 * steps + block / 8) * 64 + (block % 2) * 32 + row % 32) * 4 + block % 8 / 2;
}
inline int64_t ScaleTileBytes(int64_t rows, int64_t K) { return (rows + 31) / 32 * ((K + 255) / 256) * 256; }

struct GemmArgs {
  const uint8_t *a, *b;    // codes, row-major; a's rows padded with zeros to whole steps (what a last step
                           // reads of b past a row's end is finite, being E2M1, and multiplies those zeros)
  const uint8_t *as, *bs;  // scale tiles
  uint16_t *y;
  int64_t M, N, K;
  int bf16;
  int vec;                 // y's rows are 16-byte aligned
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t Rsrc(const void *p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)bytes, 0x00020000);
}
// Lane i's 16 (4) bytes at `voffset` land at lds + 16 i (4 i); past the
// descriptor's range they are zeros.  As assembly, so that the compiler does not
// wait for loads into the other stage; the step's barrier does.
__device__ __forceinline__ void DirectLoad16(__amdgpu_buffer_rsrc_t rs, const char *lds, unsigned voffset) {
  const unsigned m0 = (unsigned)(size_t)(lds_ptr_t)lds;
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voffset), "s"(rs), "{m0}"(m0));
}
__device__ __forceinline__ void DirectLoad4(__amdgpu_buffer_rsrc_t rs, const char *lds, unsigned voffset) {
  const unsigned m0 = (unsigned)(size_t)(lds_ptr_t)lds;
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(voffset), "s"(rs), "{m0}"(m0));
}
// This wave's loads have landed and its LDS reads are done; so for all waves.
__device__ __forceinline__ void StepBarrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ uint16_t Half(float v, int bf16) {
  unsigned r;
  if (bf16) {
    asm("v_cvt_pk_bf16_f32 %0, %1, %1" : "=v"(r) : "v"(v));
    return (uint16_t)r;
  }
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// E2M1 operands take the first four registers.
__device__ __forceinline__ v8i Operand(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
__device__ __forceinline__ v8i Operand(v8i v) { return v; }

template <bool A4, int MB, int NB> struct Shape {
  static constexpr int BM = 64 * MB, BN = 64 * NB;
  static constexpr int kRowA = A4 ? 128 : 256;  // bytes of an a row per step
  static constexpr int kA = BM * kRowA, kB = BN * 128, kS = (BM + BN) * 8;
  static constexpr int kStage = kA + kB + kS;
  static constexpr int kLds = 2 * kStage;
};

template <bool A4, int MB, int NB>
__global__ __launch_bounds__(256, (Shape<A4, MB, NB>::kLds > 80 * 1024 ? 1 : 2)) void GemmKernel(const GemmArgs p) {
  using S = Shape<A4, MB, NB>;
  constexpr int BM = S::BM, BN = S::BN, kRowA = S::kRowA;
  constexpr int LA = S::kA / 4096, LB = S::kB / 4096;  // 1 KB loads per wave and step
  constexpr int LS = MB > NB ? MB : NB;                // 256-byte scale loads per wave and step
  __shared__ __align__(1024) char lds[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, r = lane & 31, h = lane >> 5;

  // each XCD a contiguous run of tiles, kGroupM tile rows high, so that tiles
  // sharing rows of a and b share an L2
  const int nbm = (int)((p.M + BM - 1) / BM), nbn = (int)((p.N + BN - 1) / BN), total = nbm * nbn;
  const int pid = (int)blockIdx.x, xcd = pid % kXcds, per = total / kXcds, extra = total % kXcds;
  const int t_all = xcd * per + (xcd < extra ? xcd : extra) + pid / kXcds;
  const int first_m = t_all / (kGroupM * nbn) * kGroupM;
  const int gsize = nbm - first_m < kGroupM ? nbm - first_m : kGroupM;
  const int64_t row0 = (int64_t)__builtin_amdgcn_readfirstlane(first_m + t_all % (kGroupM * nbn) % gsize) * BM;
  const int64_t col0 = (int64_t)__builtin_amdgcn_readfirstlane(t_all % (kGroupM * nbn) / gsize) * BN;

  const int nk = (int)((p.K + 255) / 256);
  const int64_t pitch_a = (int64_t)nk * kRowA, pitch_b = p.K / 2;
  const int64_t rows_a = p.M - row0 < BM ? p.M - row0 : BM, rows_b = p.N - col0 < BN ? p.N - col0 : BN;
  const __amdgpu_buffer_rsrc_t rsA = Rsrc(p.a + row0 * pitch_a, rows_a * pitch_a), rsB = Rsrc(p.b + col0 * pitch_b, rows_b * pitch_b);
  // scale tiles: waves 0 and 1 load those of a's 32-row blocks, 2 and 3 of b's;
  // blocks past the last are not read
  const int sblk = wave < 2 ? MB : NB;
  const uint8_t *scales = wave < 2 ? p.as + row0 / 32 * nk * 256 : p.bs + col0 / 32 * nk * 256;
  const __amdgpu_buffer_rsrc_t rsS = Rsrc(scales, ((wave < 2 ? rows_a : rows_b) + 31) / 32 * nk * 256);
  const __amdgpu_buffer_rsrc_t rs0 = Rsrc(p.a, 0);  // loads past the last step: every access out of range

  // A piece is 1 KB: 8 rows of 128 bytes or 4 of 256; lane -> (row, position),
  // position c of row x holding chunk c ^ key(x).  Piece q of a wave is some rows
  // further and differs in the key by q's low bits alone.
  static_assert(LA % 4 == 0 && LB % 2 == 0, "keys repeat within a wave's pieces");
  unsigned a_g = A4 ? (unsigned)((8 * wave * LA + (lane >> 3)) * pitch_a + 16 * ((lane & 7) ^ (lane >> 3)))
                          : (unsigned)((4 * wave * LA + (lane >> 4)) * pitch_a + 16 * ((lane & 15) ^ (lane >> 4)));
  const unsigned b_row = (unsigned)((8 * wave * LB + (lane >> 3)) * pitch_b);
  unsigned b_g0 = b_row + 16 * ((lane & 7) ^ (lane >> 3)), b_g1 = b_row + 16 * ((lane & 7) ^ (lane >> 3) ^ 1);
  const unsigned a_piece = (unsigned)(A4 ? 8 * pitch_a : 4 * pitch_a), b_piece = (unsigned)(8 * pitch_b);

  constexpr int L = LA + LB + LS;
  // load x (0 .. L - 1) of step t into stage s
  auto issue = [&](int t, int s, int x) __attribute__((always_inline)) {
    const bool live = t < nk;
    char *st = lds + s * S::kStage;
    if (x < LA) {
      DirectLoad16(live ? rsA : rs0, st + (wave * LA + x) * 1024, 
                   (a_g ^ (A4 ? 16 * (x & 1) : 64 * (x & 3))) + ((unsigned)x * a_piece + (unsigned)t * kRowA));
    } else if (x < LA + LB) {
      DirectLoad16(live ? rsB : rs0, st + S::kA + (wave * LB + x - LA) * 1024, 
                   ((x - LA) & 1 ? b_g1 : b_g0) + ((unsigned)(x - LA) * b_piece + (unsigned)t * 128));
    } else {
      const int blk = (wave & 1) * sblk + (x - LA - LB) % sblk;
      DirectLoad4(live ? rsS : rs0, st + S::kA + S::kB + ((wave < 2 ? 0 : 2 * MB) + blk) * 256,
                  (unsigned)((blk * nk + t) * 256 + lane * 4));
    }
  };

  typedef std::conditional_t<A4, v4i, v8i> FragA;
  FragA fa[2][MB];
  v4i fb[2][NB];
  int sa[2][MB], sb[2][NB];
  // fragment x (a's blocks, then b's) of sub-step kk of stage s: 32 rows are 32
  // LDS rows further, a sub-step other bits of the chunk
  int a_rd[2], b_rd[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int row = wm * 32 * MB + r;
    a_rd[s] = s * S::kStage + row * kRowA + 16 * (A4 ? h ^ (r & 7) ^ (r >> 3 & 1) : h ^ (r & 15));
    b_rd[s] = s * S::kStage + S::kA + (wn * 32 * NB + r) * 128 + 16 * (h ^ (r & 7) ^ (r >> 3 & 1));
  }
  auto read = [&](int buf, int s, int kk, int x) __attribute__((always_inline)) {
    if (x < MB) {
      if constexpr (A4) {
        fa[buf][x] = *reinterpret_cast<const v4i *>(lds + (a_rd[s] ^ 32 * kk) + 32 * 128 * x);
      } else {
        const v4i v = *reinterpret_cast<const v4i *>(lds + (a_rd[s] ^ 64 * kk) + 32 * 256 * x);
        const v4i w = *reinterpret_cast<const v4i *>(lds + (a_rd[s] ^ (64 * kk + 32)) + 32 * 256 * x);
        fa[buf][x] = __builtin_shufflevector(v, w, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    } else {
      fb[buf][x - MB] = *reinterpret_cast<const v4i *>(lds + (b_rd[s] ^ 32 * kk) + 32 * 128 * (x - MB));
    }
  };
  auto read_scale = [&](int buf, int s, int x) __attribute__((always_inline)) {
    const char *st = lds + s * S::kStage + S::kA + S::kB;
    if (x < MB)
      sa[buf][x] = *reinterpret_cast<const int *>(st + (wm * MB + x) * 256 + lane * 4);
    else
      sb[buf][x - MB] = *reinterpret_cast<const int *>(st + (2 * MB + wn * NB + x - MB) * 256 + lane * 4);
  };

  v16f acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = v16f{0};
  // b is the instruction's first operand: a result lane then holds 4
  // consecutive columns of y
  auto mma = [&](auto kk, int buf, int sbuf, int x) __attribute__((always_inline)) {
    const int i = x / NB, j = x % NB;
    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(Operand(fb[buf][j]), Operand(fa[buf][i]), acc[i][j], 4,
                                                                A4 ? 4 : 0, kk, sb[sbuf][j], kk, sa[sbuf][i]);
  };

  constexpr int NM = MB * NB, NR = MB + NB;
  // A sub-step: every MFMA with its share of the next sub-step's reads before
  // it and of the direct loads [l0, l1) after it, pinned in that order.
  auto sub = [&](auto kk, int t, int s, int buf, int l0, int l1) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < NM; ++x) {
#pragma unroll
      for (int y = x * NR / NM; y < (x + 1) * NR / NM; ++y) read(buf ^ 1, s, kk + 1, y);
      mma(kk, buf, s, x);
#pragma unroll
      for (int y = l0 + (l1 - l0) * x / NM; y < l0 + (l1 - l0) * (x + 1) / NM; ++y) issue(t + 1, s ^ 1, y);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int kEarly = L / 3, kMid = 2 * L / 3;  // loads issued in the last sub-step of the step before
  // step t in stage s; its fragments of sub-step 0 and its scales are in
  // registers and the first kEarly loads of step t + 1 are out
  auto step = [&](int t, int s) __attribute__((always_inline)) {
    // the loads' and reads' addresses are made where they are used: all of them
    // kept across the loop do not fit beside 256 accumulators
    asm volatile("" : "+v"(a_g), "+v"(b_g0), "+v"(b_g1), "+v"(a_rd[0]), "+v"(a_rd[1]), "+v"(b_rd[0]), "+v"(b_rd[1]));
    sub(std::integral_constant<int, 0>{}, t, s, 0, kEarly, kMid);
    sub(std::integral_constant<int, 1>{}, t, s, 1, kMid, L);
    sub(std::integral_constant<int, 2>{}, t, s, 0, 0, 0);
#pragma unroll
    for (int x = 0; x < NM / 2; ++x) mma(std::integral_constant<int, 3>{}, 1, s, x);
    __builtin_amdgcn_sched_barrier(0);
    StepBarrier();
#pragma unroll
    for (int x = 0; x < NM / 2; ++x) {
      constexpr int H = NM / 2 > 0 ? NM / 2 : 1;
#pragma unroll
      for (int y = x * NR / H; y < (x + 1) * NR / H; ++y) {
        read(0, s ^ 1, 0, y);
        read_scale(s ^ 1, s ^ 1, y);
      }
      mma(std::integral_constant<int, 3>{}, 1, s, NM / 2 + x);
#pragma unroll
      for (int y = kEarly * x / H; y < kEarly * (x + 1) / H; ++y) issue(t + 2, s, y);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int x = 0; x < L; ++x) issue(0, 0, x);
  StepBarrier();
#pragma unroll
  for (int x = 0; x < kEarly; ++x) issue(1, 1, x);
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    read(0, 0, 0, x);
    read_scale(0, 0, x);
  }
  int t = 0;
  do {  // K = 0 runs one step of zeros
    step(t, 0);
    if (t + 1 < nk) step(t + 1, 1);
    t += 2;
  } while (t < nk);
  StepBarrier();  // the loads past the last step, before the LDS is used again

  // ---- output: 32 rows at a time through LDS into whole rows ----
  constexpr int kPitch = 64 * NB + 16;  // bytes of a staged row
  char *st = lds + wave * 32 * kPitch;
  const int64_t c0 = col0 + wn * 32 * NB;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint16_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = Half(acc[i][j][4 * q + e], p.bf16);
        *reinterpret_cast<uint2 *>(st + r * kPitch + (32 * j + 8 * q + 4 * h) * 2) =
            make_uint2(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16);
      }
    // written and read by this wave alone; the LDS keeps its order
    __builtin_amdgcn_sched_barrier(0);
    const int64_t m0 = row0 + (wm * MB + i) * 32;
    if (p.vec) {
      for (int x = lane; x < 32 * 4 * NB; x += 64) {
        const int row = x / (4 * NB), chunk = x % (4 * NB);
        const v4i v = *reinterpret_cast<const v4i *>(st + row * kPitch + chunk * 16);
        if (m0 + row < p.M && c0 + 8 * chunk < p.N) *reinterpret_cast<v4i *>(p.y + (m0 + row) * p.N + c0 + 8 * chunk) = v;
      }
    } else {
      for (int x = lane; x < 32 * 32 * NB; x += 64) {
        const int row = x / (32 * NB), col = x % (32 * NB);
        const uint16_t v = *reinterpret_cast<const uint16_t *>(st + row * kPitch + col * 2);
        if (m0 + row < p.M && c0 + col < p.N) p.y[(m0 + row) * p.N + c0 + col] = v;
      }
    }
  }
}

}  // namespace mx
}  // namespace onnxl_amd
