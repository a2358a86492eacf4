// Block-scaled GEMM for many rows: y[M, N] = a[M, K] b[N, K]^T with a MXFP4 or
// MXFP8 and b MXFP4, on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// Both operands are rows with consecutive k, which is how the instruction wants
// them: lane l holds row l % 32 and, with h = l / 32, for E2M1 the 32 values
// from 32 h (16 bytes), for E4M3 the 16 from 16 h and the 16 from 32 + 16 h; the
// E8M0 scale of k block h comes from the same lane, one byte of a register that
// the instruction selects.
//
// Workgroup: WM x WN waves, 4 (2 x 2) or 8 (2 x 4, 4 x 2), each with MB x NB
// blocks of 32 x 32.  A K step is 256 values: 128 bytes of an E2M1 row, 256 of
// an E4M3 row, two 16-byte chunks (four) per 64-value sub-step and lane.  Two
// or more stages in LDS, filled by direct loads (16 bytes a lane, nothing held in
// registers) while another is multiplied; a row's chunks are XOR-swizzled by
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
// What bounds it: the matrix cores work half of the time.  A product takes 56 cycles
// of its SIMD where the instruction needs 32 (MXFP4, 4096 rows, plain or gated; with MXFP8
// and 1000 rows 120 to 180 and 64).  The fragments take LDS about as long as the products
// the matrix cores: a step of the large MXFP4 tile reads 192 KB and writes 64, 2000
// cycles at the nominal 128 bytes a cycle, beside 2048 of products, and the two meet only in part;
// at 4096 rows the clock falls to the power as well.
//
// A gated product (MxOutput) has the 32-row blocks of both weights in turn in the
// tile's b, so that a wave's two blocks of b are gate and up of the same 32
// columns of y and meet in the registers.
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
#include "mx_gate.hpp"
#include "quant8.hpp"

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
  const uint8_t *up = nullptr, *ups = nullptr;  // gated: the second weight [N, K], its scale tiles
  int activation = 0;
  uint8_t *y_scale = nullptr;                   // kGatedMx: y is codes, these their scales [M, N / 32]
  int first = 0;           // the launch's first workgroup
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
// This wave's loads but the last LEFT have landed and its LDS reads are done; so for all waves.
template <int LEFT = 0> __device__ __forceinline__ void StepBarrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// To nearest even, by conversions that the compiler knows: v may be a matrix product's register, for which it puts
// in the wait states (behind an assembly statement it does not).
__device__ __forceinline__ uint16_t Half(float v, int bf16) {
  return bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// E2M1 operands take the first four registers.
__device__ __forceinline__ v8i Operand(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
__device__ __forceinline__ v8i Operand(v8i v) { return v; }

template <bool A4, int MB, int NB, int STAGES, int WM, int WN> struct Shape {
  static constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
  static constexpr int kRowA = A4 ? 128 : 256;  // bytes of an a row per step
  static constexpr int kA = BM * kRowA, kB = BN * 128, kS = (BM + BN) * 8;
  static constexpr int kStage = kA + kB + kS;
  static constexpr int kLds = STAGES * kStage;
};

// Waves of a SIMD that the registers have to suffice for: those of one workgroup, or of two
// where LDS has room for them.
template <typename S, int W> constexpr int kGemmFit = W / 4 * (S::kLds > 80 * 1024 ? 1 : 2);

template <bool A4, int MB, int NB, int STAGES, int WM, int WN, int OUT = kPlain>
__global__ __launch_bounds__(64 * WM * WN, (kGemmFit<Shape<A4, MB, NB, STAGES, WM, WN>, WM * WN>)) void GemmKernel(const GemmArgs p) {
  using S = Shape<A4, MB, NB, STAGES, WM, WN>;
  constexpr int W = WM * WN;
  constexpr int NW = OUT == kPlain ? 1 : 2, NO = NB / NW;  // weights, a wave's blocks of y's columns
  static_assert(NB % NW == 0, "gate and up in pairs");
  constexpr int BM = S::BM, BN = S::BN / NW, kRowA = S::kRowA;  // rows and columns of y
  constexpr int LA = S::kA / (1024 * W), LB = S::kB / (1024 * W);  // 1 KB loads per wave and step
  constexpr int LS = W == 4 ? (MB > NB ? MB : NB) : WN == 4 ? 2 : 1;  // 256-byte scale loads per wave and step
  __shared__ __align__(1024) char lds[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, r = lane & 31, h = lane >> 5;

  // each XCD a contiguous run of tiles, kGroupM tile rows high, so that tiles
  // sharing rows of a and b share an L2
  const int nbm = (int)((p.M + BM - 1) / BM), nbn = (int)((p.N + BN - 1) / BN), total = nbm * nbn;
  const int pid = p.first + (int)blockIdx.x, xcd = pid % kXcds, per = total / kXcds, extra = total % kXcds;
  const int t_all = xcd * per + (xcd < extra ? xcd : extra) + pid / kXcds;
  const int first_m = t_all / (kGroupM * nbn) * kGroupM;
  const int gsize = nbm - first_m < kGroupM ? nbm - first_m : kGroupM;
  const int64_t row0 = (int64_t)__builtin_amdgcn_readfirstlane(first_m + t_all % (kGroupM * nbn) % gsize) * BM;
  const int64_t col0 = (int64_t)__builtin_amdgcn_readfirstlane(t_all % (kGroupM * nbn) / gsize) * BN;

  const int nk = (int)((p.K + 255) / 256);
  const int64_t pitch_a = (int64_t)nk * kRowA, pitch_b = p.K / 2;
  const int64_t rows_a = p.M - row0 < BM ? p.M - row0 : BM, rows_b = p.N - col0 < BN ? p.N - col0 : BN;
  // gated: a wave's pieces of b are one of the weights', blocks of 32 rows in turn
  const bool b_up = OUT != kPlain && (LB == 2 ? wave / 2 : wave) % 2;
  const __amdgpu_buffer_rsrc_t rsA = Rsrc(p.a + row0 * pitch_a, rows_a * pitch_a);
  const __amdgpu_buffer_rsrc_t rsB = Rsrc((b_up ? p.up : p.b) + col0 * pitch_b, rows_b * pitch_b);
  // scale tiles, blocks of 32 rows, those past the last not read.  Four waves: 0 and 1 load
  // those of a, 2 and 3 of b; 4 x 2: each one, the first four of a; 2 x 4: each one of b's
  // and one of a's, which two load where there are four.  Gated: odd blocks of b are the
  // second weight's
  static_assert(W == 4 ? OUT == kPlain : NB == 2 && (WN == 4 ? MB <= 4 : MB == 1), "scale blocks by waves");
  const uint8_t *as = p.as + row0 / 32 * nk * 256, *bs = (OUT != kPlain && wave % 2 ? p.ups : p.bs) + col0 / 32 * nk * 256;
  const int64_t as_bytes = (rows_a + 31) / 32 * nk * 256, bs_bytes = (rows_b + 31) / 32 * nk * 256;
  const bool for_a = WN == 4 || wave < W / 2;
  const __amdgpu_buffer_rsrc_t rsS = Rsrc(for_a ? as : bs, for_a ? as_bytes : bs_bytes), rsT = Rsrc(bs, WN == 4 ? bs_bytes : 0);
  const __amdgpu_buffer_rsrc_t rs0 = Rsrc(p.a, 0);  // loads past the last step: every access out of range

  // A piece is 1 KB: 8 rows of 128 bytes or 4 of 256; lane -> (row, position),
  // position c of row x holding chunk c ^ key(x).  Piece q of a wave is some rows
  // further and differs in the key by q's low bits alone.
  static_assert(LA % (A4 ? 2 : 4) == 0 && LB % 2 == 0, "keys repeat within a wave's pieces");
  unsigned a_g = A4 ? (unsigned)((8 * wave * LA + (lane >> 3)) * pitch_a + 16 * ((lane & 7) ^ (lane >> 3)))
                          : (unsigned)((4 * wave * LA + (lane >> 4)) * pitch_a + 16 * ((lane & 15) ^ (lane >> 4)));
  static_assert(OUT == kPlain || LB == 4 || LB == 2, "a block a wave, or half of one");
  const int b_first = OUT == kPlain ? wave * LB : LB == 4 ? wave / 2 * 4 : wave / 4 * 4 + wave % 2 * 2;  // in eights, of the weight
  const unsigned b_row = (unsigned)((8 * b_first + (lane >> 3)) * pitch_b);
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
      const int piece = x - LA;
      DirectLoad16(live ? rsB : rs0, st + S::kA + (wave * LB + piece) * 1024,
                   (piece & 1 ? b_g1 : b_g0) + ((unsigned)piece * b_piece + (unsigned)t * 128));
    } else {
      const int i = x - LA - LB;
      const bool of_a = WN == 4 ? i == 0 : wave < W / 2;
      const int blocks = of_a ? WM * MB : WN * NB;  // of the tile
      const int blk = W == 4 ? wave % 2 * (blocks / 2) + i % (blocks / 2) : wave % blocks;
      const int from = OUT != kPlain && !of_a ? blk / 2 : blk;  // of the matrix
      DirectLoad4(live ? (WN == 4 && i ? rsT : rsS) : rs0, st + S::kA + S::kB + ((of_a ? 0 : WM * MB) + blk) * 256,
                  (unsigned)((from * nk + t) * 256 + lane * 4));
    }
  };

  typedef std::conditional_t<A4, v4i, v8i> FragA;
  FragA fa[2][MB];
  v4i fb[2][NB];
  int sa[2][MB], sb[2][NB];
  // fragment x (a's blocks, then b's) of sub-step kk of stage s: 32 rows are 32
  // LDS rows further, a sub-step other bits of the chunk
  int a_rd[STAGES], b_rd[STAGES];
#pragma unroll
  for (int s = 0; s < STAGES; ++s) {
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
      sb[buf][x - MB] = *reinterpret_cast<const int *>(st + (WM * MB + wn * NB + x - MB) * 256 + lane * 4);
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
  auto sub = [&](auto kk, int t, int s, int sbuf, int buf, int l0, int l1) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < NM; ++x) {
#pragma unroll
      for (int y = x * NR / NM; y < (x + 1) * NR / NM; ++y) read(buf ^ 1, s, kk + 1, y);
      mma(kk, buf, sbuf, x);
#pragma unroll
      for (int y = l0 + (l1 - l0) * x / NM; y < l0 + (l1 - l0) * (x + 1) / NM; ++y) issue(t + STAGES - 1, (s + STAGES - 1) % STAGES, y);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int kEarly = L / 3, kMid = 2 * L / 3;  // loads issued in the last sub-step of the step before
  // step t in stage s; its fragments of sub-step 0 and its scales are in
  // registers and the first kEarly loads of step t + 1 are out
  auto step = [&](int t, int s, int sbuf) __attribute__((always_inline)) {
    // the loads' and reads' addresses are made where they are used: all of them
    // kept across the loop do not fit beside 256 accumulators
    asm volatile("" : "+v"(a_g), "+v"(b_g0), "+v"(b_g1));
#pragma unroll
    for (int i = 0; i < STAGES; ++i) asm volatile("" : "+v"(a_rd[i]), "+v"(b_rd[i]));
    sub(std::integral_constant<int, 0>{}, t, s, sbuf, 0, kEarly, kMid);
    sub(std::integral_constant<int, 1>{}, t, s, sbuf, 1, kMid, L);
    sub(std::integral_constant<int, 2>{}, t, s, sbuf, 0, 0, 0);
#pragma unroll
    for (int x = 0; x < NM / 2; ++x) mma(std::integral_constant<int, 3>{}, 1, sbuf, x);
    __builtin_amdgcn_sched_barrier(0);
    StepBarrier<(STAGES - 2) * L>();
#pragma unroll
    for (int x = 0; x < NM / 2; ++x) {
      constexpr int H = NM / 2 > 0 ? NM / 2 : 1;
#pragma unroll
      for (int y = x * NR / H; y < (x + 1) * NR / H; ++y) {
        read(0, (s + 1) % STAGES, 0, y);
        read_scale(sbuf ^ 1, (s + 1) % STAGES, y);
      }
      mma(std::integral_constant<int, 3>{}, 1, sbuf, NM / 2 + x);
#pragma unroll
      for (int y = kEarly * x / H; y < kEarly * (x + 1) / H; ++y) issue(t + STAGES, s, y);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
#pragma unroll
    for (int x = 0; x < L; ++x) issue(i, i, x);
  StepBarrier<(STAGES - 2) * L>();
#pragma unroll
  for (int x = 0; x < kEarly; ++x) issue(STAGES - 1, STAGES - 1, x);
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    read(0, 0, 0, x);
    read_scale(0, 0, x);
  }
  // (the scales' two buffers take turns as well)
  constexpr int kUnroll = STAGES % 2 ? 2 * STAGES : STAGES;
  int t = 0;
  do {  // K = 0 runs one step of zeros
    step(t, 0, 0);
#pragma unroll
    for (int i = 1; i < kUnroll; ++i) {
      if (t + i >= nk) break;
      step(t + i, i % STAGES, i % 2);
    }
    t += kUnroll;
  } while (t < nk);
  StepBarrier();  // the loads past the last step, before the LDS is used again

  // ---- output: 32 rows at a time through LDS into whole rows ----
  constexpr int kSize = OUT == kGatedMx ? 1 : 2, kCols = 32 * NO;  // bytes of a value, a wave's columns of y
  constexpr int kPitch = kCols * kSize + 16;                       // bytes of a staged row
  char *st = lds + wave * 32 * kPitch;
  const int64_t c0 = col0 + wn * kCols;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t m0 = row0 + (wm * MB + i) * 32;
#pragma unroll
    for (int j = 0; j < NO; ++j) {
      if constexpr (OUT != kPlain) {
        v16f &f = acc[i][2 * j];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = Activate(f[e], p.activation) * acc[i][2 * j + 1][e];
      }
      if constexpr (OUT == kGatedMx) {
        // a lane and the one 32 further have the 32 columns, a block
        const v16f &f = acc[i][2 * j];
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, __builtin_bit_cast(unsigned, (float)f[e]) & 0x7fffffffu);
        top = max(top, (unsigned)__shfl_xor((int)top, 32));
        const BlockScale b = MxScaleOf(__builtin_bit_cast(float, top), 8);
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const float v[8] = {f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3], f[4 * q + 4], f[4 * q + 5], f[4 * q + 6], f[4 * q + 7]};
          const uint2 w = MxFp8Codes8(v, b);
          *reinterpret_cast<unsigned *>(st + r * kPitch + 32 * j + 8 * q + 4 * h) = w.x;
          *reinterpret_cast<unsigned *>(st + r * kPitch + 32 * j + 8 * q + 8 + 4 * h) = w.y;
        }
        if (h == 0 && m0 + r < p.M && c0 + 32 * j < p.N) p.y_scale[(m0 + r) * (p.N / 32) + c0 / 32 + j] = b.e8m0;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint16_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = Half(acc[i][NW * j][4 * q + e], p.bf16);
          *reinterpret_cast<uint2 *>(st + r * kPitch + (32 * j + 8 * q + 4 * h) * 2) =
              make_uint2(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16);
        }
      }
    }
    // written and read by this wave alone; the LDS keeps its order
    __builtin_amdgcn_sched_barrier(0);
    uint8_t *y = reinterpret_cast<uint8_t *>(p.y);
    if (p.vec) {
      constexpr int kChunks = kCols * kSize / 16;
      for (int x = lane; x < 32 * kChunks; x += 64) {
        const int row = x / kChunks, chunk = x % kChunks;
        const v4i v = *reinterpret_cast<const v4i *>(st + row * kPitch + chunk * 16);
        if (m0 + row < p.M && c0 + 16 / kSize * chunk < p.N)
          *reinterpret_cast<v4i *>(y + ((m0 + row) * p.N + c0) * kSize + 16 * chunk) = v;
      }
    } else if constexpr (OUT != kGatedMx) {  // whose rows are whole blocks of 32
      for (int x = lane; x < 32 * kCols; x += 64) {
        const int row = x / kCols, col = x % kCols;
        const uint16_t v = *reinterpret_cast<const uint16_t *>(st + row * kPitch + col * 2);
        if (m0 + row < p.M && c0 + col < p.N) p.y[(m0 + row) * p.N + c0 + col] = v;
      }
    }
  }
}

}  // namespace mx
}  // namespace onnxl_amd
