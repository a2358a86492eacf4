// Which kernel an MX product takes and how that covers it: rules on sizes and types
// alone, plain host code.
#pragma once

#include <algorithm>
#include <cstdint>

namespace onnxl_amd {

// y = a b^T; or gated, act(a b^T) * (a up^T), in 16 bits or as MXFP8.
enum MxOutput : int { kPlain = 0, kGated = 1, kGatedMx = 2 };

namespace mx {

struct Sizes {
  int64_t M, N, K;
  bool x;      // a has 16 bits and is quantized by the call
  bool a_fp4;  // E2M1, else E4M3
  int output;  // MxOutput
  int64_t cus;
};

inline int64_t Ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of a product's weight, or of both weights of a gated one.
inline int64_t WeightRows(const Sizes &p) { return p.output ? 2 * p.N : p.N; }

// Few rows take the streaming kernel, whose time goes with the weight's bytes and the row
// tiles; that of the GEMM's one round of tiles goes with K alone, so from some width of the
// weight on it is less, whatever K is.  That width falls with the rows.  us, rows x K x N,
// stream | GEMM (gated: N of each weight), activations of 16 bits:
//   MXFP8  17 x 4096 x 14336 15.5 | 17.1    17 x 8192 x 20480 31.5 | 30.5
//          24 x 14336 x 12288 38.7 | 44.7   32 x 2048 x 12288 13.6 | 11.8
//          33 x 4096 x 8192 15.2 | 16.1     33 x 28672 x 4096 42.9 | 68.3
//          48 x 14336 x 8192 46.4 | 39.8    64 x 512 x 20480 17.3 | 8.0
//   MXFP4  17 x 4096 x 12288 13.8 | 13.7    24 x 14336 x 14336 43.7 | 41.0
//          33 x 28672 x 8192 54.4 | 63.0    48 x 4096 x 8192 13.3 | 13.2
//          64 x 512 x 28672 15.6 | 7.7      64 x 28672 x 4096 43.4 | 49.6
//   gated, MXFP8
//          17 x 4096 x 8192 15.5 | 18.0     24 x 4096 x 11008 21.4 | 20.3
//          32 x 8192 x 8192 33.8 | 28.3     33 x 4096 x 4096 15.5 | 17.1
//   gated, MXFP4
//          17 x 4096 x 8192 14.2 | 15.1     24 x 4096 x 11008 21.0 | 17.7
//          33 x 8192 x 4096 18.9 | 20.5     48 x 4096 x 5632 18.5 | 14.7
// To MXFP8 a gated product streams with four row tiles, for which more than 32 rows leave
// no registers.  Where its four waves have a chunk of 512 each, up to K = 2048, E4M3 streams
// any width; from E2M1 longer K lowers it.  From codes:
//   MXFP8  17 x 4096 x 11008 19.6 | 20.0    32 x 2048 x 11008 13.5 | 13.7
//          24 x 8192 x 14336 40.0 | 31.0    32 x 4096 x 8192 18.4 | 17.4
//   MXFP4  17 x 2048 x 14336 10.9 | 12.4    20 x 4096 x 11008 21.5 | 17.5
//          24 x 4096 x 8192 13.5 | 14.8     32 x 8192 x 8192 26.0 | 22.4
// Of 1600 such sizes, K from 512 to 28672 and N from 1024 to 28672, the side taken is 0.1 to
// 1.2 % behind the other in the mean of each form, and at most 23 % (gated MXFP8 32 x 2048 x
// 8192, 10.3 | 12.7).
inline bool Streams(const Sizes &p) {
  if (p.M <= 16 || p.M > 64) return p.M <= 16;
  const int64_t rows = WeightRows(p);
  if (p.output == kGatedMx) {
    if (p.M > 32) return false;
    if (p.a_fp4) return rows < 10000 + 46000000 / std::max<int64_t>(p.K, 1);
    return p.K <= 2048 || rows < 36000 - 640 * p.M;
  }
  if (p.M > 32) return rows < (p.a_fp4 ? 13200 - 97 * p.M : 12300 - 105 * p.M);
  if (p.output) return rows < (p.a_fp4 ? 18000 - 70 * p.M : 27000 - 340 * p.M);
  return rows < (p.a_fp4 ? 15000 - 90 * p.M : 18400 - 200 * p.M);
}

// Up to this many values every workgroup quantizes its activations itself
// (eight at a time per thread); a launch for all costs 2 to 4 us.  us, MXFP8, itself |
// in a launch, by N:
//               2048        4096       8192        14336       28672
//   1 x 4096    4.7 | 7.4   5.0 | 7.5   6.3 | 8.1    9.9 | 11.6  16.6 | 18.7
//   2 x 4096    4.8 | 7.3   5.1 | 7.8   7.3 | 8.1   11.7 | 11.9  20.5 | 19.4
//   4 x 4096    6.3 | 7.3   6.3 | 8.0   9.5 | 8.5   15.6 | 12.5  25.8 | 20.3
//   8 x 4096    8.8 | 7.5   8.8 | 8.2  13.3 | 8.9   23.1 | 13.3  37.9 | 21.9
//   8 x 2048    5.6 | 7.5   5.6 | 7.3   7.1 | 7.1   12.6 | 9.7   21.0 | 14.7
//   1 x 8192    6.5 | 8.8   9.4 | 9.4  16.9 | 14.8  20.7 | 25.0  41.0 | 35.4
//   2 x 8192    7.8 | 9.1  11.4 | 9.7  20.5 | 15.2  24.3 | 25.5  45.2 | 36.2
// The rule does not look at N, with which the workgroups that repeat the work grow:
// it holds up to 8192 values and for narrow weights, and loses up to 35 % between
// that and its end by wide ones.
constexpr int64_t kOwnQuant = 16384;
inline bool OwnQuant(const Sizes &p) { return p.x && p.M <= 16 && p.M * Ceil(p.K, 512) * 512 <= kOwnQuant; }

// How the streaming kernel covers a problem: row tiles of 16 nt rows of the
// weight, `split` workgroups of `waves` waves for each.
struct StreamPlan {
  int nt, mt, waves, split;
  int64_t tiles;
};

inline StreamPlan PlanStream(const Sizes &p) {
  StreamPlan s;
  const int64_t chunks = Ceil(p.K, 512);
  s.mt = (int)Ceil(p.M, 16);
  // Activations from memory are read by every wave for itself, all over the chip
  // the same ones at about the same time, and cost as much per 16 rows as the
  // weight: several row tiles share a read, while a wave for every CU's SIMD is
  // left.  More than these do not fit the registers of two waves per SIMD.  us,
  // K = 4096, N = 14336, with these | with one: 8 rows 13.3 | 15.0, 16 rows 15.0 |
  // 18.3, MXFP4 32 rows 14.7 | 19.1, 48 rows 18.2 | 24.0.
  // A gated product's row tiles come in pairs, for MXFP8 blocks in two.
  const int least = p.output == kGatedMx ? 4 : p.output ? 2 : 1;
  s.nt = OwnQuant(p) ? least : s.mt == 1 ? 2 : s.mt <= (p.a_fp4 ? 3 : 2) ? 4 : 2;
  while (s.nt > 1 && Ceil(WeightRows(p), 16 * s.nt) * chunks < 4 * p.cus) s.nt /= 2;
  s.nt = std::max(s.nt, least);
  s.waves = s.nt == 4 ? 4 : 8;
  s.tiles = Ceil(WeightRows(p), 16 * s.nt);
  // as many as give every wave one chunk, while there are not more than about
  // two rounds of them
  s.split = (int)std::max<int64_t>(1, std::min<int64_t>(Ceil(chunks, s.waves), 32 * p.cus / (s.waves * s.tiles)));
  return s;
}

// Large tiles (256 x 256, 128 x 256 for E4M3 activations) feed more MFMAs per
// byte, small ones (128 x 128) leave fewer CUs idle; E4M3 has 128 x 192 between
// them.  A round of small, middle and large ones takes about 20, 24 and 29 parts of
// time (of the small ones two fit a CU for E2M1), and the shortest sum is taken.
// us, large / small: MXFP4 4096 x 4096 x 4096 48 / 55, 4096 x 8192 x 8192 145 / 178, 1000 x 4096 x
// 6144 34 / 28, 256 x 4096 x 4096 28 / 14, gated 1000 x 4096 x 14336 78 / 84; MXFP8 2000 x 4096 x
// 4096 38 / 43, 4096 x 4096 x 4096 71 / 79, 700 x 8192 x 8192 52 / 61, 256 x 4096 x 4096 26 / 18,
// gated 1000 x 4096 x 14336 119 / 124, 1000 x 2048 x 5632 38 / 36 (the rule's loss).  Large /
// middle / small: 1000 x 4096 x 6144 33 / 31 / 38.
//
// A small tile has as many stages as LDS has room for, since a step of its own takes
// less time than a load: three for E4M3, and for E2M1 four, where there are no more tiles
// than CUs, else two, so that two workgroups share a CU.  us, two stages | more: MXFP8 (four
// waves) 128 x 4096 x 4096 20.5 | 18.2, 1000 x 14336 x 4096 66.9 | 61.7; MXFP4 128 x 4096 x
// 4096 17.0 | 13.5, 1000 x 14336 x 4096 55.0 | 47.7, but 1000 x 4096 x 6144 27.5 | 28.9,
// 2000 x 4096 x 4096 31.8 | 32.9.
//
// Tiles have eight waves, two a SIMD, of which one multiplies while the other waits or
// stores.  Four read less of LDS, which wins along a long K of E4M3 by large tiles.
// us, four waves | eight, large tiles: MXFP8 4096 x 512 x 14336 58 | 52, 4096 x 1024 x 8192
// 53 | 49, 1000 x 4096 x 14336 61 | 61, 16384 x 4096 x 4096 264 | 266, 2000 x 8192 x 8192
// 113 | 114, 4096 x 8192 x 8192 220 | 224, 1000 x 14336 x 14336 177 | 188.  When they were
// chosen, MXFP4 1000 x 4096 x 14336 44.4 | 39.8, gated 4096 x 8192 x 14336 572 | 472, gated
// MXFP8 500 x 4096 x 14336 72.6 | 63.0; small ones MXFP8 128 x 4096 x 4096 18.2 | 16.5, MXFP4
// 128 x 4096 x 4096 14.4 | 13.1, 2000 x 4096 x 4096 30.7 | 31.1, gated 33 x 5120 x 13001
// 27.6 | 23.7.  (Three blocks of 32 columns, the middle tile's, are not two waves' to share.)
struct GemmPlan {
  int mb, nb, stages, wm, wn;  // GemmKernel's: blocks of 32 x 32 of a wave, stages, waves
};
inline GemmPlan PlanGemm(const Sizes &p) {
  // a gated tile has half the columns, of two weights
  auto rounds = [&](int64_t m, int64_t n, int64_t at_once) {
    return Ceil(Ceil(p.M, m) * Ceil(p.N, p.output ? n / 2 : n), at_once * p.cus);
  };
  const int64_t small = 20 * rounds(128, 128, p.a_fp4 ? 2 : 1), large = 29 * rounds(p.a_fp4 ? 256 : 128, 256, 1);
  if (!p.a_fp4 && !p.output && 24 * rounds(128, 192, 1) < std::min(small, large)) return {2, 3, 2, 2, 2};
  if (large <= small) {
    if (p.a_fp4) return {4, 2, 2, 2, 4};
    return p.output || p.K < 8192 ? GemmPlan{2, 2, 2, 2, 4} : GemmPlan{2, 4, 2, 2, 2};
  }
  return {1, 2, !p.a_fp4 ? 3 : rounds(128, 128, 1) == 1 ? 4 : 2, 4, 2};
}

}  // namespace mx
}  // namespace onnxl_amd
