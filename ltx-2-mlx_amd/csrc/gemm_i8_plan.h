// Which kernels an int8 product of M x N x K runs on: plain host arithmetic, in a header of its
// own so that host code can ask for every size.
#pragma once

#include <cstdint>

namespace ltx {

struct I8Plan {
  int64_t head;  // rows on 256 x head_bn tiles in a launch before the others' (0: none)
  int head_bn;
  int bm, bn;   // rows and columns of a tile; bn < 0: the few-row kernel, bm rows and -16 bn columns
  int splits;   // K ranges (tiles)
  int k_split;  // k of one, a multiple of 128
};

// Modelled times (us).  Tiles: a round of one workgroup per CU costs `fixed` (epilogue) and per
// 128 k `idle` to `full`, as it fills the CUs (they share the L2s and the chip's power); a
// split's second launch and its partials.  Model against measured (weights from HBM): 1296 x
// 4096 -> 4096 in tiles of 256 x 256, 256 x 128, 128 x 128, 64 x 128 40 / 28 / 33 / 40
// against 45 / 31 / 37 / 41, 3456 x 4096 -> 16384 in tiles of 288 x 256 and these 174 / 202 / 220 / 260 / 335
// against 176 / 195 / 209 / 254 / 330, 512 x 4096 -> 4096 64 x 128 16 / 17, 68 x 8192 -> 2048 in 8 ranges 11 / 13.
// 288 rows take 12 % more than 256 where both fill as many rounds: 6144 x 4096 -> 16384 337 against 313
// (bias; with a residual their epilogue spills and they are up to 7 % slower also with a round less);
// one round instead of two: 4100 x 4096 -> 4096 61 against 82 (256 x 128).
inline double i8_time(int64_t M, int64_t N, int bm, int bn, int splits, double per) {
  const double wgs = (double)(((M + bm - 1) / bm) * ((N + bn - 1) / bn) * splits);
  double fixed = 1.6, idle = 0.30, full = 0.34;
  if (bm == 288) fixed = 6.6, idle = 1.00, full = 1.56;
  else if (bm == 256 && bn == 256) fixed = 6.0, idle = 0.85, full = 1.40;
  else if (bm == 256) fixed = 4.6, idle = 0.62, full = 0.78;
  else if (bm == 128) fixed = 2.5, idle = 0.42, full = 0.48;
  const double rounds = (double)(int64_t)(wgs / 256), rest = wgs / 256 - rounds;
  double t = 4.0 + rounds * (fixed + per * full);
  if (rest > 0) t += fixed + per * (idle + (full - idle) * rest);
  if (splits > 1) t += 2.5 + (double)(M * N) * splits * 8 / 4e6;
  return t;
}
// The few-row kernel: a CU gets 33 bytes of operands per ns.
inline double i8_rows_time(int64_t M, int64_t N, int64_t K, int mb, int nb) {
  const double wgs = (double)(((M + 16 * mb - 1) / (16 * mb)) * ((N + 16 * nb - 1) / (16 * nb)));
  const double rounds = wgs < 256 ? 1.0 : wgs / 256;
  return 3.2 + rounds * (double)(16 * (mb + nb) * K) / 33e3;
}

// The fastest single launch (or, where `split`, K ranges and a combining one) and its time
inline double i8_one(int64_t M, int64_t N, int64_t K, bool split, I8Plan* pl) {
  static const int tile[5][2] = {{288, 256}, {256, 256}, {256, 128}, {128, 128}, {64, 128}};
  // rows of the few-row kernel; 32 columns where that leaves a workgroup for every CU
  const int mb = M <= 16 ? 1 : (M <= 32 ? 2 : 4), nb = N >= 32 * 256 ? 2 : 1;
  const int64_t units = (K + 127) / 128;
  *pl = {0, 0, 16 * mb, -nb, 1, (int)K};
  double best = i8_rows_time(M, N, K, mb, nb);
  if (M <= 32) return best;
  for (const auto& t : tile) {
    const int64_t tiles = ((M + t[0] - 1) / t[0]) * ((N + t[1] - 1) / t[1]);
    for (int want = 1; want <= (split ? 16 : 1); ++want) {
      // splits: at least two stages each, within one round of the CUs, 10 % faster
      if (want > 1 && (units / want < 2 || tiles * want > 256)) break;
      const int64_t per = (units + want - 1) / want;
      const int s = (int)((units + per - 1) / per);
      const double us = i8_time(M, N, t[0], t[1], s, (double)per);
      if (us < best * (s > 1 ? 0.9 : 1.0)) {
        best = us;
        *pl = {0, 0, t[0], t[1], s, (int)(per * 128)};
      }
    }
  }
  return best;
}

// Rows [0, head) on 256-row tiles, where those make (nearly) whole rounds of the CUs and another
// kernel takes the rows left over for less than one more round: 5120 x 4096 -> 4096 as 4096
// rows of 256 x 256 tiles and 1024 of 128 x 128 77 us, in one launch 90; 1497 x 4032 -> 12744 77 and 93.
inline I8Plan i8_plan(int64_t M, int64_t N, int64_t K) {
  I8Plan pl;
  double best = i8_one(M, N, K, true, &pl);
  const double units = (double)((K + 127) / 128);
  for (int64_t b = (M - 1) / 256, tries = 0; b >= 1 && tries < 8; --b, ++tries) {
    I8Plan rest;
    const double left = i8_one(M - 256 * b, N, K, false, &rest);
    for (int bn = 128; bn <= 256; bn += 128) {
      const double t = i8_time(256 * b, N, 256, bn, 1, units) + left;
      if (t < 0.95 * best) {
        best = t;
        pl = rest;
        pl.head = 256 * b;
        pl.head_bn = bn;
      }
    }
  }
  return pl;
}

}  // namespace ltx
