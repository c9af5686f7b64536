// The 8-wave tile kernel of the projection GEMMs (gemm.hip: bf16, int8, MXFP8
// weights, MXFP8 x MXFP8; gemm_fp4.hip: MXFP4 weights) and its launches.
#pragma once

#include "gemm_fp4.h"

namespace ltx {

// ---- 8-wave ping-pong kernel (8-bit weights; bf16 weights in 32-deep stages) --
// 256x256 tile, K step 64, eight waves (two per SIMD) in two groups of four:
// group 0 (waves 0-3) owns output rows 0-127 of the tile, group 1 (waves 4-7)
// rows 128-255; wave w & 3 owns 64 output columns.  The groups run half a
// stage apart: while one group issues its memory cluster (LDS fragment reads
// of a stage, its direct global->LDS loads of later stages, the scale loads),
// the other group's compute cluster (the stage's 64 16x16x32 MFMAs with the
// weight dequantisation of fragments 2-7 interleaved) keeps the SIMD's matrix
// pipe busy.  The memory cluster ends, once its fragment
// reads have landed, by decoding the stage's E8M0 scales and dequantising
// fragments 0 and 1, so the compute cluster's first MFMAs issue right after
// the barrier (FF up 402 -> 382 us: the dependent decode -> convert chain had
// left the matrix pipe idle at the start of every compute cluster).
// A workgroup barrier separates the clusters.  Both operands reach LDS by
// direct loads (no staging registers, no LDS write instructions) of whole
// 128-byte lines: stages of bf16 activations (256 x 128 B), moved by group 0
// one stage ahead, and pairs of stages of raw weight codes (256 x 128 B),
// moved by group 1 with the scales a pair ahead, two slots each (all that fits
// beside the scales; against three single stages, 64 bytes of codes per row,
// moved by all waves: FF up 329 -> 321 us, QKV 250 -> 244, 6144 x 4096 -> 12320
// 428 -> 420, 3888 x 16384 -> 4096 340 -> 333; int8 FF up 383 -> 377).  The MXFP8
// / int8 codes are dequantised per fragment with the exact format arithmetic, so
// the bf16 MFMA sees bit-exact weights.  bf16 weights: 32-deep stages that reach
// LDS in pairs (128-byte rows of both operands), 32 MFMAs per cluster, no
// dequantisation; 64-byte rows, twice the L2 requests, measured 354 against 326
// us on FF up at M = 3456, 267 against 248 on QKV, 197 against 184 on 2048 x 4096
// -> 16384.
// MXFP4 weights: units of four stages (256 x 128 B of codes), a fragment read of
// 8 bytes per lane and stage, the scale words of 512 k as four rows of 256.
// MX (8-bit codes of both operands): 16 scaled 32x32x64 MFMAs per cluster.
//
// Inside a stage the k order of the MFMA slots is permuted so that a lane
// reads the codes of both k-steps of the stage with one 16-byte LDS read:
// k-step s, lane quarter q covers k = 16q + 8s + [0, 8) for both operands
// (the E8M0 block of that k range is q / 2).  MX: k-step pair p of the
// scaled MFMA, lane half h, k = 32p + 16h + [0, 16).  The sum over the stage
// is the same set of products.
constexpr int kG8Threads = 512;
// the automatic tile choice uses the 8-wave kernel from 100 256x256 tiles on

template <int BKIND, int BM_ = 256>
struct G8Cfg {
  static constexpr bool MX = BKIND == B_MX;
  // bf16 weights: stages are 32 deep, but both operands reach LDS in pairs of
  // stages, rows of 128 bytes: a 64-byte piece costs the L2 a request like a
  // whole line does (FF up in 64-byte rows: 52 M requests in the 256-row
  // launch, 0.70 per L2 channel and cycle; 27 M and 0.39 here).  Rings of A_SLOTS and B_SLOTS
  // pairs -- all that 160 KB hold: the activations (mostly L2 hits) one pair
  // ahead, the weights (HBM) two.
  static constexpr bool BF = BKIND == B_BF16;
  static constexpr int BM = BM_, BN = 256, BK = BF ? 32 : 64;
  // 8-bit weights (W8): the codes in pairs of 64-deep stages too (activation
  // rows are 128 bytes as they are).  MX: single stages of both.
  static constexpr bool W8 = !BF && !MX;
  // MXFP4: codes of half a byte, so a 128-byte row holds four stages
  static constexpr bool FP4 = BKIND == B_MXFP4;
  static constexpr int BU = FP4 ? 4 : 2;  // stages per weight unit (W8)
  // ring slots: A stages (BF: pairs), B pairs (MX: stages)
  static constexpr int A_SLOTS = MX ? 3 : (BM == 256 ? 2 : 3), B_SLOTS = W8 && BM == 256 ? 2 : 3;
  // stages of one turn of both rings, the loop's unrolling
  static constexpr int STAGES = MX ? 3 : (BF ? (BM == 256 ? 12 : 6) : (BM == 256 ? 2 * BU : 3 * BU));
  // 128x64 wave tiles: each weight fragment is dequantised by the two waves
  // that share its columns rather than four (64x128 tiles read fewer LDS
  // bytes per MFMA, but MXFP8 measured 2.5 % slower with them: the
  // conversions cost more power than the extra fragment reads).  Tiles of
  // 128 rows (BM_ = 128: 64x64 wave tiles) for products whose 256-row tiles
  // fill only part of one round.
  static constexpr int WM = BM / 2, WN = 64;
  static constexpr int TM = WM / 32, TN = WN / 32;
  static constexpr int WAVES_M = BM / WM;
  // bf16 MFMAs (bf16 or dequantised 8-bit weights) in the 16x16x32 shape:
  // same flops per cycle as 32x32x16, but the chip holds a ~12 % higher clock
  // under it at full load (2.0 vs 1.7-1.8 GHz in a register-only loop of
  // either shape on all 256 CUs); the wave tile, hence the LDS reads and the
  // accumulator registers, is unchanged.  MX keeps the scaled 32x32x64.
  static constexpr bool S16 = !MX;
  static constexpr int TM16 = WM / 16, TN16 = WN / 16;
  // bf16 activations (MX: 8-bit codes like the weights), 8-bit weight codes
  // (BF: bf16 weights)
  // (BF: a pair of stages; W8: of the weights)
  static constexpr int A_ROWB = MX ? BK : 128, B_ROWB = MX ? BK : 128;
  static constexpr int A_BYTES = BM * A_ROWB, B_BYTES = BN * B_ROWB;
  // LDS: the A stages, then the B stages (every fragment read is then a fixed
  // per-lane register plus an immediate offset below 64 KiB)
  static constexpr int B_REGION = A_SLOTS * A_BYTES;
  // direct loads per wave and stage (BF: pair).  W8: group 0 moves the
  // activations, group 1 the weights and scales, per wave and stage / pair
  static constexpr int LOADERS = W8 ? 4 : 8;
  static constexpr int A_DMA = A_BYTES / 1024 / LOADERS, B_DMA = B_BYTES / 1024 / LOADERS;
  // epilogue staging rows: 16x16 accumulators, 128-byte rows with their
  // 16-byte chunks XORed by (row / 2) % 8 (conflict-free for both the 8-byte
  // accumulator writes and the 16-byte row reads, probed); 32x32 (MX), rows
  // padded to 144 bytes
  static constexpr int EPI_ROWB = S16 ? WN * 2 : WN * 2 + 16;
  static constexpr int EPI_WAVE = WM * EPI_ROWB;
  static constexpr int EPI_BYTES = 8 * EPI_WAVE;
  static constexpr int COL_BYTES = 2 * BN * 4;
  // the column values (bias, gate) follow the epilogue's staging area; they
  // are written after the main loop, so they may lie inside the stage ring
  static constexpr int COL_OFF = EPI_BYTES;
  static constexpr int RING = B_REGION + B_SLOTS * B_BYTES;
  static constexpr bool COL_IN_RING = COL_OFF < RING;
  static constexpr int LDS_BYTES = (RING > EPI_BYTES + COL_BYTES) ? RING : EPI_BYTES + COL_BYTES;
  // MXFP8 scales of eight stages (256 rows x 16 E8M0 bytes), double buffered;
  // MX: the weights' then the activations' octets
  static constexpr int SC_OCT = BN * 16;
  static constexpr int SC_BYTES = BKIND == B_MXFP8 || FP4 ? 2 * SC_OCT : (MX ? 4 * SC_OCT : 0);
  // the scale octets after the column values, or (MX) right after the
  // stages, inside the epilogue's staging area (dead by then: every scale
  // load has landed before the epilogue's first barrier)
  static constexpr int SC_OFF = MX ? RING : LDS_BYTES;
  static constexpr int TOTAL = MX ? LDS_BYTES : LDS_BYTES + SC_BYTES;
  static_assert(!MX || SC_OFF + SC_BYTES <= EPI_BYTES, "MX scales inside the staging area");
  static_assert(TOTAL <= 160 * 1024, "LDS");
  static_assert(BM == 256 || (BM == 128 && !MX), "256-row tiles, or 128 without MX activations");
};

template <int BKIND, int EPI, int BM_ = 256>
__global__ __launch_bounds__(kG8Threads, 1) void gemm8_kernel(GemmArgs p) {
  using Cfg = G8Cfg<BKIND, BM_>;
  constexpr int BN = Cfg::BN, WM = Cfg::WM, WN = Cfg::WN, TM = Cfg::TM, TN = Cfg::TN;
  constexpr int A_ROWB = Cfg::A_ROWB, B_ROWB = Cfg::B_ROWB, A_BYTES = Cfg::A_BYTES, B_BYTES = Cfg::B_BYTES;
  constexpr int B_REGION = Cfg::B_REGION;
  constexpr int A_DMA = Cfg::A_DMA, B_DMA = Cfg::B_DMA;
  constexpr int EPI_ROWB = Cfg::EPI_ROWB, EPI_WAVE = Cfg::EPI_WAVE;
  constexpr bool RESID = EPI == LTX_GEMM_EPI_RESIDUAL || EPI == LTX_GEMM_EPI_RESIDUAL_ROUND;
  constexpr bool MX = Cfg::MX, BF = Cfg::BF, W8 = Cfg::W8, S16 = Cfg::S16, FP4 = Cfg::FP4;
  constexpr int BU = Cfg::BU;
  constexpr int TM16 = Cfg::TM16, TN16 = Cfg::TN16;
  constexpr int STAGES = Cfg::STAGES;
  constexpr int AP = Cfg::A_SLOTS, BP = Cfg::B_SLOTS;
  constexpr int LOADERS = Cfg::LOADERS;
  __shared__ __attribute__((aligned(1024))) char lds[Cfg::TOTAL];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  // wave-uniform values live in scalar registers: the memory clusters then
  // compute their LDS destinations and load bases with scalar instructions
  // (vector instructions of one wave take matrix-pipe slots from the other)
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2;  // waves w and w + 4 share a SIMD
  const int wm = wave % Cfg::WAVES_M, wn = wave / Cfg::WAVES_M;

  int tmi, tni;
  tile_coords((int)blockIdx.x, (int)gridDim.x, p.tiles_m, p.tiles_n, tmi, tni);
  const int m0 = tmi * Cfg::BM, n0 = tni * BN;
  const int KT = p.K / Cfg::BK;
  // a wave whose 128 x 64 sub-tile lies wholly past M or N (the last row or
  // column of tiles) reads no fragments and issues no MFMAs: it still moves
  // its share of every stage and meets every barrier
  // (an int from a scalar register: a bool kept across the loop becomes a lane
  // mask whose tests cost vector instructions in every cluster)
  const int live = __builtin_amdgcn_readfirstlane((m0 + wm * WM < p.M && n0 + wn * WN < p.N) ? 1 : 0);

  float* col_lds = reinterpret_cast<float*>(lds + Cfg::COL_OFF);

  // ---- direct-load sources.  A wave instruction fills one contiguous 1 KiB
  // block of LDS, lane j its 16-byte slot j; the lane's source address picks
  // the logical chunk that the slot holds under the XOR swizzle of its row
  // (g8_swz128 for the 128-byte A rows, 8 per block; g8_swz64 for the 64-byte
  // rows, 16 per block; swz_pair for rows of a stage pair), the one under which
  // this kernel's fragment reads are conflict-free.  Rows past M / N re-read the
  // last row.
  // Direct loads as buffer loads: a buffer descriptor per operand (scalar
  // registers), a fixed 32-bit per-lane byte offset in one vector register,
  // the stage's advance as the scalar offset and the LDS destination in M0
  // -- no vector instructions per load (vector instructions of one wave take
  // matrix-pipe slots from the other).  The descriptors' record counts bound the
  // lane offsets to their operand (the launchers check the 31-bit extents: g8_ok, for
  // MXFP4 fp4_rows_per_launch), the clamps
  // on the stage the scalar offset, which the counts do not cover.
  const int a_records = (int)((int64_t)p.M * p.lda * (MX ? 1 : 2)),
            b_records = FP4 ? (int)((int64_t)(p.N - 1) * p.ldb + p.K / 2)
                            : (int)(((int64_t)(p.N - 1) * p.ldb + p.K) * (BF ? 2 : 1));
  const int loader = W8 ? wave & 3 : wave;
  uint32_t a_src[A_DMA];
#pragma unroll
  for (int d = 0; d < A_DMA; ++d) {
    if constexpr (MX) {
      // activation codes: 64-byte rows laid out like the weight codes
      const int r = 16 * (8 * d + wave) + (lane >> 2);
      int gm = m0 + r;
      gm = gm < p.M ? gm : p.M - 1;
      const int chunk = (lane & 3) ^ g8_swz64(r, S16);
      a_src[d] = (uint32_t)((int64_t)gm * p.lda) + chunk * 16;
    } else {
      const int r = 8 * (LOADERS * d + loader) + (lane >> 3);
      int gm = m0 + r;
      gm = gm < p.M ? gm : p.M - 1;
      const int chunk = BF ? pair_chunk(lane) : (lane & 7) ^ g8_swz128(r, S16);
      a_src[d] = (uint32_t)((int64_t)gm * p.lda * 2) + chunk * 16;
    }
  }
  uint32_t b_src[B_DMA];
#pragma unroll
  for (int d = 0; d < B_DMA; ++d) {
    const int r = MX ? 16 * (8 * d + wave) + (lane >> 2) : 8 * (LOADERS * d + loader) + (lane >> 3);
    int gn = n0 + r;
    gn = gn < p.N ? gn : p.N - 1;
    // MXFP4: fragment reads of 8 bytes, 16 rows of a chunk together: (r / 2) % 8
    // gives the 16 rows 16 different pieces of two LDS rows
    const int chunk = MX ? (lane & 3) ^ g8_swz64(r, S16) : (FP4 ? (lane & 7) ^ ((r >> 1) & 7) : pair_chunk(lane));
    b_src[d] = (uint32_t)((int64_t)gn * p.ldb * (BF ? 2 : 1)) + chunk * 16;
  }
  // the activations' stage (BF: pair) `u` / the weights' pair into ring slot
  // `slot`; gemm_addr.h keeps every load inside its row
  const int a_units = BF ? KT >> 1 : KT, b_units = FP4 ? (KT + 3) >> 2 : stage_pairs(KT);
  auto dma_a = [&](int u, int slot) __attribute__((always_inline)) {
    u = clamp_unit(u, a_units);
#pragma unroll
    for (int d = 0; d < A_DMA; ++d)
      buffer_dma16(p.A, a_records, a_src[d], u * A_ROWB, lds + slot * A_BYTES + (LOADERS * d + loader) * 1024);
  };
  auto dma_b = [&](int u, int slot) __attribute__((always_inline)) {
    u = clamp_unit(u, b_units);
    if constexpr (FP4) {
      const int rem = KT & 3;
      if (rem != 0 && u == b_units - 1) {  // lanes of missing stages load the unit's first
#pragma unroll
        for (int d = 0; d < B_DMA; ++d) {
          const int r = 8 * (LOADERS * d + loader) + (lane >> 3);
          const int chunk = (lane & 7) ^ ((r >> 1) & 7);
          const uint32_t back = (chunk >> 1) >= rem ? (uint32_t)(chunk & ~1) * 16 : 0u;
          buffer_dma16(p.B, b_records, b_src[d] - back, u * B_ROWB,
                       lds + B_REGION + slot * B_BYTES + (LOADERS * d + loader) * 1024);
        }
        return;
      }
    }
    if constexpr (BKIND == B_INT8) {  // bf16: 32-deep stages, MXFP8: whole octets -- always even counts
      if (half_pair(u, KT)) {
        const uint32_t back = half_pair_back(lane);
#pragma unroll
        for (int d = 0; d < B_DMA; ++d)
          buffer_dma16(p.B, b_records, b_src[d] - back, u * B_ROWB,
                       lds + B_REGION + slot * B_BYTES + (LOADERS * d + loader) * 1024);
        return;
      }
    }
#pragma unroll
    for (int d = 0; d < B_DMA; ++d)
      buffer_dma16(p.B, b_records, b_src[d], u * B_ROWB,
                   lds + B_REGION + slot * B_BYTES + (LOADERS * d + loader) * 1024);
  };
  auto dma_stage = [&](int kt, int buf) __attribute__((always_inline)) {
    char* As = lds + buf * A_BYTES;
    char* Bs = lds + B_REGION + buf * B_BYTES;
#pragma unroll
    for (int d = 0; d < A_DMA; ++d)
      buffer_dma16(p.A, a_records, a_src[d], kt * Cfg::A_ROWB, As + (8 * d + wave) * 1024);
#pragma unroll
    for (int d = 0; d < B_DMA; ++d)
      buffer_dma16(p.B, b_records, b_src[d], kt * Cfg::B_ROWB, Bs + (8 * d + wave) * 1024);
  };

  // ---- per-lane fragment read bases: LDS byte addresses of the lane's first
  // fragment per XOR pattern, so that every fragment read is base + immediate.
  // MX (32x32x64): lane (row fr, half h) reads chunk 2 pp + h of its 64-byte
  // code rows for the stage's k-step pair pp, both operands.
  const int fr = lane & 31, h = lane >> 5;
  const int b_swz = g8_swz64(fr, false);
  int b_base[2], a_mx[2];
#pragma unroll
  for (int pp = 0; pp < 2; ++pp) {
    b_base[pp] = B_REGION + (wn * WN + fr) * B_ROWB + (((2 * pp + h) ^ b_swz) * 16);
    a_mx[pp] = (wm * WM + fr) * A_ROWB + (((2 * pp + h) ^ b_swz) * 16);
  }
  // 16x16x32 fragments: lane (r16, q) = row r16 of a 16-row block, k-quarter
  // q.  Weights: one 16-byte read per block and stage, chunk q of the stage's
  // half row (8-bit codes: k = 16 q + [0, 16), both k-steps).  8-bit codes:
  // k-step s of the stage is k = 16 q + 8 s + [0, 8) in lane q for both operands
  // -- the activation fragment is chunk 2 q + s of the 128-byte row -- so the
  // E8M0 block of a lane's codes is q / 2 in both k-steps.  Every 16 lanes read
  // 16 consecutive rows of one logical chunk (conflict-free under swz_pair and
  // g8_swz128 of the 16x16 form; the row's bits 0-3 are those of r16).
  // The activation bases come as a low / high pair (stage buffers 0-1 / 1-2
  // of the 8-bit-code ring) so that the offsets fit the 16-bit immediate.
  const int r16 = lane & 15, q = lane >> 4;
  // Pairs: chunk 4 s + q of a row is the lane's fragment of the pair's stage s;
  // the weights' bases as a low / high pair too (slots 0 and 1-2).
  int x16_lo[2], x16_hi[2], w16_lo[2], w16_hi[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int pair_chunk = ((4 * s + q) ^ swz_pair(r16)) * 16;
    x16_lo[s] = (wm * WM + r16) * A_ROWB + (BF ? pair_chunk : ((2 * q + s) ^ g8_swz128(r16, true)) * 16);
    x16_hi[s] = x16_lo[s] + A_BYTES;
    w16_lo[s] = B_REGION + (wn * WN + r16) * B_ROWB + pair_chunk;
    w16_hi[s] = w16_lo[s] + B_BYTES;
  }
  // MXFP4: the lane's 8 bytes of stage s of a unit, half q & 1 of chunk 2 s + q / 2
  int w4_rd[FP4 ? 4 : 1];
  if constexpr (FP4) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      w4_rd[s] = B_REGION + (wn * WN + r16) * B_ROWB + ((2 * s + (q >> 1)) ^ (r16 >> 1)) * 16 + (q & 1) * 8;
  }
  // MXFP8 scales reach LDS by direct loads too, eight stages at a time: the
  // loop then holds no register-destined global load, whose first use would
  // make the compiler wait for every load in flight (its wait counting does
  // not see the direct loads).  Octet o of a tile is 256 weight rows x 16
  // bytes (the E8M0 of k-blocks 16o..16o+15, i.e. stages 8o..8o+7), laid out
  // [row][16]; the four waves of group 1, which moves the codes, take 64 rows
  // per octet each.  int8: the row scale in a register.
  // MX: group 0 moves the weights' octets, group 1 the activations' (256
  // activation rows x 16 bytes, after the weights' two octet buffers).
  char* const sc_lds = lds + Cfg::SC_OFF;
  // MXFP4: an octet is four rows of 256 scale words, one per wave of group 1.
  constexpr bool SCALED = BKIND == B_MXFP8 || MX || FP4;
  const int sc_words = (p.K + 127) >> 7;
  const int sc_records = FP4 ? (int)word_bytes(sc_words, p.ld_scale, p.N) : (SCALED ? (int)((int64_t)p.N * p.ld_scale) : 0);
  const int asc_records = MX ? (int)((int64_t)p.M * p.ld_ascale) : 0;
  const int sc_read = Cfg::SC_OFF + (wn * WN + (S16 ? r16 : fr)) * (FP4 ? 4 : 16);
  const int asc_read = Cfg::SC_OFF + 2 * Cfg::SC_OCT + (wm * WM + fr) * 16;
  uint32_t sc_src = 0;
  if constexpr (FP4) {
    sc_src = (uint32_t)word_piece(n0 + 4 * lane, p.N) * 4;
  } else if (grp == 0 || !MX) {
    int gn = n0 + (wave & 3) * 64 + lane;
    gn = gn < p.N ? gn : p.N - 1;
    sc_src = (uint32_t)((int64_t)gn * p.ld_scale);
  } else {
    int gm = m0 + (wave & 3) * 64 + lane;
    gm = gm < p.M ? gm : p.M - 1;
    sc_src = (uint32_t)((int64_t)gm * p.ld_ascale);
  }
  const int noct = KT >> 3;
  auto dma_scales = [&](int oct) {
    if constexpr (FP4) {
      int w = oct * 4 + (wave & 3);
      w = w < sc_words ? w : sc_words - 1;  // past the end: the last row again
      buffer_dma16(p.bscale, sc_records, sc_src + (uint32_t)((int64_t)w * p.ld_scale * 4), 0,
                   sc_lds + (oct & 1) * Cfg::SC_OCT + (wave & 3) * 1024);
    } else if constexpr (SCALED) {
      oct = oct < noct ? oct : noct - 1;  // past the end: re-read the last octet
      if (W8 || grp == 0)  // W8: called by group 1 only
        buffer_dma16(p.bscale, sc_records, sc_src, oct * 16, sc_lds + (oct & 1) * Cfg::SC_OCT + (wave & 3) * 1024);
      else if (MX)
        buffer_dma16(p.ascale, asc_records, sc_src, oct * 16,
                     sc_lds + (2 + (oct & 1)) * Cfg::SC_OCT + (wave & 3) * 1024);
    }
  };
  // weight row blocks of a wave: TN of 32 rows, or (S16) TN16 of 16
  constexpr int NWB = S16 ? TN16 : TN, WB_ROWS = S16 ? 16 : 32;
  float s_i8[NWB];
#pragma unroll
  for (int j = 0; j < NWB; ++j) {
    int gn = n0 + wn * WN + j * WB_ROWS + (S16 ? r16 : fr);
    gn = gn < p.N ? gn : p.N - 1;
    if (BKIND == B_INT8) s_i8[j] = ((const float*)p.bscale)[gn];
  }
  uint32_t scw[NWB];  // this stage pair's E8M0 bytes of the lane's weight rows
  // global memory instructions of a stage's first memory cluster: the direct
  // loads of stage kt+2, plus (group 0, MXFP8) the scales in the first stage
  // of an octet
  constexpr int VM_DMA = A_DMA + B_DMA;
  constexpr int VM_SCALES = SCALED ? 1 : 0;

  // MX: the scaled 32x32x64 fragments
  u32x4 fb[2][MX ? TN : 1];   // weight codes of the stage's two k-step pairs (16 per lane)
  u32x4 fa8[2][MX ? TM : 1];  // activation codes, read like the weight codes
  uint32_t sca[MX ? TM : 1];  // this stage pair's E8M0 bytes of the lane's activation rows
  // 16x16x32: the stage's weight fragments (codes, or bf16 weights) and its
  // activation fragments per k-step
  constexpr int XS = BF ? 1 : 2;
  u32x4 w16f[S16 && !FP4 ? TN16 : 1];
  u32x2 w4f[FP4 ? TN16 : 1];
  bf16x8 x16f[XS][S16 ? TM16 : 1];
  // fragment reads of stage kt, which sits in buffer BUF (compile-time)
  auto read_stage = [&](int kt, auto bufc) __attribute__((always_inline)) {
    constexpr int BUF = decltype(bufc)::value;
    if constexpr (SCALED) {
      const int sa = sc_read + ((kt >> 3) & 1) * Cfg::SC_OCT + ((kt & 7) >> 1) * (FP4 ? 1024 : 4);
#pragma unroll
      for (int j = 0; j < NWB; ++j)
        scw[j] = *reinterpret_cast<const uint32_t*>(lds + sa + j * WB_ROWS * (FP4 ? 4 : 16));
    }
    if constexpr (MX) {
      const int sa = asc_read + ((kt >> 3) & 1) * Cfg::SC_OCT + ((kt & 7) >> 1) * 4;
#pragma unroll
      for (int i = 0; i < TM; ++i) sca[i] = *reinterpret_cast<const uint32_t*>(lds + sa + i * 32 * 16);
#pragma unroll
      for (int pp = 0; pp < 2; ++pp) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
          fb[pp][j] = *reinterpret_cast<const u32x4*>(lds + b_base[pp] + BUF * B_BYTES + j * 32 * B_ROWB);
#pragma unroll
        for (int i = 0; i < TM; ++i)
          fa8[pp][i] = *reinterpret_cast<const u32x4*>(lds + a_mx[pp] + BUF * A_BYTES + i * 32 * A_ROWB);
      }
    } else {
      // BUF = kt % STAGES: the weights in slot BUF / 2 % BP, the activations
      // in slot BUF / 2 % AP (BF) or BUF % AP
      // (MXFP4: in slot BUF / 4 % BP)
      constexpr int SA = (BF ? BUF / 2 : BUF) % AP, SB = BUF / BU % BP, S = BUF & 1;
      if constexpr (FP4) {
#pragma unroll
        for (int jb = 0; jb < TN16; ++jb)
          w4f[jb] = *reinterpret_cast<const u32x2*>(lds + w4_rd[BUF % BU] + SB * B_BYTES + jb * 16 * B_ROWB);
      } else {
        const int wb = SB == 0 ? w16_lo[S] : w16_hi[S] + (SB - 1) * B_BYTES;
#pragma unroll
        for (int jb = 0; jb < TN16; ++jb) w16f[jb] = *reinterpret_cast<const u32x4*>(lds + wb + jb * 16 * B_ROWB);
      }
#pragma unroll
      for (int s = 0; s < XS; ++s) {
        const int h = BF ? S : s;
        const int xb = SA == 0 ? x16_lo[h] : x16_hi[h] + (SA - 1) * A_BYTES;
#pragma unroll
        for (int ib = 0; ib < TM16; ++ib) x16f[s][ib] = *reinterpret_cast<const bf16x8*>(lds + xb + ib * 16 * A_ROWB);
      }
    }
  };

  // accumulators: (32x32) TM x TN blocks of 16 values, or (16x16) TM16 x TN16
  // blocks of 4 -- the same 128 per lane
  constexpr int AM = S16 ? TM16 : TM, AN = S16 ? TN16 : TN, AE = S16 ? 4 : 16;
  using AccT = std::conditional_t<S16, f32x4, f32x16>;
  AccT acc[AM][AN];
#pragma unroll
  for (int i = 0; i < AM; ++i)
#pragma unroll
    for (int j = 0; j < AN; ++j)
#pragma unroll
      for (int e = 0; e < AE; ++e) acc[i][j][e] = 0.0f;

  // codes of one k-step (two 4-byte words) -> bf16 fragment
  auto dequant = [&](uint32_t w0, uint32_t w1, float sc) -> bf16x8 {
    uint32_t o[4];
    if constexpr (BKIND == B_MXFP8) {
      o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, sc, false));
      o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, sc, true));
      o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, sc, false));
      o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, sc, true));
    } else {
      // bf16(fp32(q * s)): each signed byte converted by one sign-extending
      // byte-select conversion, one fp32 product (a single rounding), then
      // two values per bf16 conversion
      const uint32_t ws[2] = {w0, w1};
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const uint32_t u = ws[d];
        bf16x2 p0, p1;
        p0[0] = (bf16)((float)(int8_t)u * sc);
        p0[1] = (bf16)((float)(int8_t)(u >> 8) * sc);
        p1[0] = (bf16)((float)(int8_t)(u >> 16) * sc);
        p1[1] = (bf16)((float)((int32_t)u >> 24) * sc);
        o[2 * d] = __builtin_bit_cast(uint32_t, p0);
        o[2 * d + 1] = __builtin_bit_cast(uint32_t, p1);
      }
    }
    return __builtin_bit_cast(bf16x8, u32x4{o[0], o[1], o[2], o[3]});
  };

  // Weight fragment f of a stage (k-step f / TN16, row block f % TN16) in two
  // alternating register sets; the scale of each row block (its E8M0 byte of
  // the lane's k-block q / 2, or the int8 row scale) set once per stage.
  float scf[NWB];
  bf16x8 bq[2];
  constexpr int NF = XS * TN16;
  const int q_sh = 8 * (q >> 1);
  auto frag_dequant = [&](int f) -> bf16x8 {
    const int s = f / TN16, jb = f % TN16;
    if constexpr (FP4) return fp4x8_bf16(w4f[jb][s], scf[jb]);
    else return dequant(w16f[jb][2 * s], w16f[jb][2 * s + 1], scf[jb]);
  };
  // end of the memory cluster of stage kt (its fragment reads have landed):
  // the stage's scales and fragments 0 and 1 (MX, bf16: nothing to decode)
  auto prep_stage = [&](int kt) __attribute__((always_inline)) {
    if constexpr (MX || BF) return;
#pragma unroll
    for (int j = 0; j < NWB; ++j) {
      if constexpr (BKIND == B_MXFP8 || FP4)
        scf[j] = e8m0_to_f32_valu(__builtin_amdgcn_ubfe(scw[j], 16 * (kt & 1) + q_sh, 8));
      else
        scf[j] = s_i8[j];
    }
    bq[0] = frag_dequant(0);
    bq[1] = frag_dequant(1);
  };
  // compute cluster of stage kt.  8-bit codes: 2 k-steps x TN16 weight
  // fragments x TM16 MFMAs; fragment f+1 (f >= 1) is dequantised while the
  // MFMAs of fragment f run.  bf16: TN16 x TM16 MFMAs of the stage's 32 k.
  // MX: TN x TM scaled fp8 MFMAs of 64 k.  Their operand contract (probed on
  // the device): lane (row r, half h) holds k = 16h + [0, 16) in bytes 0-15
  // and k = 32 + 16h + [0, 16) in bytes 16-31 -- the two 16-byte code chunks
  // h and 2 + h of the row, as read above -- and lane r + 32b carries the
  // E8M0 scale of row r's k-block b (opsel 0: bits 0-7).  The stage's two
  // blocks are bytes 2 (kt & 1) + b of the octet word.
  auto compute_stage = [&](int kt) __attribute__((always_inline)) {
    if constexpr (MX) {
      const int sh = 16 * (kt & 1) + 8 * h;
      int ws[TN], as[TM];
#pragma unroll
      for (int j = 0; j < TN; ++j) ws[j] = (int)(scw[j] >> sh);
#pragma unroll
      for (int i = 0; i < TM; ++i) as[i] = (int)(sca[i] >> sh);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const i32x8 w = __builtin_bit_cast(i32x8, __builtin_shufflevector(fb[0][j], fb[1][j], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const i32x8 a =
              __builtin_bit_cast(i32x8, __builtin_shufflevector(fa8[0][i], fa8[1][i], 0, 1, 2, 3, 4, 5, 6, 7));
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, acc[i][j], 0, 0, 0, ws[j], 0, as[i]);
        }
      }
    } else if constexpr (BF) {
#pragma unroll
      for (int jb = 0; jb < TN16; ++jb)
#pragma unroll
        for (int ib = 0; ib < TM16; ++ib)
          acc[ib][jb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w16f[jb]), x16f[0][ib],
                                                                acc[ib][jb], 0, 0, 0);
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int s = f / TN16, jb = f % TN16;
        if (f >= 1 && f + 1 < NF) bq[(f + 1) & 1] = frag_dequant(f + 1);
#pragma unroll
        for (int ib = 0; ib < TM16; ++ib)
          acc[ib][jb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bq[f & 1], x16f[s][ib], acc[ib][jb], 0, 0, 0);
      }
    }
  };

  // ---- prologue: scales of octet 0 and all slots but one in flight, the first
  // stage landed, then one barrier for all waves
  // loads in flight when those of a pair (W8: a stage of the activations) must
  // have landed: BF those of the AP - 2 activation pairs and of the one weight
  // pair after it, W8 those of the AP - 2 stages or BP - 2 pairs after it
  constexpr int BF_FLIGHT = (AP - 2) * A_DMA + B_DMA;
  constexpr int A_FLIGHT = (AP - 2) * A_DMA, B_FLIGHT = (BP - 2) * B_DMA;
  if constexpr (BF) {
    dma_a(0, 0);
    dma_b(0, 0);
    if constexpr (AP == 3) dma_a(1, 1);
    dma_b(1, 1);
    wait_vmcnt<BF_FLIGHT>();
    barrier_nofence();
  } else if constexpr (W8) {
    if (grp == 0) {
      static_for<0, AP - 1>([&](auto ic) { dma_a(decltype(ic)::value, decltype(ic)::value); });
      wait_vmcnt<A_FLIGHT>();
    } else {
      dma_scales(0);
      static_for<0, BP - 1>([&](auto ic) { dma_b(decltype(ic)::value, decltype(ic)::value); });
      wait_vmcnt<B_FLIGHT>();
    }
    barrier_nofence();
  } else {
    dma_scales(0);
    dma_stage(0, 0);
    if (KT > 1) dma_stage(1, 1);
    wait_vmcnt<0>();
    __syncthreads();
  }
  if (grp == 1) barrier_nofence();  // group 1 runs half a stage behind

  // Clusters are whole stages.  Stage s is first read by group 0's memory
  // cluster of stage s (global half-stage 2s), so its data must be in LDS by
  // the barrier before it.  Direct loads go into the slot that stage s-1 left,
  // in the memory cluster of stage s; each group waits for them in its last
  // cluster before that barrier -- group 0 at the end of its compute cluster
  // of stage s-1, group 1 at the end of its memory cluster of stage s-1 --
  // leaving only the loads of later stages in flight.  Past the last stage the
  // direct loads re-read the last one into the buffer nobody reads any more,
  // so every stage issues the same loads and the waits are exact.  The scales
  // of octet o+1 go out with stage 8o's loads (8-bit weights: by group 1; MX:
  // by both groups, an operand each).
  // BF: the memory cluster of a pair's first stage issues the activations'
  // next free pair, that of its second stage the weights'; only the last
  // stage of a pair waits, for the next pair.
  // The loop is compiled once per group (GRP), so the group-specific waits
  // and scale loads are resolved at compile time.
  auto stage_iter = [&](int kt, auto bufc, auto grpc) __attribute__((always_inline)) {
    constexpr int BUF = decltype(bufc)::value;
    constexpr int GRP = decltype(grpc)::value;
    const bool oct_start = SCALED && (kt & 7) == 0;
    constexpr bool PAIR_END = (BUF & 1) != 0;
    // W8: the weights' unit (a pair; MXFP4: four stages)
    constexpr bool UNIT_START = BUF % BU == 0, UNIT_END = BUF % BU == BU - 1;
    // memory cluster (MX: group 1 moves the activations' scale octets)
    if constexpr (BF) {
      if (PAIR_END) dma_b((kt >> 1) + BP - 1, (BUF / 2 + BP - 1) % BP);
      else dma_a((kt >> 1) + AP - 1, (BUF / 2 + AP - 1) % AP);
    } else if constexpr (W8) {
      if constexpr (GRP == 0) {
        dma_a(kt + AP - 1, (BUF + AP - 1) % AP);
      } else {
        if (oct_start) dma_scales((kt >> 3) + 1);
        if (UNIT_START) dma_b(kt / BU + BP - 1, (BUF / BU + BP - 1) % BP);
      }
    } else {
      if (oct_start) dma_scales((kt >> 3) + 1);
      dma_stage(kt + 2 < KT ? kt + 2 : KT - 1, (BUF + 2) % STAGES);
    }
    if (live) read_stage(kt, bufc);
    wait_lgkmcnt0();
    if (live) prep_stage(kt);
    if (GRP == 1) {
      if constexpr (BF) {
        if (PAIR_END) wait_vmcnt<BF_FLIGHT>();
      } else if constexpr (W8) {
        if (UNIT_END) wait_vmcnt<B_FLIGHT>();
      } else if (oct_start) {
        wait_vmcnt<VM_DMA + VM_SCALES>();
      } else {
        wait_vmcnt<VM_DMA>();
      }
    }
    barrier_nofence();
    // compute cluster
    __builtin_amdgcn_s_setprio(1);
    if (live) compute_stage(kt);
    __builtin_amdgcn_s_setprio(0);
    if (GRP == 0) {
      if constexpr (BF) {
        if (PAIR_END) wait_vmcnt<BF_FLIGHT>();
      } else if constexpr (W8) {
        wait_vmcnt<A_FLIGHT>();
      } else if (oct_start) {
        wait_vmcnt<VM_DMA + VM_SCALES>();
      } else {
        wait_vmcnt<VM_DMA>();
      }
    }
    barrier_nofence();
  };
  // the loop unrolled over one turn of the rings, then the remainder (stage
  // kt + i sits in buffer i; BF: i / 2 counts pairs)
  auto main_loop = [&](auto grpc) __attribute__((always_inline)) {
    int kt = 0;
    for (; kt + STAGES - 1 < KT; kt += STAGES)
      static_for<0, STAGES>([&](auto ic) { stage_iter(kt + decltype(ic)::value, ic, grpc); });
    static_for<0, STAGES - 1>([&](auto ic) {
      if (kt + decltype(ic)::value < KT) stage_iter(kt + decltype(ic)::value, ic, grpc);
    });
  };
  if (grp == 0) main_loop(std::integral_constant<int, 0>{});
  else main_loop(std::integral_constant<int, 1>{});
  if (grp == 0) barrier_nofence();
  wait_vmcnt<0>();
  // column values inside the ring: every wave's last direct loads have landed
  if constexpr (Cfg::COL_IN_RING) __syncthreads();

  // ---- epilogue (every wave is past its last LDS fragment read)
  if (tid < BN) {
    float col_bias = 0.0f, col_gate = 0.0f;
    if (n0 + tid < p.N) {
      if (p.bias) col_bias = p.bias[n0 + tid];
      if (RESID) col_gate = p.gate[n0 + tid];
    }
    col_lds[tid] = col_bias;
    col_lds[BN + tid] = col_gate;
  }
  __syncthreads();
  constexpr int CHUNKS = WN / 8;
  constexpr int ROWS_PER_IT = 64 / CHUNKS;
  constexpr int ITS = WM / ROWS_PER_IT;
  const int ch = lane % CHUNKS;
  const int rsub = lane / CHUNKS;
  const int gn2 = n0 + wn * WN + ch * 8;
  const bool col_ok = gn2 < p.N;
  char* E = lds + wave * EPI_WAVE;
  if constexpr (FP4 && RESID) {
    static_assert(EPI_WAVE == TM16 / 2 * 4096 && WN == 64, "half the row blocks per pass");
    fp4_residual_rows<EPI, TM16, TM16 / 2>(
        p, E, col_lds + wn * WN, col_lds + BN + wn * WN, m0 + wm * WM, n0 + wn * WN, lane,
        [&](int i, int j) __attribute__((always_inline)) { return acc[i][j]; });
    return;
  }
  auto phase1 = [&](auto sig_tag, auto rtb_tag) {
    constexpr bool SIG = decltype(sig_tag)::value;
    constexpr bool RTB = decltype(rtb_tag)::value;
    // accumulator block (i, j), values 4 g .. 4 g + 3: output columns nl ..
    // nl + 3 of tile row (32x32) i * 32 + fr, or (16x16) i * 16 + r16
#pragma unroll
    for (int j = 0; j < AN; ++j) {
#pragma unroll
      for (int g = 0; g < AE / 4; ++g) {
        const int nl = S16 ? j * 16 + 4 * q : j * 32 + 8 * g + 4 * h;
        const int gn = n0 + wn * WN + nl;
        const f32x4 bias4 = *reinterpret_cast<const f32x4*>(col_lds + wn * WN + nl);
#pragma unroll
        for (int i = 0; i < AM; ++i) {
          // bf16 roundings two at a time (one conversion per pair)
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = acc[i][j][4 * g + e];
          if (RTB) {
            round_bf2(y[0], y[1]);
            round_bf2(y[2], y[3]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] += bias4[e];
          if (EPI == LTX_GEMM_EPI_GELU || EPI == kEpiGeluMx || EPI == LTX_GEMM_EPI_SIGMOID2 || SIG) {
            float r[4] = {y[0], y[1], y[2], y[3]};
            if constexpr (!FP4) {  // MXFP4 reproduces no reference rounding here
              round_bf2(r[0], r[1]);
              round_bf2(r[2], r[3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (EPI == LTX_GEMM_EPI_GELU || EPI == kEpiGeluMx) y[e] = gelu_tanh(r[e]);
              if (EPI == LTX_GEMM_EPI_SIGMOID2) y[e] = sigmoid2_bf(r[e]);
              if (SIG && gn + e >= p.sig_from) y[e] = sigmoid2_bf(r[e]);
            }
          }
          bf16x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (bf16)y[e];
          if constexpr (S16) {
            const int row = i * 16 + r16;
            *reinterpret_cast<bf16x4*>(E + row * EPI_ROWB + ((((nl >> 3) ^ (row >> 1)) & 7) << 4) + (nl & 7) * 2) = v;
          } else {
            *reinterpret_cast<bf16x4*>(E + (i * 32 + fr) * EPI_ROWB + nl * 2) = v;
          }
        }
      }
    }
  };
  const bool sig = EPI == LTX_GEMM_EPI_BIAS && n0 + wn * WN + WN > p.sig_from;
  if (p.round_then_bias) {
    if (sig) phase1(std::true_type{}, std::true_type{});
    else phase1(std::false_type{}, std::true_type{});
  } else {
    if (sig) phase1(std::true_type{}, std::false_type{});
    else phase1(std::false_type{}, std::false_type{});
  }
  // residual rows after the accumulators are in LDS (fewer live registers);
  // every residual element of the tile is read before its output is written
  bf16x8 res[RESID ? ITS : 1];
  if constexpr (RESID) {
    const int gnc = col_ok ? gn2 : 0;
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
      int gm = m0 + wm * WM + it * ROWS_PER_IT + rsub;
      gm = gm < p.M ? gm : p.M - 1;
      res[it] = *reinterpret_cast<const bf16x8*>(p.R + (int64_t)gm * p.ldr + gnc);
    }
  }
  __syncthreads();
  float g8[8];
  if constexpr (RESID) {
    const f32x4 ga = *reinterpret_cast<const f32x4*>(col_lds + BN + wn * WN + ch * 8);
    const f32x4 gb = *reinterpret_cast<const f32x4*>(col_lds + BN + wn * WN + ch * 8 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g8[e] = ga[e];
      g8[4 + e] = gb[e];
    }
  }
#pragma unroll
  for (int it = 0; it < ITS; ++it) {
    const int ml = it * ROWS_PER_IT + rsub;
    const int gm = m0 + wm * WM + ml;
    bf16x8 v = *reinterpret_cast<const bf16x8*>(E + ml * EPI_ROWB + (S16 ? ((ch ^ (ml >> 1)) & 7) : ch) * 16);
    if constexpr (RESID) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = (float)v[e];
        float o;
        if (EPI == LTX_GEMM_EPI_RESIDUAL)
          o = fmaf(g8[e], y, (float)res[it][e]);
        else
          o = round_bf(y * g8[e]) + (float)res[it][e];
        v[e] = (bf16)o;
      }
    }
    if constexpr (EPI == kEpiGeluMx) {
      // the row's 32-column block spans lanes ch & ~3 .. ch | 3 (N % 32 == 0:
      // a block lies wholly inside or outside the output); its maximum takes
      // two lane exchanges, then 8 codes per lane and one scale byte per block
      float f[8], amax = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = (float)v[e];
        amax = fmaxf(amax, fabsf(f[e]));
      }
      amax = fmaxf(amax, __shfl_xor(amax, 1, 64));
      amax = fmaxf(amax, __shfl_xor(amax, 2, 64));
      const int X = mxfp8_block_exponent(amax);
      const float sx = ldexpf(1.0f, X), lim = 448.0f * sx;
      const uint32_t w0 = e4m3x4_ocp(f[0], f[1], f[2], f[3], sx, lim);
      const uint32_t w1 = e4m3x4_ocp(f[4], f[5], f[6], f[7], sx, lim);
      if (gm < p.M && col_ok) {
        uint8_t* cq = reinterpret_cast<uint8_t*>(p.C);
        *reinterpret_cast<u32x2*>(cq + (int64_t)gm * p.ldc + gn2) = u32x2{w0, w1};
        if ((ch & 3) == 0) p.cscale[(int64_t)gm * p.ld_cscale + gn2 / 32] = (uint8_t)(X + 127);
      }
    } else {
      if (gm < p.M && col_ok) *reinterpret_cast<bf16x8*>(p.C + (int64_t)gm * p.ldc + gn2) = v;
    }
    if constexpr (EPI == LTX_GEMM_EPI_BIAS) {
      // the row's sum of squares over this wave's 64 columns: eight per lane,
      // then over the row's eight lanes (consecutive: lane = 8 rsub + ch)
      if (p.rowss != nullptr && n0 + wn * WN < p.ss_cols) {
        float q = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = (float)v[e];
          q = fmaf(f, f, q);
        }
        q += __shfl_xor(q, 1, 64);
        q += __shfl_xor(q, 2, 64);
        q += __shfl_xor(q, 4, 64);
        if (ch == 0 && gm < p.M) p.rowss[(int64_t)gm * p.ld_rowss + (n0 + wn * WN) / WN] = q;
      }
    }
  }
}

template <int BKIND, int EPI, int BM = 256>
static void launch_g8(GemmArgs p, hipStream_t s) {
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + 255) / 256;
  gemm8_kernel<BKIND, EPI, BM><<<p.tiles_m * p.tiles_n, kG8Threads, 0, s>>>(p);
}

// Whether the 8-wave kernel takes a problem: operand extents within its 31-bit
// buffer record counts; for MXFP8 whole eight-stage scale octets (K % 512) in
// 16-byte aligned pieces.
template <int BKIND>
static bool g8_ok(const GemmArgs& p) {
  // operand extents are 31-bit buffer record counts in the kernel
  if ((int64_t)p.M * p.lda * (BKIND == B_MX ? 1 : 2) >= ((int64_t)1 << 31) ||
      (int64_t)p.N * p.ldb * (BKIND == B_BF16 ? 2 : 1) >= ((int64_t)1 << 31) ||
      (int64_t)p.N * p.ld_scale >= ((int64_t)1 << 31))
    return false;
  if (BKIND == B_MX)
    return p.K % 512 == 0 && p.ld_scale % 16 == 0 && ((uintptr_t)p.bscale & 15u) == 0 &&
           p.ld_ascale % 16 == 0 && ((uintptr_t)p.ascale & 15u) == 0 &&
           (int64_t)p.M * p.ld_ascale < ((int64_t)1 << 31);
  if (BKIND == B_MXFP8)
    return p.K % 512 == 0 && p.ld_scale % 16 == 0 && ((uintptr_t)p.bscale & 15u) == 0;
  return true;
}

// Automatic 8-wave launches split M when that shortens a partial last round:
// rows [0, r0) in 256-row tiles, rows [r0, M) in 128-row tiles by a second
// launch of the 128-row form (same per-element arithmetic, bit-identical
// outputs).  Cost model in rounds of one workgroup per CU on the MI355X's
// 256 CUs: a round of 128-row tiles takes 0.67 of a 256-row round (FF up
// alone: 1728 tiles of 128 rows in 7 rounds, 436 us, against 896 of 256 rows
// in 4 rounds, 373 us).  At M = 3456 the FF up-projection (14 x 64 tiles =
// 3.5 rounds, i.e. 4) runs 12 tile rows of 256 (3 rounds) plus 3 of 128
// (one partial round): 392.5 -> 373.1 us alone.  A split must model >= 3 %
// faster; r0 = M means one launch.
constexpr int kG8Cus = 256;
static inline int g8_split_rows(int M, int N) {
  const int64_t tn = (N + 255) / 256, tm = (M + 255) / 256;
  auto rounds = [](int64_t tiles) { return (double)((tiles + kG8Cus - 1) / kG8Cus); };
  const double one = rounds(tm * tn);
  double best = one;
  int r0 = M;
  for (int64_t b = tm - 1; b >= 1 && b >= tm - 8; --b) {
    const int64_t small = (M - 256 * b + 127) / 128;
    const double t = rounds(b * tn) + 0.67 * rounds(small * tn);
    if (t < best && t < 0.97 * one) {
      best = t;
      r0 = (int)(256 * b);
    }
  }
  return r0;
}
// The rows [r0, M) of a product: the same operands from row r0 on.
static inline GemmArgs rows_from(const GemmArgs& p, int64_t r0) {
  GemmArgs q = p;
  q.A = p.A + (int64_t)r0 * p.lda;
  q.C = p.C + (int64_t)r0 * p.ldc;
  if (p.R) q.R = p.R + (int64_t)r0 * p.ldr;
  if (p.rowss) q.rowss = p.rowss + (int64_t)r0 * p.ld_rowss;
  q.M = (int)(p.M - r0);
  return q;
}

}  // namespace ltx
