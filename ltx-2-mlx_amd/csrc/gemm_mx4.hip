// Projection GEMMs of MXFP4 rows and MXFP4 weights on the scaled FP4 MFMA
// (v_mfma_scale_f32_32x32x64_f8f6f4):
//
//   C[m, n] = epilogue( sum_k a[m, k] w[n, k] + bias[n] ),
//   a = e2m1(A) 2^(XA), w = e2m1(W) 2^(XW), a scale per 32 k on both sides.
//
// Operand storage: gemm_fp4.h.
//
// A workgroup computes a BM x BN tile.  A stage is 256 k: rows of 128 code bytes,
// one line each, and two scale words per row; stages reach LDS by direct loads
// into a ring of NST.  A stage has four k-steps of 64; lane (row r32, half h) of a
// fragment holds the 16 bytes of its row's block h, and its scale operand that
// block's byte.  The fragments of the next k-step are read while the MFMAs of the
// current one run, also across the one barrier per stage.
//
// What bounds it: a stage of 256 x 256 tiles takes 1.69-1.74 us with every CU busy,
// 4.9-5.1 PFLOP/s (4096 x K -> 4096 and 6144 x K -> 16384, over K), 1.58 on 224 CUs
// (3456 x 16384 -> 4096: 109-114 us in all, 4.1-4.25 PFLOP/s).  A loop of nothing but
// these MFMAs on random codes reaches 5.9-6.4 at the chip's power limit (9.8 on
// zeros; this kernel whole, 3456 x 16384 -> 4096, 5.6); its loads and fragment reads
// alone take 1.15 us per stage, the MFMAs without loads 1.65.  First loads and
// epilogue take 5.5 us a round with no MFMAs beside them, one workgroup per CU, and
// GELU 4 more: 60 of the 222 us of 6144 x 4096 -> 16384.  Measured beside it: the 16 x 16 x 128 form 117 us; four
// waves of 128 x 128 117 (a third less LDS traffic); all loads in one k-step 117
// against 113 for two; touching the lines two stages ahead, to take the L2
// misses off the loads, 116: no change.
#include "gemm_fp4.h"

namespace ltx {

template <int BM_, int BN_, int WAVES_M_, int WAVES_N_, int NST_>
struct M4Tile {
  static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, NST = NST_;
  static constexpr int WAVES = WAVES_M * WAVES_N, THREADS = WAVES * 64;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, AM = WM / 32, AN = WN / 32;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128;
  // two scale words per row; at least one direct-load instruction (1 KiB)
  static constexpr int SA_BYTES = BM * 8 < 1024 ? 1024 : BM * 8, SB_BYTES = BN * 8 < 1024 ? 1024 : BN * 8;
  static constexpr int B_OFF = A_BYTES, SA_OFF = B_OFF + B_BYTES, SB_OFF = SA_OFF + SA_BYTES;
  static constexpr int STAGE = SB_OFF + SB_BYTES;
  // direct loads of a wave per stage: code rows, and a share of the scales'
  static constexpr int A_DMA = BM / 8 / WAVES, B_DMA = BN / 8 / WAVES;
  static constexpr int SA_DMA = SA_BYTES / 1024, SB_DMA = SB_BYTES / 1024;
  // scale instructions go to the waves in turn, the same count for each (a
  // wave without one of its own repeats one)
  static constexpr int S_DMA = (SA_DMA + SB_DMA + WAVES - 1) / WAVES;
  static constexpr int DMA = A_DMA + B_DMA + S_DMA;
  // staged output rows of a wave: its tile as bf16; a residual's branch as fp32,
  // R_PASS 32-row blocks at a time
  static constexpr int EPI_ROWB = WN * 2, R_PASS = AM > 1 ? AM / 2 : 1, R_ROWB = WN * 4;
  static constexpr int EPI_WAVE = WM * EPI_ROWB > R_PASS * 32 * R_ROWB ? WM * EPI_ROWB : R_PASS * 32 * R_ROWB;
  static constexpr int RING = NST * STAGE, EPI = WAVES * EPI_WAVE;
  static constexpr int LDS_BYTES = RING > EPI ? RING : EPI;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole direct-load instructions per wave");
  static_assert(LDS_BYTES <= 160 * 1024 && (NST - 1) * DMA < 60, "LDS, vmcnt range");
};

template <class Cfg, int EPI>
__global__ __launch_bounds__(Cfg::THREADS, 1) void gemm_mx4_kernel(GemmArgs p, int k_split) {
  constexpr int BM = Cfg::BM, BN = Cfg::BN, WM = Cfg::WM, WN = Cfg::WN, AM = Cfg::AM, AN = Cfg::AN;
  constexpr int NST = Cfg::NST, A_DMA = Cfg::A_DMA, B_DMA = Cfg::B_DMA, WAVES = Cfg::WAVES;
  constexpr bool RESID = EPI == LTX_GEMM_EPI_RESIDUAL || EPI == LTX_GEMM_EPI_RESIDUAL_ROUND;
  __shared__ __attribute__((aligned(1024))) char lds[Cfg::LDS_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % Cfg::WAVES_M, wn = wave / Cfg::WAVES_M;
  const int r32 = lane & 31, h = lane >> 5;
  const int tiles = p.tiles_m * p.tiles_n;
  const int kz = EPI == kEpiPartial ? (int)blockIdx.x / tiles : 0;
  int tmi, tni;
  tile_coords(EPI == kEpiPartial ? (int)blockIdx.x % tiles : (int)blockIdx.x, tiles, p.tiles_m, p.tiles_n, tmi, tni);
  const int m0 = tmi * BM, n0 = tni * BN;
  const int k0 = kz * k_split;
  const int depth = p.K - k0 < k_split ? p.K - k0 : k_split;  // a multiple of 128
  const int T = (depth + 255) / 256;
  const bool half = (depth & 128) != 0;  // the last stage has one k-step

  // ---- direct-load sources (bytes from the operand's start).  Instruction d
  // of a wave fills 8 LDS rows of 128 bytes, lane j the 16-byte slot j & 7 of
  // row j >> 3 (pair_chunk: the chunk that the row's swizzle puts there).  Rows
  // past M / N re-read the last one.  A last half stage: the lanes of the
  // missing k-step load the other's bytes.
  const int a_records = (int)((int64_t)(p.M - 1) * p.lda + p.K / 2);
  const int b_records = (int)((int64_t)(p.N - 1) * p.ldb + p.K / 2);
  const int chunk = (lane & 7) ^ g8_swz128(8 * wave + (lane >> 3), false);  // (8 waves a multiple of 16 rows)
  const int back = (chunk & 4) * 16;
  uint32_t a_src[A_DMA], b_src[B_DMA];
#pragma unroll
  for (int d = 0; d < A_DMA; ++d) {
    int gm = m0 + 8 * (WAVES * d + wave) + (lane >> 3);
    gm = gm < p.M ? gm : p.M - 1;
    a_src[d] = (uint32_t)((int64_t)gm * p.lda + k0 / 2) + chunk * 16;
  }
#pragma unroll
  for (int d = 0; d < B_DMA; ++d) {
    int gn = n0 + 8 * (WAVES * d + wave) + (lane >> 3);
    gn = gn < p.N ? gn : p.N - 1;
    b_src[d] = (uint32_t)((int64_t)gn * p.ldb + k0 / 2) + chunk * 16;
  }
  // Scales: 16 bytes (4 rows' words) per lane.  Piece i of an operand's stage
  // (BM or BN words for each of the two k-steps) is words 4 i .. 4 i + 3.  Pieces
  // past the operand's rows (word_piece) and k-steps past the last re-read the last.
  constexpr int S_DMA = Cfg::S_DMA, SA_DMA = Cfg::SA_DMA, SB_DMA = Cfg::SB_DMA;
  const int words = p.K / 128;
  const void* s_base[S_DMA];
  int s_ld[S_DMA], s_dst[S_DMA];
  int s_row[S_DMA], s_ks[S_DMA], s_records[S_DMA];
#pragma unroll
  for (int d = 0; d < S_DMA; ++d) {
    int i = (WAVES * d + wave) % (SA_DMA + SB_DMA);  // the activations' instructions, then the weights'
    const bool of_a = i < SA_DMA;
    i = of_a ? i : i - SA_DMA;
    const int rows = of_a ? BM : BN, piece = i * 64 + lane;
    s_base[d] = of_a ? (const void*)p.ascale : p.bscale;
    s_ld[d] = (int)(of_a ? p.ld_ascale : p.ld_scale);
    s_dst[d] = (of_a ? Cfg::SA_OFF : Cfg::SB_OFF) + i * 1024;
    s_ks[d] = k0 / 128 + piece * 4 / rows;
    s_row[d] = word_piece((of_a ? m0 : n0) + piece * 4 % rows, of_a ? p.M : p.N);
    s_records[d] = (int)word_bytes(words, s_ld[d], of_a ? p.M : p.N);
  }
  // load instruction l of stage t: code rows, then scales
  auto load = [&](int t, int slot, int l) __attribute__((always_inline)) {
    t = t < T ? t : T - 1;
    char* S = lds + slot * Cfg::STAGE;
    const uint32_t bk = half && t == T - 1 ? back : 0;
    if (l < A_DMA) {
      buffer_dma16(p.A, a_records, a_src[l < A_DMA ? l : 0] - bk, t * 128, S + (WAVES * l + wave) * 1024);
    } else if (l < A_DMA + B_DMA) {
      const int d = l >= A_DMA && l < A_DMA + B_DMA ? l - A_DMA : 0;
      buffer_dma16(p.B, b_records, b_src[d] - bk, t * 128, S + Cfg::B_OFF + (WAVES * d + wave) * 1024);
    } else {
      const int d = l >= A_DMA + B_DMA ? l - A_DMA - B_DMA : 0;
      int kw = s_ks[d] + 2 * t;
      kw = kw < words ? kw : words - 1;
      buffer_dma16(s_base[d], s_records[d], (uint32_t)(kw * s_ld[d] + s_row[d]) * 4, 0, S + s_dst[d]);
    }
  };

  // ---- fragments of a k-step of 64: lane (row r32, half h) holds the 16 bytes of
  // block h, chunk 2 ks + h of its row, and that block's scale byte
  // (scales: a word per row holds the blocks of two k-steps; shifted by the
  // lane's half, byte 0 is the first's and byte 2 the second's)
  struct Frags {
    u32x4 a[AM], w[AN];
  };
  struct Scales {
    uint32_t a[AM], w[AN];
  };
  Frags f0, f1;
  Scales s0, s1;
  int c_off[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) c_off[ks] = ((2 * ks + h) ^ g8_swz128(r32, false)) * 16;
  const int a_rd = (wm * WM + r32) * 128, w_rd = Cfg::B_OFF + (wn * WN + r32) * 128;
  const int sa_rd = Cfg::SA_OFF + (wm * WM + r32) * 4, sw_rd = Cfg::SB_OFF + (wn * WN + r32) * 4;
  auto read_a = [&](Frags& f, int slot, int ks, int i) __attribute__((always_inline)) {
    const char* S = lds + slot * Cfg::STAGE;
    f.a[i] = *reinterpret_cast<const u32x4*>(S + a_rd + c_off[ks] + i * 4096);
  };
  auto read_w = [&](Frags& f, int slot, int ks, int j) __attribute__((always_inline)) {
    const char* S = lds + slot * Cfg::STAGE;
    f.w[j] = *reinterpret_cast<const u32x4*>(S + w_rd + c_off[ks] + j * 4096);
  };

  auto read_scales = [&](Scales& s, int slot, int pair) __attribute__((always_inline)) {
    const char* S = lds + slot * Cfg::STAGE;
#pragma unroll
    for (int i = 0; i < AM; ++i) s.a[i] = *reinterpret_cast<const uint32_t*>(S + sa_rd + pair * BM * 4 + i * 128);
#pragma unroll
    for (int j = 0; j < AN; ++j) s.w[j] = *reinterpret_cast<const uint32_t*>(S + sw_rd + pair * BN * 4 + j * 128);
  };
  auto shift = [&](Scales& s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AM; ++i) s.a[i] >>= 8 * h;
#pragma unroll
    for (int j = 0; j < AN; ++j) s.w[j] >>= 8 * h;
  };

  f32x16 acc[AM][AN];
#pragma unroll
  for (int i = 0; i < AM; ++i)
#pragma unroll
    for (int j = 0; j < AN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  auto wide = [](u32x4 v) __attribute__((always_inline)) {
    const i32x4 x = __builtin_bit_cast(i32x4, v);
    return __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  };
  // a k-step's MFMAs in groups of one weight fragment (weights as the MFMA's first
  // operand: a lane then holds runs of four consecutive output columns); f(j)
  // issues what goes beside group j
  // (BYTE: of the scale words)
  auto step = [&](const Frags& x, const Scales& s, auto byte, auto f) __attribute__((always_inline)) {
    constexpr int BYTE = decltype(byte)::value;
#pragma unroll
    for (int j = 0; j < AN; ++j) {
      f(j);
#pragma unroll
      for (int i = 0; i < AM; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(x.w[j]), wide(x.a[i]), acc[i][j], 4, 4,
                                                                    BYTE, (int)s.w[j], BYTE, (int)s.a[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // the reads of k-step ks, share j of AN
  auto read_share = [&](Frags& f, int slot, int ks, int j) __attribute__((always_inline)) {
    if (j < AN) read_w(f, slot, ks, j);
#pragma unroll
    for (int i = 0; i < AM; ++i)
      if (i * AN / AM == j) read_a(f, slot, ks, i);
  };

  // ---- prologue: the ring filled, stage 0 landed
  // (of the last slot's stage the first HL loads)
  constexpr int HL = (Cfg::DMA + 1) / 2;
#pragma unroll
  for (int t = 0; t < NST; ++t)
#pragma unroll
    for (int l = 0; l < (t < NST - 1 ? Cfg::DMA : HL); ++l) load(t, t, l);
  wait_vmcnt<(NST - 2) * Cfg::DMA + HL>();
  barrier_nofence();
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 2>;
  read_scales(s0, 0, 0);
#pragma unroll
  for (int j = 0; j < AN; ++j) read_share(f0, 0, 0, j);

  // Stage t: each k-step's MFMAs while the next one's fragments arrive; before the
  // last, with every read of the stage done and stage t + 1 landed, the barrier,
  // after which the loads of stage t + NST go into this slot.  Past the last
  // stage the loads repeat it.
  int slot = 0;
  constexpr int LPJ = (HL + AN - 1) / AN;  // load instructions per group
  int prev = NST - 1;                      // the slot of stage t - 1
  for (int t = 0; t < depth / 256; ++t) {
    shift(s0);
    step(f0, s0, Even{}, [&](int j) __attribute__((always_inline)) {
      read_share(f1, slot, 1, j);
#pragma unroll
      for (int l = HL; l < Cfg::DMA; ++l)
        if ((l - HL) / LPJ == j) load(t + NST - 1, prev, l);
    });
    step(f1, s0, Odd{}, [&](int j) __attribute__((always_inline)) {
      if (j == 0) read_scales(s1, slot, 1);
      read_share(f0, slot, 2, j);
    });
    shift(s1);
    step(f0, s1, Even{}, [&](int j) __attribute__((always_inline)) {
      if (j == 0)
#pragma unroll
        for (int i = 0; i < AN; ++i) read_share(f1, slot, 3, i);
    });
    wait_lgkmcnt0();
    wait_vmcnt<(NST - 2) * Cfg::DMA>();
    barrier_nofence();
    prev = slot;
    slot = slot + 1 < NST ? slot + 1 : 0;
    step(f1, s1, Odd{}, [&](int j) __attribute__((always_inline)) {
      if (j == 0) read_scales(s0, slot, 0);
      read_share(f0, slot, 0, j);
#pragma unroll
      for (int l = 0; l < HL; ++l)
        if (l / LPJ == j) load(t + NST, prev, l);
    });
  }
  if (half) {
    shift(s0);
    step(f0, s0, Even{}, [&](int j) __attribute__((always_inline)) { read_share(f1, slot, 1, j); });
    step(f1, s0, Odd{}, [](int) {});
  }
  wait_vmcnt<0>();
  if constexpr (EPI == kEpiPartial) {
    float* P = p.partial + (int64_t)kz * p.M * p.N;
#pragma unroll
    for (int i = 0; i < AM; ++i) {
      const int gm = m0 + wm * WM + i * 32 + r32;
#pragma unroll
      for (int j = 0; j < AN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int gn = n0 + wn * WN + j * 32 + 8 * g + 4 * h;  // N % 8 == 0: four columns inside or outside
          if (gm < p.M && gn < p.N)
            *reinterpret_cast<f32x4*>(P + (int64_t)gm * p.N + gn) =
                f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
    }
    return;
  } else {
    // ---- epilogue: the tile through LDS, 16-byte chunks XORed by the row so that
    // both the writes and the 16-byte reads spread over the banks
    __syncthreads();
    constexpr int CH = WN / 8, RPI = 64 / CH;
    char* E = lds + wave * Cfg::EPI_WAVE;  // a wave reads back only what it wrote itself
    const int ch = lane % CH, rsub = lane / CH;
    const int gn = n0 + wn * WN + ch * 8;
    // the values of columns 8 g + 4 h on of fragment column j, rows of block i, to put(i, j, g, value)
    auto branch = [&](int i0, int i1, auto sig_tag, auto rtb_tag, auto put) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < AN; ++j) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = n0 + wn * WN + j * 32 + 8 * g + 4 * h;
          f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
          if (p.bias && c < p.N)
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[e] = p.bias[c + e];
#pragma unroll
          for (int i = 0; i < AM; ++i) {
            if (i < i0 || i >= i1) continue;
            const f32x4 y = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            put(i, j, g, fp4_branch4<EPI, decltype(sig_tag)::value, decltype(rtb_tag)::value>(p, y, bias, c));
          }
        }
      }
    };
    if constexpr (RESID) {
      constexpr int PASS = Cfg::R_PASS, ROWB = Cfg::R_ROWB, C4 = WN / 4, ITS = PASS * 32 / RPI;
      float g8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) g8[e] = gn < p.N ? p.gate[gn + e] : 0.0f;
#pragma unroll
      for (int i0 = 0; i0 < AM; i0 += PASS) {
        auto put = [&](int i, int j, int g, f32x4 y) __attribute__((always_inline)) {
          const int row = (i - i0) * 32 + r32;
          *reinterpret_cast<f32x4*>(E + row * ROWB + (((8 * j + 2 * g + h) ^ row) & (C4 - 1)) * 16) = y;
        };
        if (p.round_then_bias) branch(i0, i0 + PASS, std::false_type{}, std::true_type{}, put);
        else branch(i0, i0 + PASS, std::false_type{}, std::false_type{}, put);
        bf16x8 res[ITS];
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          int gm = m0 + wm * WM + i0 * 32 + it * RPI + rsub;
          gm = gm < p.M ? gm : p.M - 1;
          res[it] = *reinterpret_cast<const bf16x8*>(p.R + (int64_t)gm * p.ldr + (gn < p.N ? gn : 0));
        }
        wait_lgkmcnt0();
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          const int row = it * RPI + rsub, gm = m0 + wm * WM + i0 * 32 + row;
          const f32x4 a = *reinterpret_cast<const f32x4*>(E + row * ROWB + (((2 * ch) ^ row) & (C4 - 1)) * 16);
          const f32x4 b = *reinterpret_cast<const f32x4*>(E + row * ROWB + (((2 * ch + 1) ^ row) & (C4 - 1)) * 16);
          bf16x8 v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = fp4_residual<EPI>(e < 4 ? a[e & 3] : b[e & 3], res[it][e], g8[e]);
          if (gm < p.M && gn < p.N) *reinterpret_cast<bf16x8*>(p.C + (int64_t)gm * p.ldc + gn) = v;
        }
        __builtin_amdgcn_wave_barrier();
      }
    } else {
      constexpr int ITS = WM / RPI;
      auto swz = [](int row) { return CH == 16 ? row & 15 : (CH == 8 ? (row >> 1) & 7 : (row >> 2) & 3); };
      auto put = [&](int i, int j, int g, f32x4 y) __attribute__((always_inline)) {
        const int row = i * 32 + r32;
        *reinterpret_cast<bf16x4*>(E + row * Cfg::EPI_ROWB + ((4 * j + g) ^ swz(row)) * 16 + h * 8) = fp4_bf16(y);
      };
      const bool sig = EPI == LTX_GEMM_EPI_BIAS && n0 + wn * WN + WN > p.sig_from;
      if (p.round_then_bias) {
        if (sig) branch(0, AM, std::true_type{}, std::true_type{}, put);
        else branch(0, AM, std::false_type{}, std::true_type{}, put);
      } else {
        if (sig) branch(0, AM, std::true_type{}, std::false_type{}, put);
        else branch(0, AM, std::false_type{}, std::false_type{}, put);
      }
      wait_lgkmcnt0();
      __builtin_amdgcn_wave_barrier();
      if (gn >= p.N) return;
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const int row = it * RPI + rsub, gm = m0 + wm * WM + row;
        if (gm >= p.M) break;
        *reinterpret_cast<bf16x8*>(p.C + (int64_t)gm * p.ldc + gn) =
            *reinterpret_cast<const bf16x8*>(E + row * Cfg::EPI_ROWB + (ch ^ swz(row)) * 16);
      }
    }
  }
}

using M4Large = M4Tile<256, 256, 2, 4, 2>;
using M4Tall = M4Tile<256, 128, 4, 2, 3>;
using M4Mid = M4Tile<128, 128, 2, 4, 4>;
using M4Small = M4Tile<64, 128, 2, 4, 4>;

struct Mx4Plan {
  int bm, bn, splits;
  int k_split;  // k of one range, a multiple of 256
};

// Modelled time (us): a round of one workgroup per CU costs `fixed` (first loads
// and epilogue) and per 256 k `idle` to `full`, as it fills the CUs (they share the
// L2s and the chip's power); a split's second launch and its partials.  Model
// against measured: 1296 x 4096 -> 4096 in tiles of 256 x 256, 256 x 128, 128 x 128,
// 64 x 128 29 / 21 / 24 / 28 against 26 / 20 / 25 / 28, 3456 x 4096 -> 4096 34 / 41 /
// 48 / 66 against 35 / 43 / 55 / 70, 1296 x 4096 -> 12320 60 / 58 / 59 / 71 against 58 /
// 55 / 60 / 72, 68 x 8192 -> 2048 64 x 128 in 4 splits 11 / 11, 256 x 4096 -> 8192 64 x
// 128 11 / 11, 6144 x 1024 -> 16384 256 x 256 77 / 79.
static double mx4_time(int64_t M, int64_t N, int bm, int bn, int splits, double per) {
  const double wgs = (double)(((M + bm - 1) / bm) * ((N + bn - 1) / bn) * splits);
  double fixed = 2.2, idle = 0.37, full = 0.40;
  if (bm == 256 && bn == 256) fixed = 5.5, idle = 1.15, full = 1.75;
  else if (bm == 256) fixed = 4.3, idle = 0.80, full = 0.94;
  else if (bm == 128) fixed = 2.6, idle = 0.49, full = 0.57;
  const double rounds = (double)(int64_t)(wgs / 256), rest = wgs / 256 - rounds;
  double t = 2.2 + rounds * (fixed + per * full);
  if (rest > 0) t += fixed + per * (idle + (full - idle) * rest);
  if (splits > 1) t += 2.5 + (double)(M * N) * splits * 8 / 4e6;
  return t;
}

static Mx4Plan mx4_plan(int64_t M, int64_t N, int64_t K) {
  static const int tile[4][2] = {{256, 256}, {256, 128}, {128, 128}, {64, 128}};
  const int64_t units = (K + 255) / 256;
  Mx4Plan pl = {64, 128, 1, (int)(units * 256)};
  double best = 1e30;
  for (const auto& t : tile) {
    const int64_t tiles = ((M + t[0] - 1) / t[0]) * ((N + t[1] - 1) / t[1]);
    for (int want = 1; want <= 16; ++want) {
      // splits: at least two stages each, within one round of the CUs, 10 % faster
      if (want > 1 && (units / want < 2 || tiles * want > 256)) break;
      const int64_t per = (units + want - 1) / want;
      const int s = (int)((units + per - 1) / per);
      const double us = mx4_time(M, N, t[0], t[1], s, (double)per);
      if (us < best * (s > 1 ? 0.9 : 1.0)) {
        best = us;
        pl = {t[0], t[1], s, (int)(per * 256)};
      }
    }
  }
  return pl;
}

template <int EPI>
static void mx4_launch(const GemmArgs& p, const Mx4Plan& pl, hipStream_t s) {
  GemmArgs a = p;
  a.tiles_m = (p.M + pl.bm - 1) / pl.bm;
  a.tiles_n = (p.N + pl.bn - 1) / pl.bn;
  const int blocks = a.tiles_m * a.tiles_n * pl.splits;
  auto go = [&](auto t) {
    using T = decltype(t);
    gemm_mx4_kernel<T, EPI><<<blocks, T::THREADS, 0, s>>>(a, pl.k_split);
  };
  if (pl.bm == 256 && pl.bn == 256) go(M4Large{});
  else if (pl.bm == 256) go(M4Tall{});
  else if (pl.bm == 128) go(M4Mid{});
  else go(M4Small{});
}

}  // namespace ltx

using namespace ltx;

extern "C" int64_t ltx_gemm_mx4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return -1;
  if (M == 0 || N == 0 || K == 0 || M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2) return 0;
  const Mx4Plan pl = mx4_plan(M, N, K);
  return pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0;
}

extern "C" int ltx_gemm_mx4_bf16(const uint8_t* A, int64_t lda, const uint32_t* a_scale, int64_t ld_ascale,
                                 const uint8_t* Wq, int64_t ldw, const uint32_t* w_scale, int64_t ld_scale,
                                 const float* bias, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K,
                                 int epilogue, const void* residual, int64_t ldr, const float* gate,
                                 int64_t sigmoid_from, float* workspace, int64_t workspace_bytes, void* stream) {
  const int st = fp4_check(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, epilogue, residual, ldr, gate,
                           K / 2, 16);
  if (st != LTX_OK) return st;
  if (!a_scale || ld_ascale < M) return LTX_ERR_INVALID_ARG;
  if (K % 128) return LTX_ERR_UNSUPPORTED;
  if (((uintptr_t)a_scale & 15u) || ld_ascale % 4) return LTX_ERR_ALIGNMENT;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  // operand extents are 31-bit buffer record counts in the kernel
  const int64_t lim = (int64_t)1 << 31;
  if (M > lim / lda || N > lim / ldw || ld_ascale > lim / (K / 32) || ld_scale > lim / (K / 32) || M * lda >= lim ||
      N * ldw >= lim || ld_ascale * (K / 32) >= lim || ld_scale * (K / 32) >= lim)
    return LTX_ERR_UNSUPPORTED;
  const Mx4Plan pl = mx4_plan(M, N, K);
  const int64_t need = pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return LTX_ERR_INVALID_ARG;
  if (need > 0 && ((uintptr_t)workspace & 15u)) return LTX_ERR_ALIGNMENT;
  GemmArgs p = fp4_args(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, epilogue, residual, ldr, gate,
                        sigmoid_from);
  p.ascale = (const uint8_t*)a_scale;
  p.ld_ascale = ld_ascale;
  hipStream_t s = (hipStream_t)stream;
  const int epi = epilogue & 0xff;
  if (pl.splits > 1) {
    p.partial = workspace;
    mx4_launch<kEpiPartial>(p, pl, s);
    const int e = ltx_launch_status();
    return e != LTX_OK ? e : fp4_combine(p, epi, pl.splits, s);
  }
  fp4_epilogue(epi, [&](auto e) { mx4_launch<decltype(e)::value>(p, pl, s); });
  return ltx_launch_status();
}
