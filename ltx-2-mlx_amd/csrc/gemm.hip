// Projection GEMMs of the DiT block on CDNA4 matrix cores.
//
//   C[m, n] = epilogue( sum_k A[m, k] * W[n, k] + bias[n] )
//
// A: bf16 activations (M, K) row-major.  W: the weight in its storage layout
// (N, K) row-major -- nn.Linear's layout -- in one of three formats:
//   bf16                          (reference: nn.Linear / mx.addmm,
//                                  attention.py:425-437, feed_forward.py:91-112)
//   int8 + fp32 per-row scale     (W8A16: w = bf16(fp32(q) * s))
//   MXFP8: E4M3 codes + E8M0 scale per 32 consecutive k
//                                 (loader/transformer_cache.py:1255-1267; the
//                                  reference dequantises to bf16 and runs a bf16
//                                  MMA, docs/PERFORMANCE_NOTES.md:1450-1470)
// Both operands are K-contiguous, which is what the MFMA fragments want.
//
// Kernel structure (one 256-thread workgroup = 4 waves in a 2x2 grid):
//   * block tile BM x BN (256x256 or 128x128), K step 64, two LDS stages plus
//     a third stage in flight, by one of two loaders:
//       - registers (default): the global loads of stage k+2 go to VGPRs while
//         stage k computes; during stage k each lane writes its registers of
//         stage k+1 to LDS and reloads them with stage k+2, one pair every
//         few MFMAs, so loads and LDS writes never idle the matrix pipe;
//       - LDS DMA (global_load_lds_dwordx4) straight into the freed buffer,
//         spread over the last k-step's MFMAs.
//     One barrier per K step.
//   * quantised weights travel to LDS as their 8-bit codes (half the bytes)
//     and are dequantised to bf16 as each lane reads its MFMA fragment, with
//     the exact format arithmetic, so the bf16 MFMA sees bit-exact weights.
//   * LDS rows are 128 bytes (64 bf16; 64 codes for 8-bit weights); 16-byte
//     chunks are XOR-swizzled ((row/2)%8, or (row/4)%4 for 64-byte rows) so
//     the fragment reads of consecutive rows spread over the banks.  The load
//     source address of each lane implements the swizzle.
//   * fragments of k-step kk+1 are read from LDS before the MFMAs of kk issue,
//     across the stage boundary too.
//   * v_mfma_f32_32x32x16_bf16 with the weight fragment as the MFMA "A"
//     operand: each lane then holds 4 consecutive output columns, so the
//     epilogue packs 4 bf16 per LDS write and streams the tile out through LDS
//     in coalesced 16-byte chunks, fusing bias, GELU-tanh, the 2*sigmoid head
//     gate or the gated residual add (fused_ops.py:345-348 semantics).  Bias
//     and gate columns come from LDS and residual rows are fetched before the
//     tile is staged, so the epilogue never waits on memory per element.
//   * blockIdx -> tile: consecutive tiles go to the same XCD (the hardware
//     round-robins workgroups over the 8 XCDs), grouped 4 tile-rows at a
//     time: the 32 concurrent tiles of an XCD form 4 x 8, the fewest distinct
//     activation and weight bytes per K step.
#include "gemm8.h"

namespace ltx {

// How stage tiles reach LDS: LDS DMA (global_load_lds), or global loads into
// registers one stage ahead that are written to LDS during the next stage.
enum Loader { LOAD_DMA = 0, LOAD_REG = 1 };

constexpr int kGemmThreads = 256;

template <int BM, int BN, int BK, int STAGES_, int BKIND, int EPI, int SWZ, int LOADER>
struct GemmCfg {
  static constexpr int WM = BM / 2, WN = BN / 2;    // wave tile (2 x 2 waves)
  static constexpr int TM = WM / 32, TN = WN / 32;  // 32x32 MFMA tiles per wave
  static constexpr bool B8 = BKIND != B_BF16;
  // 8-bit weights stay 8-bit in LDS with the DMA loader (dequantised per
  // fragment); the register loader dequantises them once, on the way to LDS.
  static constexpr bool B_RAW = B8 && LOADER == LOAD_DMA;
  static constexpr int KSTEPS = BK / 16;             // MFMA k-steps per stage
  static constexpr int A_ROWB = BK * 2;              // bytes per LDS row
  static constexpr int B_ROWB = B_RAW ? BK : BK * 2;
  static constexpr int B_GROWB = B8 ? BK : BK * 2;   // global bytes per weight row per stage
  static constexpr int A_BYTES = BM * A_ROWB, B_BYTES = BN * B_ROWB;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = STAGES_;
  // per-lane 16-byte loads per stage (each wave instruction moves 1 KiB)
  static constexpr int A_DMA = A_BYTES / 1024 / 4;
  static constexpr int B_DMA = BN * B_GROWB / 1024 / 4;
  static constexpr int L = A_DMA + B_DMA;
  static constexpr int EPI_ROWB = WN * 2 + 16;  // padded epilogue row
  static constexpr int EPI_WAVE = WM * EPI_ROWB;
  static constexpr int EPI_BYTES = 4 * EPI_WAVE;
  static constexpr int LDS_BYTES = (STAGES * STAGE > EPI_BYTES) ? STAGES * STAGE : EPI_BYTES;
  static_assert(BK == 32 || BK == 64, "K step");
  static_assert(!B8 || BK == 64, "8-bit weights use 64-byte rows");
  static_assert(!B_RAW || BKIND != B_MXFP8 || STAGES == 2, "MXFP8 scales ride one stage ahead");
  static_assert(LOADER == LOAD_DMA || STAGES == 2, "register staging is the third stage");
  static constexpr int COL_BYTES = 2 * BN * 4;  // epilogue bias + gate columns
  static_assert(LDS_BYTES + COL_BYTES <= 160 * 1024, "LDS");
  static_assert((STAGES - 1) * L < 64, "vmcnt range");
};

// 16-byte chunk XOR of an LDS row.  128-byte rows: SWZ 0 uses (row/2)%8
// (conflict-free per 16 lanes over 256 bytes of banks), SWZ 1 uses row%8.
// 64-byte rows: (row/4)%4.
template <int ROWB, int SWZ>
__device__ __forceinline__ int chunk_xor(int r) {
  if constexpr (ROWB == 128) return SWZ == 0 ? ((r >> 1) & 7) : (r & 7);
  else return (r >> 2) & 3;
}

template <int BM, int BN, int BK, int STAGES_, int BKIND, int EPI, int SWZ, int LOADER>
__global__ __launch_bounds__(kGemmThreads, 1) void gemm_kernel(GemmArgs p) {
  using Cfg = GemmCfg<BM, BN, BK, STAGES_, BKIND, EPI, SWZ, LOADER>;
  constexpr bool REG = LOADER == LOAD_REG;
  constexpr int WM = Cfg::WM, WN = Cfg::WN, TM = Cfg::TM, TN = Cfg::TN;
  constexpr bool B8 = Cfg::B8, B_RAW = Cfg::B_RAW;
  constexpr bool B_CONV = B8 && !B_RAW;  // 8-bit weights dequantised by the loader
  constexpr int STAGES = Cfg::STAGES, KSTEPS = Cfg::KSTEPS;
  constexpr int STAGE = Cfg::STAGE;
  constexpr int A_BYTES = Cfg::A_BYTES;
  constexpr int A_ROWB = Cfg::A_ROWB, B_ROWB = Cfg::B_ROWB;
  constexpr int A_DMA = Cfg::A_DMA, B_DMA = Cfg::B_DMA, L = Cfg::L;
  constexpr int EPI_ROWB = Cfg::EPI_ROWB, EPI_WAVE = Cfg::EPI_WAVE;
  __shared__ __attribute__((aligned(1024))) char lds[Cfg::LDS_BYTES + Cfg::COL_BYTES];
  constexpr bool RESID = EPI == LTX_GEMM_EPI_RESIDUAL || EPI == LTX_GEMM_EPI_RESIDUAL_ROUND;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wm = wave >> 1, wn = wave & 1;

  int tmi, tni;
  // split-K: block b works on split b / tiles of tile b % tiles, the split's
  // k range starting at kz * K
  constexpr bool PARTIAL = EPI == kEpiPartial;
  const int tiles = p.tiles_m * p.tiles_n;
  const int kz = PARTIAL ? (int)blockIdx.x / tiles : 0;
  tile_coords(PARTIAL ? (int)blockIdx.x % tiles : (int)blockIdx.x, PARTIAL ? tiles : (int)gridDim.x,
              p.tiles_m, p.tiles_n, tmi, tni);
  const int m0 = tmi * BM, n0 = tni * BN;
  const int KT = p.K / BK;
  const int64_t k0 = (int64_t)kz * p.K;

  // The epilogue's per-column vectors (bias; gate of the residual forms) are
  // loaded once here, one column per thread, and reach the epilogue through
  // LDS, so no column group waits on global memory there.
  float col_bias = 0.0f, col_gate = 0.0f;
  if (tid < BN && n0 + tid < p.N) {
    if (p.bias) col_bias = p.bias[n0 + tid];
    if (RESID) col_gate = p.gate[n0 + tid];
  }
  float* col_lds = reinterpret_cast<float*>(lds + Cfg::LDS_BYTES);

  // ---- DMA source addresses (k = 0).  Wave instruction i of a tile covers
  // its 1 KiB block 4*i + wave: rows (1024 / ROWB) * (4*i + wave) + lane / LPR
  // with LPR = ROWB / 16 lanes per row; lane slot lane % LPR holds logical
  // chunk slot ^ chunk_xor(row).  Rows past M / N re-read the last row.
  constexpr int A_LPR = A_ROWB / 16, B_LPR = B_ROWB / 16;
  const char* a_src[A_DMA];
#pragma unroll
  for (int i = 0; i < A_DMA; ++i) {
    const int r = (1024 / A_ROWB) * (4 * i + wave) + lane / A_LPR;
    int gm = m0 + r;
    gm = gm < p.M ? gm : p.M - 1;
    const int chunk = (lane % A_LPR) ^ chunk_xor<A_ROWB, SWZ>(r);
    a_src[i] = (const char*)(p.A + (int64_t)gm * p.lda + k0) + chunk * 16;
  }
  const char* b_src[B_DMA];
  int b_dst[B_CONV ? B_DMA : 1];            // loader dequant: LDS byte offset of the row
  int b_c16[B_CONV ? B_DMA : 1];            // ... and the 16-code chunk of it
  const uint8_t* b_scr[B_CONV ? B_DMA : 1];  // MXFP8 scale row
  float b_s8[B_CONV ? B_DMA : 1];           // int8 row scale
#pragma unroll
  for (int i = 0; i < B_DMA; ++i) {
    if constexpr (!B_CONV) {
      const int r = (1024 / B_ROWB) * (4 * i + wave) + lane / B_LPR;
      const int chunk = (lane % B_LPR) ^ chunk_xor<B_ROWB, SWZ>(r);
      int gn = n0 + r;
      gn = gn < p.N ? gn : p.N - 1;
      b_src[i] = (const char*)p.B + ((int64_t)gn * p.ldb + k0) * (B8 ? 1 : 2) + chunk * 16;
    } else {
      // 64-byte code rows, 16 per wave instruction: lane -> row +lane/4,
      // codes 16*(lane%4) .. +16 (no swizzle: it applies to the bf16 writes)
      const int r = 16 * (4 * i + wave) + (lane >> 2);
      int gn = n0 + r;
      gn = gn < p.N ? gn : p.N - 1;
      b_c16[i] = lane & 3;
      b_dst[i] = r * B_ROWB;
      b_src[i] = (const char*)p.B + (int64_t)gn * p.ldb + k0 + b_c16[i] * 16;
      if (BKIND == B_MXFP8) b_scr[i] = (const uint8_t*)p.bscale + (int64_t)gn * p.ld_scale + k0 / 32;
      if (BKIND == B_INT8) b_s8[i] = ((const float*)p.bscale)[gn];
    }
  }

  // Per-lane weight rows of the B fragments and their scales.
  const int frag_r = lane & 31;
  const int frag_c = lane >> 5;
  float s_i8[TN];
  const uint8_t* sc_row[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    int gn = n0 + wn * WN + j * 32 + frag_r;
    gn = gn < p.N ? gn : p.N - 1;
    if (B_RAW && BKIND == B_INT8) s_i8[j] = ((const float*)p.bscale)[gn];
    if (B_RAW && BKIND == B_MXFP8) sc_row[j] = (const uint8_t*)p.bscale + (int64_t)gn * p.ld_scale + k0 / 32;
  }
  // MXFP8 scales of one stage: 2 E8M0 bytes (k blocks 0/1 of the 64) per row.
  uint32_t sc_cur[TN], sc_next[TN];

  // DMA instruction d (0 <= d < L) of stage kt into buffer buf.  Every stage
  // issues all L instructions; stages past the last one re-read stage KT-1
  // into a buffer that is never read again, so the number of outstanding
  // instructions per stage is the same everywhere.
  auto dma_op = [&](int d, int kt, int buf) {
    char* As = lds + buf * STAGE;
    if (d < A_DMA) {
      dma16(a_src[d] + (int64_t)kt * (BK * 2), As + (4 * d + wave) * 1024);
    } else {
      const int i = d - A_DMA;
      dma16(b_src[i] + (int64_t)kt * (B8 ? BK : BK * 2), As + A_BYTES + (4 * i + wave) * 1024);
    }
  };
  // Register-staged loader: load d of stage kt into rg[d], and its LDS write.
  // 8-bit weight loads carry 16 codes (and, for MXFP8, the E8M0 scale of
  // their 32-block), written to LDS as 16 dequantised bf16 in two chunks.
  typedef __attribute__((address_space(1))) const u32x4* g16_t;
  typedef __attribute__((address_space(1))) const uint32_t* g4_t;
  u32x4 rg[REG ? L : 1];
  // MXFP8: the aligned 4-byte scale word holding this load's E8M0 byte, and
  // the byte's bit offset in it (ld_scale % 4 == 0)
  uint32_t rsc[(REG && BKIND == B_MXFP8) ? B_DMA : 1], rsh[(REG && BKIND == B_MXFP8) ? B_DMA : 1];
  auto gload = [&](int d, int kt) {
    if constexpr (REG) {
      if (d < A_DMA) {
        rg[d] = *(g16_t)(a_src[d] + (int64_t)kt * (BK * 2));
      } else {
        rg[d] = *(g16_t)(b_src[d - A_DMA] + (int64_t)kt * (B8 ? BK : BK * 2));
        if constexpr (BKIND == B_MXFP8) {
          const int byte = kt * (BK / 32) + (b_c16[d - A_DMA] >> 1);
          rsc[d - A_DMA] = *(g4_t)(b_scr[d - A_DMA] + (byte & ~3));
          rsh[d - A_DMA] = 8 * (byte & 3);
        }
      }
    }
  };
  // LDS write of load d, in NPART pieces (part = 0 .. NPART-1) issued in
  // consecutive MFMA slots: an 8-bit weight load is dequantised a quarter at
  // a time (its ~16 VALU instructions in one slot would idle the matrix pipe
  // for two MFMAs), the last piece writes the 16 bf16 to LDS.
  float b_sc[B_CONV ? B_DMA : 1];      // dequantisation scale of the load in flight
  uint32_t b_o[B_CONV ? B_DMA : 1][8];  // its bf16 pairs
  auto lwrite = [&](int d, int buf, int part, int nparts) {
    if constexpr (REG) {
      char* As = lds + buf * STAGE;
      if (!B_CONV || d < A_DMA) {
        if (part != nparts - 1) return;
        char* dst = d < A_DMA ? As + (4 * d + wave) * 1024 : As + A_BYTES + (4 * (d - A_DMA) + wave) * 1024;
        *reinterpret_cast<u32x4*>(dst + lane * 16) = rg[d];
      } else {
        const int i = d - A_DMA;
        if (part == 0 && (b_dst[i] / B_ROWB) & 1) {
          // odd rows convert their upper 8 codes first, so their first LDS
          // write fills the chunks the even row above leaves free
          const u32x4 v = rg[d];
          rg[d] = u32x4{v[2], v[3], v[0], v[1]};
        }
        const u32x4 w = rg[d];
        // pieces of a load in four slots: the odd-row swap (part 0), the scale
        // and the first code word (1), two words (2), the last word and the
        // LDS writes (3) -- at most ~8 VALU instructions under one MFMA
        const int dec_part = nparts == 4 ? 1 : 0;
        if (part == dec_part) {
          if constexpr (BKIND == B_MXFP8) {
            // The loaded word goes straight into the empty asm, which pins the
            // byte extraction and decode here: hoisted to the top of the loop
            // they made every iteration wait for the previous stage's loads.
            uint32_t e = rsc[i];
            asm volatile("" : "+v"(e));
            b_sc[i] = e8m0_to_f32((e >> rsh[i]) & 0xffu);
          } else {
            b_sc[i] = b_s8[i];
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int q_part = nparts == 4 ? (q == 0 ? 1 : (q == 3 ? 3 : 2)) : q * nparts / 4;
          if (q_part != part) continue;
          const float sc = b_sc[i];
          if constexpr (BKIND == B_MXFP8) {
            b_o[i][2 * q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[q], sc, false));
            b_o[i][2 * q + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[q], sc, true));
          } else {
            const float nb = -128.0f * sc;
            const uint32_t u = w[q] ^ 0x80808080u;
            bf16x2 p0, p1;
            p0[0] = (bf16)fmaf((float)(u & 0xffu), sc, nb);
            p0[1] = (bf16)fmaf((float)((u >> 8) & 0xffu), sc, nb);
            p1[0] = (bf16)fmaf((float)((u >> 16) & 0xffu), sc, nb);
            p1[1] = (bf16)fmaf((float)(u >> 24), sc, nb);
            b_o[i][2 * q] = __builtin_bit_cast(uint32_t, p0);
            b_o[i][2 * q + 1] = __builtin_bit_cast(uint32_t, p1);
          }
          // keep this piece in its slot (pure arithmetic would otherwise be
          // sunk to the LDS write)
          asm volatile("" : "+v"(b_o[i][2 * q]), "+v"(b_o[i][2 * q + 1]));
        }
        if (part == nparts - 1) {
          // rows 2m and 2m+1 share their chunk swizzle: the even row writes
          // its even chunks first, the odd row its odd chunks, so each write
          // instruction covers every chunk position of the two rows once
          const int r = b_dst[i] / B_ROWB, odd = r & 1;
          char* row = As + A_BYTES + b_dst[i];
          const int x = chunk_xor<B_ROWB, SWZ>(r);
          *reinterpret_cast<u32x4*>(row + ((2 * b_c16[i] + odd) ^ x) * 16) =
              u32x4{b_o[i][0], b_o[i][1], b_o[i][2], b_o[i][3]};
          *reinterpret_cast<u32x4*>(row + ((2 * b_c16[i] + 1 - odd) ^ x) * 16) =
              u32x4{b_o[i][4], b_o[i][5], b_o[i][6], b_o[i][7]};
        }
      }
    }
  };
  auto load_scales = [&](int kt) {
#pragma unroll
    for (int j = 0; j < TN; ++j) sc_next[j] = *reinterpret_cast<const uint16_t*>(sc_row[j] + kt * 2);
  };
  // Stage kt+1 landed while the (STAGES-2) younger stages stay in flight.
  auto wait_next_stage = [&]() {
    if constexpr (REG) return;  // the compiler tracks register loads itself
    else if constexpr (B_RAW && BKIND == B_MXFP8) wait_vmcnt<0>();  // scale loads share the counter
    else wait_vmcnt<(STAGES - 2) * L>();
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  int a_off[TM], b_off[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) a_off[i] = (wm * WM + i * 32 + frag_r) * A_ROWB;
#pragma unroll
  for (int j = 0; j < TN; ++j) b_off[j] = (wn * WN + j * 32 + frag_r) * B_ROWB;
  const int a_swz = chunk_xor<A_ROWB, SWZ>(frag_r);  // same for rows i*32+frag_r
  const int b_swz = chunk_xor<B_ROWB, SWZ>(frag_r);

  // Fragment reads of k-step kk of the stage in buffer `buf`.  8-bit weights
  // are read as their raw codes and dequantised only as their MFMAs issue
  // (conv), so no MFMA waits for a conversion that waits for LDS.
  using BFrag = std::conditional_t<B_RAW, u32x2, bf16x8>;
  auto read_frags = [&](int buf, int kk, bf16x8* fa, BFrag* fb) {
    const char* As = lds + buf * STAGE;
    const char* Bs = As + A_BYTES;
    const int ca = ((kk * 2 + frag_c) ^ a_swz) * 16;
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = *reinterpret_cast<const bf16x8*>(As + a_off[i] + ca);
    if constexpr (!B_RAW) {
      const int cbf = ((kk * 2 + frag_c) ^ b_swz) * 16;
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = *reinterpret_cast<const bf16x8*>(Bs + b_off[j] + cbf);
    } else {
      const int c8 = kk * 2 + frag_c;  // 8-byte chunk of the 64-byte row
      const int cb = ((c8 >> 1) ^ b_swz) * 16 + (c8 & 1) * 8;
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = *reinterpret_cast<const u32x2*>(Bs + b_off[j] + cb);
    }
  };
  // fragment f of k-step kk: A fragments 0..TM-1, then B fragments
  auto read_frag = [&](int buf, int kk, int f, bf16x8* fa, BFrag* fb) {
    const char* As = lds + buf * STAGE;
    const char* Bs = As + A_BYTES;
    if (f < TM) {
      const int ca = ((kk * 2 + frag_c) ^ a_swz) * 16;
      fa[f] = *reinterpret_cast<const bf16x8*>(As + a_off[f] + ca);
    } else if constexpr (!B_RAW) {
      const int cbf = ((kk * 2 + frag_c) ^ b_swz) * 16;
      fb[f - TM] = *reinterpret_cast<const bf16x8*>(Bs + b_off[f - TM] + cbf);
    } else {
      const int c8 = kk * 2 + frag_c;
      const int cb = ((c8 >> 1) ^ b_swz) * 16 + (c8 & 1) * 8;
      fb[f - TM] = *reinterpret_cast<const u32x2*>(Bs + b_off[f - TM] + cb);
    }
  };
  // B fragment j of k-step kk as bf16 (MXFP8 scales of the current stage in
  // sc_cur; int8 per-row scales in s_i8).
  auto conv = [&](const BFrag* fb, int j, int kk) -> bf16x8 {
    if constexpr (!B_RAW) {
      return fb[j];
    } else {
      const u32x2 raw = fb[j];
      uint32_t o[4];
      if constexpr (BKIND == B_INT8) {
        const float sc = s_i8[j], nb = -128.0f * sc;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const uint32_t u = raw[d] ^ 0x80808080u;
          bf16x2 p0, p1;
          p0[0] = (bf16)fmaf((float)(u & 0xffu), sc, nb);
          p0[1] = (bf16)fmaf((float)((u >> 8) & 0xffu), sc, nb);
          p1[0] = (bf16)fmaf((float)((u >> 16) & 0xffu), sc, nb);
          p1[1] = (bf16)fmaf((float)(u >> 24), sc, nb);
          o[2 * d] = __builtin_bit_cast(uint32_t, p0);
          o[2 * d + 1] = __builtin_bit_cast(uint32_t, p1);
        }
      } else {
        const float sc = e8m0_to_f32((sc_cur[j] >> (8 * (kk >> 1))) & 0xffu);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          o[2 * d] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d], sc, false));
          o[2 * d + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d], sc, true));
        }
      }
      return __builtin_bit_cast(bf16x8, u32x4{o[0], o[1], o[2], o[3]});
    }
  };
  // MFMAs of k-step kk, weight-fragment-major, with memory instructions spread
  // between them: op(m) issues what belongs after MFMA m.  Issuing loads or
  // LDS writes this way never idles the matrix pipe, and the dequantisation
  // of weight fragment j+1 runs under the MFMAs of fragment j.
  auto mfmas_with = [&](const bf16x8* fa, const BFrag* fb, int kk, auto&& op) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const bf16x8 b = conv(fb, j, kk);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b, fa[i], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);  // the MFMA issues first; op runs under it
        op(j * TM + i);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto mfmas = [&](const bf16x8* fa, const BFrag* fb, int kk) { mfmas_with(fa, fb, kk, [](int) {}); };
  // the L loads of stage kt_src, spread over the NM MFMAs of one k-step
  auto loads_at = [&](int kt_src, int buf) {
    return [&, kt_src, buf](int m) {
      constexpr int NM = TM * TN;
#pragma unroll
      for (int d = 0; d < L; ++d)
        if ((d * NM) / L == m) {
          dma_op(d, kt_src, buf);
        }
    };
  };

  // Software pipeline: all STAGES buffers are filled ahead; fragments of the
  // next k-step are read while the MFMAs of the current one run, including
  // across the stage boundary, whose barrier sits between the fragment reads
  // of the last k-step and its MFMAs.
  bf16x8 fa[2][TM];
  BFrag fb[2][TN];
  if constexpr (REG) {
#pragma unroll
    for (int d = 0; d < L; ++d) gload(d, 0);
#pragma unroll
    for (int d = 0; d < L; ++d) lwrite(d, 0, 0, 1);
#pragma unroll
    for (int d = 0; d < L; ++d) gload(d, KT > 1 ? 1 : 0);
  } else {
#pragma unroll
    for (int st = 0; st < STAGES; ++st)
#pragma unroll
      for (int d = 0; d < L; ++d) dma_op(d, st < KT ? st : KT - 1, st);
  }
  if (B_RAW && BKIND == B_MXFP8) {
    load_scales(0);
    wait_vmcnt<0>();
#pragma unroll
    for (int j = 0; j < TN; ++j) sc_cur[j] = sc_next[j];
    load_scales(KT > 1 ? 1 : 0);
  } else if constexpr (!REG) {
    wait_vmcnt<(STAGES - 1) * L>();
  }
  __syncthreads();
  read_frags(0, 0, fa[0], fb[0]);
  wait_lgkmcnt0();

  // k-steps 0..KSTEPS-2 of the stage in `buf`: read k-step kk+1, then MFMAs of
  // kk.  The fragments of kk were issued one MFMA block earlier; waiting for
  // them before issuing the next reads keeps at most one group (TM+TN <= 8
  // reads) in flight, which the 4-bit LDS counter can track exactly.
  // With the register loader, the fragment reads of k-step kk+1 go one after
  // each of the first TM+TN MFMAs of kk, and the LDS writes of the next stage
  // (into wbuf), each followed one MFMA later by the global load of the stage
  // after it into the same registers (kt_load), are spread evenly over these
  // k-steps' MFMAs: no burst of LDS traffic queues up behind the other waves'.
  auto leading_ksteps = [&](int buf, int wbuf, bool write, int kt_load) {
#pragma unroll
    for (int kk = 0; kk < KSTEPS - 1; ++kk) {
      wait_lgkmcnt0();
      if constexpr (REG) {
        constexpr int NM = TM * TN, SLOTS = (KSTEPS - 1) * NM;
        // slots of a dequantising (8-bit weight) load: up to 4, within its share
        constexpr int BPARTS = (SLOTS / L) < 4 ? (SLOTS / L) : 4;
        static_assert(!B_CONV || BPARTS >= 1, "slots per load");
        mfmas_with(fa[kk & 1], fb[kk & 1], kk, [&](int m) {
          if (m < TM + TN) read_frag(buf, kk + 1, m, fa[(kk + 1) & 1], fb[(kk + 1) & 1]);
#pragma unroll
          for (int d = 0; d < L; ++d) {
            const int np = (B_CONV && d >= A_DMA) ? BPARTS : 1;
            const int slot0 = (d * SLOTS) / L;
#pragma unroll
            for (int part = 0; part < np; ++part)
              if (slot0 + part == kk * NM + m && write) lwrite(d, wbuf, part, np);
            // the reload into the same registers goes one slot after the LDS
            // write that reads them (issued right behind it, it waits for the
            // write to take its data: 3 % of a bf16 GEMM)
            const int reload = slot0 + np < SLOTS ? slot0 + np : SLOTS - 1;
            if (reload == kk * NM + m && write) gload(d, kt_load);
          }
        });
      } else {
        read_frags(buf, kk + 1, fa[(kk + 1) & 1], fb[(kk + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
        mfmas(fa[kk & 1], fb[kk & 1], kk);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int LASTF = (KSTEPS - 1) & 1;  // fragment set of the last k-step
  int buf = 0;
  for (int kt = 0; kt < KT - 1; ++kt) {
    const int nbuf = buf + 1 == STAGES ? 0 : buf + 1;
    leading_ksteps(buf, nbuf, true, kt + 2 < KT ? kt + 2 : KT - 1);
    wait_next_stage();
    __syncthreads();  // stage kt+1 visible to all waves; stage kt's buffer free
    read_frags(nbuf, 0, fa[0], fb[0]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (REG) {
      mfmas(fa[LASTF], fb[LASTF], KSTEPS - 1);
    } else {  // DMA of stage kt+STAGES into the freed buffer
      const int kt_src = kt + STAGES < KT ? kt + STAGES : KT - 1;
      mfmas_with(fa[LASTF], fb[LASTF], KSTEPS - 1, loads_at(kt_src, buf));
    }
    if (B_RAW && BKIND == B_MXFP8) {  // the next stage's scales (the last k-step used this one's)
#pragma unroll
      for (int j = 0; j < TN; ++j) sc_cur[j] = sc_next[j];
      load_scales(kt + 2 < KT ? kt + 2 : KT - 1);
    }
    buf = nbuf;
  }
  leading_ksteps(buf, buf, false, 0);
  wait_lgkmcnt0();
  __builtin_amdgcn_sched_barrier(0);
  mfmas(fa[LASTF], fb[LASTF], KSTEPS - 1);
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (PARTIAL) {
    // acc[i][j] reg 4g+e holds C[m][n], m = i*32 + lane%32, n = j*32 + 8g +
    // 4*(lane/32) + e (wave-local): four consecutive columns per store
    float* P = p.partial + (int64_t)kz * p.M * p.ldc;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int gm = m0 + wm * WM + i * 32 + frag_r;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int gn = n0 + wn * WN + j * 32 + 8 * g + 4 * frag_c;
          if (gm < p.M && gn < p.N)
            *reinterpret_cast<f32x4*>(P + (int64_t)gm * p.ldc + gn) =
                f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
    }
    return;
  }
  wait_vmcnt<0>();  // the re-read stages land before the epilogue reuses LDS
  if (tid < BN) {
    col_lds[tid] = col_bias;
    col_lds[BN + tid] = col_gate;
  }
  __syncthreads();  // all waves done with the stage buffers; columns visible

  // ---- epilogue: registers -> bf16 tile in LDS (per wave), then coalesced
  // 16-byte row stores.  Phase-2 lane mapping: 16-byte chunk ch of rows
  // it * ROWS_PER_IT + rsub of the wave tile.
  constexpr int CHUNKS = WN / 8;  // 16-byte chunks per wave-tile row
  constexpr int ROWS_PER_IT = 64 / CHUNKS;
  constexpr int ITS = WM / ROWS_PER_IT;
  const int ch = lane % CHUNKS;
  const int rsub = lane / CHUNKS;
  const int gn2 = n0 + wn * WN + ch * 8;
  const bool col_ok = gn2 < p.N;  // N % 8 == 0: a chunk is all in or all out
  // Residual rows (rows past M re-read row M-1, columns past N read column
  // 0; neither is stored) are fetched once phase 1 has moved the
  // accumulators to LDS: fetched any earlier, next to the 256 live
  // accumulators, part of the tile spills to scratch (measured 6-15 % of the
  // residual GEMMs' time).  Their latency overlaps the barrier after phase 1.
  // The residual may alias C: every residual element of this tile is read
  // before any of its outputs is written.
  bf16x8 res[RESID ? ITS : 1];
  auto fetch_res = [&]() {
    if constexpr (RESID) {
      const int gnc = col_ok ? gn2 : 0;
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        int gm = m0 + wm * WM + it * ROWS_PER_IT + rsub;
        gm = gm < p.M ? gm : p.M - 1;
        res[it] = *reinterpret_cast<const bf16x8*>(p.R + (int64_t)gm * p.ldr + gnc);
      }
    }
  };

  // phase 1: acc[i][j] reg 4g+e holds C[m][n] with m = i*32 + lane%32 and
  // n = j*32 + 8g + 4*(lane/32) + e (wave-local coordinates).  Whether any
  // column of this wave tile takes the head-gate sigmoid is wave-uniform, so
  // the common case runs without it.
  char* E = lds + wave * EPI_WAVE;
  // sig_tag / rtb_tag: compile-time forms of two block-uniform conditions
  // (gate columns in this wave tile; bias added to the rounded product), so
  // the per-element code has no branches
  auto phase1 = [&](auto sig_tag, auto rtb_tag) {
    constexpr bool SIG = decltype(sig_tag)::value;
    constexpr bool RTB = decltype(rtb_tag)::value;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int nl = j * 32 + 8 * g + 4 * frag_c;
        const int gn = n0 + wn * WN + nl;
        const f32x4 bias4 = *reinterpret_cast<const f32x4*>(col_lds + wn * WN + nl);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = acc[i][j][4 * g + e];
            y[e] = (RTB ? round_bf(a) : a) + bias4[e];
            if (EPI == LTX_GEMM_EPI_GELU) y[e] = gelu_tanh(round_bf(y[e]));
            if (EPI == LTX_GEMM_EPI_SIGMOID2) y[e] = sigmoid2_bf(round_bf(y[e]));
            if (SIG && gn + e >= p.sig_from) y[e] = sigmoid2_bf(round_bf(y[e]));
          }
          bf16x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (bf16)y[e];
          *reinterpret_cast<bf16x4*>(E + (i * 32 + frag_r) * EPI_ROWB + nl * 2) = v;
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
  fetch_res();
  __syncthreads();

  // phase 2: coalesced 16-byte stores (+ gated residual)
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
    bf16x8 v = *reinterpret_cast<const bf16x8*>(E + ml * EPI_ROWB + ch * 16);
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
    if (gm < p.M && col_ok) *reinterpret_cast<bf16x8*>(p.C + (int64_t)gm * p.ldc + gn2) = v;
  }
}

template <int BM, int BN, int BK, int STAGES, int BKIND, int EPI, int SWZ = 0, int LOADER = LOAD_DMA>
static void launch_tile(GemmArgs p, hipStream_t s) {
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  gemm_kernel<BM, BN, BK, STAGES, BKIND, EPI, SWZ, LOADER><<<p.tiles_m * p.tiles_n, kGemmThreads, 0, s>>>(p);
}

// ---- the mid-size kernel (gemm_kg.hip): which products, tile height, splits --
// Operand extents within its 31-bit buffer record counts, whole units of 128 k
// per split, and for MXFP8 whole groups of four units (16 E8M0 bytes) per
// split in 4-byte aligned pieces.
static bool kg_ok(int bkind, int64_t M, int64_t N, int64_t Ks, int64_t lda, int64_t ldb, int64_t ld_scale) {
  const int64_t lim = (int64_t)1 << 31;
  return bkind != B_MX && Ks > 0 && Ks % (bkind == B_MXFP8 ? 512 : 128) == 0 && M * lda * 2 < lim &&
         N * ldb * (bkind == B_BF16 ? 2 : 1) < lim && (bkind != B_MXFP8 || N * ld_scale < lim);
}

// Modelled time (us) of a product on the mid-size kernel.  A round of one
// workgroup per CU costs `unit` us per 128 k (measured at K = 4096-8192,
// tiles of 64 / 128 / 192 rows, weights from HBM), and however many rounds,
// the L2s deliver about 13 TB/s of tile operands to the CUs (every shape with
// all CUs busy measured 11-15 TB/s); 4 us of launch, first loads and
// epilogue; split-K adds its second launch and one write and read of the fp32
// partials.  Model against measured (MXFP8): 1296 x 4096 -> 4096 192 rows 40 /
// 43, 128 rows 53 / 59, 64 rows 57 / 61; 1296 x 16384 -> 4096 148 / 150,
// 201 / 193, 220 / 197; 204 x 8192 -> 2048 64 rows, 1 / 2 / 4 splits
// 39 / 27 / 20 against 32 / 24 / 19.
static double kg_time(int bkind, int64_t M, int64_t N, int64_t K, int bm, int64_t splits) {
  static const double unit_us[3][3] = {{0.78, 1.08, 1.30}, {0.87, 1.00, 1.25}, {0.55, 0.77, 1.08}};
  const int64_t wgs = ((M + bm - 1) / bm) * ((N + 127) / 128) * splits;
  const double units = (double)(K / 128) / (double)splits;
  const double rounds = (double)((wgs + 255) / 256);
  const double bytes = (double)wgs * units * 128.0 * (bkind == B_BF16 ? 2.0 * (bm + 128) : 2.0 * bm + 128.0);
  double t = rounds * units * unit_us[bkind][bm / 64 - 1];
  if (bytes / 13e6 > t) t = bytes / 13e6;
  t += 4.0;
  if (splits > 1) t += 3.5 + (double)(M * N * splits) * 8.0 / 3.5e6;
  return t;
}

// The same for 128x128 tiles of gemm_kernel, at most one workgroup per CU (0.6
// us per 64 k in every format: bf16 77 x 188160 -> 2048 in 4 splits 450 us).
static double tile128_time(int64_t M, int64_t N, int64_t K, int64_t splits) {
  const double t = (double)(K / 64) / (double)splits * 0.6 + 4.0;
  return splits > 1 ? t + 3.5 + (double)(M * N * splits) * 8.0 / 3.5e6 : t;
}

// The tile height that the model finds fastest for a split count.
static int kg_rows(int bkind, int64_t M, int64_t N, int64_t K, int64_t splits, double* us) {
  int best = 64;
  double t = kg_time(bkind, M, N, K, 64, splits);
  for (int bm = 128; bm <= 192; bm += 64) {
    const double u = kg_time(bkind, M, N, K, bm, splits);
    if (u < t) {
      t = u;
      best = bm;
    }
  }
  if (us) *us = t;
  return best;
}

// Whether an automatic launch takes the mid-size kernel: below 160 tiles of
// 256x256 (from there the 256-row tiles fill the chip; 3456 x 4096 -> 4096 90
// against 121 us), except where the 8-wave kernel's single round of 100-159
// tiles models faster (2.1 us per 128 k measured; int8 2.4).  Measured, this
// kernel against that one, K = 4096: 1728 x 4096 bf16 78 / 76, MXFP8 61 / 73;
// 2048 x 4096 86 / 76, 67 / 77; 2304 x 4096 81 / 75, 81 / 75; 384 x 16384
// 55 / 71, 51 / 76; 512 x 16384 93 / 77, 74 / 76; 700 x 12320 90 / 79, 86 / 77;
// 2816 x 2080 45 / 69, 46 / 72; 3456 x 2080 70 / 69, 62 / 72 (the A2V query
// projection, for which the block asks for the 8-wave kernel: CU time).
// Shallow products of more than one round of 64-row tiles keep the older
// kernels: with one to three units the loop is over before the ring has filled,
// and two 128x128 workgroups per CU hide one's first loads behind the other's
// epilogue (1296 x 128 -> 2048 bf16 7.3 / 6.6, 700 x 256 -> 4096 8.1 / 7.5, int8
// 700 x 128 -> 4096 7.7 / 6.8, 1296 x 384 -> 2048 10.1 / 9.7; one round, 700 x
// 128 -> 2048 bf16 5.8 / 6.1).
static bool kg_auto(int bkind, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ld_scale) {
  const int64_t big = ((M + 255) / 256) * ((N + 255) / 256);
  if (big >= 160 || !kg_ok(bkind, M, N, K, lda, ldb, ld_scale)) return false;
  if (K <= (bkind == B_INT8 ? 384 : 256) && ((M + 63) / 64) * ((N + 127) / 128) > 256) return false;
  if (big < 100) return true;
  double us;
  kg_rows(bkind, M, N, K, 1, &us);
  return us < 4.0 + (K / 128) * (bkind == B_INT8 ? 2.4 : 2.1);
}

// Tile shapes (all K step 64): 256x256 and 128x128 with the register-staged
// loader (1 and 2; 128x128 runs two workgroups per CU), 256x256 with the
// LDS-DMA loader (3), 256x128 register-staged (4), and the 8-wave kernel with
// 256x256 (5) or 128x256 tiles (6).
template <int BKIND, int EPI>
static int launch_epi_w(const GemmArgs& p, int tile, hipStream_t s) {
  const bool auto_tile = tile == 0;
  if (auto_tile && kg_auto(BKIND, p.M, p.N, p.K, p.lda, p.ldb, p.ld_scale)) {
    return kg_launch(BKIND, p, EPI, kg_rows(BKIND, p.M, p.N, p.K, 1, nullptr), 1, s) ? LTX_OK : LTX_ERR_UNSUPPORTED;
  }
  if (tile == 0) {
    // What the mid-size kernel does not take: large tiles when they still give
    // most CUs a tile, 128x128 otherwise.  The 8-wave kernel from 100 tiles of
    // 256x256, every format: there it measured faster than the 4-wave kernel on
    // every block shape (int8 4096^2 109 vs 134 us, FF up 428 vs 472, FF down
    // 405 vs 435; bf16 4096^2 91 vs 105, FF up 350 vs 420, FF down 339 vs 404,
    // 1024 x 4096 -> 12320 87 vs 101).  (Two forms that are faster alone on the
    // A2V query projection, 3456 x 4096 -> 2080, 126 tiles, stay explicit, as the
    // step follows the CU time of its launches: 256x128 tiles, 14 % faster, the
    // step 0.25 ms slower; 128-row tiles, 79 -> 61 us with 48 % more CU time, the
    // step 1.0-1.6 ms slower.  The block asks for the 256-row tiles there.)
    const int64_t big = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256);
    const bool g8 = g8_ok<BKIND>(p);
    tile = big >= 160 ? (g8 ? 5 : 1) : (big >= 100 && g8 ? 5 : 2);
    // row sums of squares come from the mid-size and 8-wave kernels' epilogues
    if (p.rowss && tile != 5) tile = 5;
  }
  if (p.rowss && tile != 5 && tile != 6) return LTX_ERR_UNSUPPORTED;
  if (tile == 5 || tile == 6) {
    if (!g8_ok<BKIND>(p)) return LTX_ERR_UNSUPPORTED;
    const int r0 = (tile == 5 && auto_tile) ? g8_split_rows(p.M, p.N) : p.M;
    if (tile == 6) {
      launch_g8<BKIND, EPI, 128>(p, s);
    } else if (r0 < p.M) {
      GemmArgs top = p;
      top.M = r0;
      launch_g8<BKIND, EPI>(top, s);
      launch_g8<BKIND, EPI, 128>(rows_from(p, r0), s);
    } else {
      launch_g8<BKIND, EPI>(p, s);
    }
    return LTX_OK;
  }
  if (tile == 1)
    launch_tile<256, 256, 64, 2, BKIND, EPI, 0, LOAD_REG>(p, s);
  else if (tile == 2)
    launch_tile<128, 128, 64, 2, BKIND, EPI, 0, LOAD_REG>(p, s);
  else if (tile == 4)
    launch_tile<256, 128, 64, 2, BKIND, EPI, 0, LOAD_REG>(p, s);
  else
    launch_tile<256, 256, 64, 2, BKIND, EPI, 0, LOAD_DMA>(p, s);
  return LTX_OK;
}

template <int BKIND, int EPI>
static int launch_epi(const GemmArgs& p, int tile, hipStream_t s) {
  if constexpr (BKIND == B_MX) {
    // quantised activations: the 8-wave kernel only
    if (tile != 0 && tile != 5) return LTX_ERR_UNSUPPORTED;
    if (!g8_ok<BKIND>(p)) return LTX_ERR_UNSUPPORTED;
    launch_g8<BKIND, EPI>(p, s);
    return LTX_OK;
  } else {
    return launch_epi_w<BKIND, EPI>(p, tile, s);
  }
}

template <int BKIND>
static int launch_kind(const GemmArgs& p, int epilogue, hipStream_t s) {
  const int epi = epilogue & 0xff;
  const int tile = (epilogue >> 8) & 0xf;
  if (tile > 6) return LTX_ERR_INVALID_ARG;
  GemmArgs q = p;
  q.round_then_bias = (epilogue & LTX_GEMM_ROUND_THEN_BIAS) != 0;
  int st;
  switch (epi) {
    case LTX_GEMM_EPI_BIAS: st = launch_epi<BKIND, LTX_GEMM_EPI_BIAS>(q, tile, s); break;
    case LTX_GEMM_EPI_GELU: st = launch_epi<BKIND, LTX_GEMM_EPI_GELU>(q, tile, s); break;
    case LTX_GEMM_EPI_RESIDUAL: st = launch_epi<BKIND, LTX_GEMM_EPI_RESIDUAL>(q, tile, s); break;
    case LTX_GEMM_EPI_RESIDUAL_ROUND: st = launch_epi<BKIND, LTX_GEMM_EPI_RESIDUAL_ROUND>(q, tile, s); break;
    case LTX_GEMM_EPI_SIGMOID2: st = launch_epi<BKIND, LTX_GEMM_EPI_SIGMOID2>(q, tile, s); break;
    case kEpiGeluMx:
      if constexpr (BKIND == B_MX) {
        st = launch_epi<BKIND, kEpiGeluMx>(q, tile, s);
        break;
      } else {
        return LTX_ERR_INVALID_ARG;
      }
    default: return LTX_ERR_INVALID_ARG;
  }
  if (st != LTX_OK) return st;
  return ltx_launch_status();
}

// ---- split-K ---------------------------------------------------------------
// Few-row products (the 68-token audio stream, the 256-token text contexts)
// give too few output tiles to fill 256 CUs, and each tile's K loop is a
// serial latency chain.  Split-K runs `splits` K ranges as separate blocks
// writing fp32 partial tiles; this kernel sums them in a fixed order (so the
// result is deterministic) and applies the same epilogue as the single-pass
// kernel's phases 1 and 2, eight columns per thread.
template <int EPI>
__global__ __launch_bounds__(256) void splitk_epilogue_kernel(GemmArgs p, int splits) {
  constexpr bool RESID = EPI == LTX_GEMM_EPI_RESIDUAL || EPI == LTX_GEMM_EPI_RESIDUAL_ROUND;
  const int nvec = p.N / 8;
  const int64_t total = (int64_t)p.M * nvec;
  const int64_t plane = (int64_t)p.M * p.N;
  const bool rtb = p.round_then_bias != 0;
  for (int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; idx < total;
       idx += (int64_t)gridDim.x * blockDim.x) {
    const int m = (int)(idx / nvec);
    const int n = (int)(idx % nvec) * 8;
    float a[8];
    {
      const float* P = p.partial + (int64_t)m * p.N + n;
      const f32x4 x0 = *reinterpret_cast<const f32x4*>(P);
      const f32x4 x1 = *reinterpret_cast<const f32x4*>(P + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = x0[e];
        a[4 + e] = x1[e];
      }
      for (int z = 1; z < splits; ++z) {
        const f32x4 y0 = *reinterpret_cast<const f32x4*>(P + z * plane);
        const f32x4 y1 = *reinterpret_cast<const f32x4*>(P + z * plane + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] += y0[e];
          a[4 + e] += y1[e];
        }
      }
    }
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float b = p.bias ? p.bias[n + e] : 0.0f;
      float y = (rtb ? round_bf(a[e]) : a[e]) + b;
      if (EPI == LTX_GEMM_EPI_GELU) y = gelu_tanh(round_bf(y));
      if (EPI == LTX_GEMM_EPI_SIGMOID2) y = sigmoid2_bf(round_bf(y));
      if (EPI == LTX_GEMM_EPI_BIAS && n + e >= p.sig_from) y = sigmoid2_bf(round_bf(y));
      v[e] = (bf16)y;
    }
    if constexpr (RESID) {
      const bf16x8 r = *reinterpret_cast<const bf16x8*>(p.R + (int64_t)m * p.ldr + n);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = (float)v[e], g = p.gate[n + e];
        const float o = EPI == LTX_GEMM_EPI_RESIDUAL ? fmaf(g, y, (float)r[e]) : round_bf(y * g) + (float)r[e];
        v[e] = (bf16)o;
      }
    }
    *reinterpret_cast<bf16x8*>(p.C + (int64_t)m * p.ldc + n) = v;
  }
}

template <int BKIND>
static int launch_splitk(const GemmArgs& p0, int epilogue, int splits, float* workspace, hipStream_t s) {
  const int epi = epilogue & 0xff;
  const int tile = (epilogue >> 8) & 0xf;
  // the mid-size kernel, or (explicitly, and for what it does not take)
  // 128x128 register-staged tiles
  if (tile != 0 && tile != 2) return LTX_ERR_UNSUPPORTED;
  GemmArgs p = p0;
  p.round_then_bias = (epilogue & LTX_GEMM_ROUND_THEN_BIAS) != 0;
  // pass 1: partial products, per-split depth K / splits, row stride N
  GemmArgs q = p;
  q.K = p.K / splits;
  q.partial = workspace;
  q.ldc = p.N;
  q.tiles_m = (p.M + 127) / 128;
  q.tiles_n = (p.N + 127) / 128;
  if (tile == 0 && kg_ok(BKIND, q.M, q.N, q.K, q.lda, q.ldb, q.ld_scale)) {
    if (!kg_launch(BKIND, q, kEpiPartial, kg_rows(BKIND, p.M, p.N, p.K, splits, nullptr), splits, s))
      return LTX_ERR_UNSUPPORTED;
  } else {
    gemm_kernel<128, 128, 64, 2, BKIND, kEpiPartial, 0, LOAD_REG>
        <<<q.tiles_m * q.tiles_n * splits, kGemmThreads, 0, s>>>(q);
  }
  // pass 2: sum + epilogue
  p.partial = workspace;
  const int64_t vecs = (int64_t)p.M * (p.N / 8);
  int blocks = (int)((vecs + 255) / 256);
  if (blocks > 4096) blocks = 4096;
  switch (epi) {
    case LTX_GEMM_EPI_BIAS: splitk_epilogue_kernel<LTX_GEMM_EPI_BIAS><<<blocks, 256, 0, s>>>(p, splits); break;
    case LTX_GEMM_EPI_GELU: splitk_epilogue_kernel<LTX_GEMM_EPI_GELU><<<blocks, 256, 0, s>>>(p, splits); break;
    case LTX_GEMM_EPI_RESIDUAL:
      splitk_epilogue_kernel<LTX_GEMM_EPI_RESIDUAL><<<blocks, 256, 0, s>>>(p, splits);
      break;
    case LTX_GEMM_EPI_RESIDUAL_ROUND:
      splitk_epilogue_kernel<LTX_GEMM_EPI_RESIDUAL_ROUND><<<blocks, 256, 0, s>>>(p, splits);
      break;
    case LTX_GEMM_EPI_SIGMOID2:
      splitk_epilogue_kernel<LTX_GEMM_EPI_SIGMOID2><<<blocks, 256, 0, s>>>(p, splits);
      break;
    default: return LTX_ERR_INVALID_ARG;
  }
  return ltx_launch_status();
}

}  // namespace ltx

using namespace ltx;

static inline bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

static int gemm_check(const void* A, int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc,
                      int64_t M, int64_t N, int64_t K, int epilogue, const void* R, int64_t ldr,
                      const float* gate, int b_elem_bytes) {
  if (!A || !B || !C || M < 0 || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2) return LTX_ERR_UNSUPPORTED;
  const int epi = epilogue & 0xff;
  if (epilogue & ~(0xfff | LTX_GEMM_ROUND_THEN_BIAS)) return LTX_ERR_INVALID_ARG;
  if ((epi == LTX_GEMM_EPI_RESIDUAL || epi == LTX_GEMM_EPI_RESIDUAL_ROUND) && (!R || !gate || ldr < N))
    return LTX_ERR_INVALID_ARG;
  if (K % 64 != 0 || N % 8 != 0) return LTX_ERR_UNSUPPORTED;
  if (lda < K || ldb < K || ldc < N) return LTX_ERR_INVALID_ARG;
  if (!al16(A) || !al16(B) || !al16(C) || lda % 8 || ldc % 8 || (ldb * b_elem_bytes) % 16 ||
      (R && (!al16(R) || ldr % 8)))
    return LTX_ERR_ALIGNMENT;
  return LTX_OK;
}

static GemmArgs make_args(const void* A, int64_t lda, const void* B, int64_t ldb, const void* bscale,
                          int64_t ld_scale, const float* bias, void* C, int64_t ldc, int64_t M,
                          int64_t N, int64_t K, const void* R, int64_t ldr, const float* gate,
                          int64_t sigmoid_from) {
  GemmArgs p;
  p.A = (const bf16*)A;
  p.lda = lda;
  p.B = B;
  p.ldb = ldb;
  p.bscale = bscale;
  p.ld_scale = ld_scale;
  p.bias = bias;
  p.C = (bf16*)C;
  p.ldc = ldc;
  p.R = (const bf16*)R;
  p.ldr = ldr;
  p.gate = gate;
  p.sig_from = (int)(sigmoid_from < N ? (sigmoid_from < 0 ? 0 : sigmoid_from) : N);
  p.round_then_bias = 0;
  p.partial = nullptr;
  p.ascale = nullptr;
  p.ld_ascale = 0;
  p.cscale = nullptr;
  p.ld_cscale = 0;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.tiles_m = p.tiles_n = 0;
  return p;
}

extern "C" int ltx_gemm_bf16(const void* A, int64_t lda, const void* W, int64_t ldw,
                             const float* bias, void* C, int64_t ldc, int64_t M, int64_t N,
                             int64_t K, int epilogue, const void* residual, int64_t ldr,
                             const float* gate, int64_t sigmoid_from, void* stream) {
  int st = gemm_check(A, lda, W, ldw, C, ldc, M, N, K, epilogue, residual, ldr, gate, 2);
  if (st != LTX_OK) return st;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  GemmArgs p = make_args(A, lda, W, ldw, nullptr, 0, bias, C, ldc, M, N, K, residual, ldr, gate,
                         sigmoid_from);
  return launch_kind<B_BF16>(p, epilogue, (hipStream_t)stream);
}

extern "C" int ltx_gemm_w8a16_bf16(const void* A, int64_t lda, const int8_t* Wq, int64_t ldw,
                                   const float* w_scale, const float* bias, void* C, int64_t ldc,
                                   int64_t M, int64_t N, int64_t K, int epilogue,
                                   const void* residual, int64_t ldr, const float* gate,
                                   int64_t sigmoid_from, void* stream) {
  int st = gemm_check(A, lda, Wq, ldw, C, ldc, M, N, K, epilogue, residual, ldr, gate, 1);
  if (st != LTX_OK) return st;
  if (!w_scale) return LTX_ERR_INVALID_ARG;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  GemmArgs p = make_args(A, lda, Wq, ldw, w_scale, 0, bias, C, ldc, M, N, K, residual, ldr, gate,
                         sigmoid_from);
  return launch_kind<B_INT8>(p, epilogue, (hipStream_t)stream);
}

extern "C" int ltx_gemm_mxfp8_bf16(const void* A, int64_t lda, const uint8_t* Wq, int64_t ldw,
                                   const uint8_t* w_scale, int64_t ld_scale, const float* bias,
                                   void* C, int64_t ldc, int64_t M, int64_t N, int64_t K,
                                   int epilogue, const void* residual, int64_t ldr,
                                   const float* gate, int64_t sigmoid_from, void* stream) {
  int st = gemm_check(A, lda, Wq, ldw, C, ldc, M, N, K, epilogue, residual, ldr, gate, 1);
  if (st != LTX_OK) return st;
  if (!w_scale || ld_scale < K / 32) return LTX_ERR_INVALID_ARG;
  if (ld_scale % 4 || ((uintptr_t)w_scale & 3u)) return LTX_ERR_ALIGNMENT;  // scale words
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  GemmArgs p = make_args(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, residual, ldr,
                         gate, sigmoid_from);
  return launch_kind<B_MXFP8>(p, epilogue, (hipStream_t)stream);
}

// The bias-epilogue product of one of the three weight formats (wformat 0:
// bf16 as ltx_gemm_bf16, 1: int8 as ltx_gemm_w8a16_bf16, 2: MXFP8 as
// ltx_gemm_mxfp8_bf16) with the per-row sums of squares of its bf16 outputs in
// columns [0, ss_cols): rowss[m * ld_rowss + j] = sum of C[m, n]^2 over
// n in [64 j, 64 j + 64).  On the mid-size or the 8-wave kernel, whose epilogues
// compute them; C is bit-identical to the plain entry point's on that kernel.
extern "C" int ltx_gemm_rowss_bf16(int wformat, const void* A, int64_t lda, const void* W, int64_t ldw,
                                   const void* w_scale, int64_t ld_scale, const float* bias, void* C,
                                   int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue,
                                   int64_t sigmoid_from, float* rowss, int64_t ld_rowss, int64_t ss_cols,
                                   void* stream) {
  if (wformat < 0 || wformat > 2) return LTX_ERR_INVALID_ARG;
  if ((epilogue & 0xff) != LTX_GEMM_EPI_BIAS) return LTX_ERR_INVALID_ARG;
  const int tile = (epilogue >> 8) & 0xf;
  if (tile != 0 && tile != 5 && tile != 6) return LTX_ERR_UNSUPPORTED;
  int st = gemm_check(A, lda, W, ldw, C, ldc, M, N, K, epilogue, nullptr, 0, nullptr, wformat == 0 ? 2 : 1);
  if (st != LTX_OK) return st;
  if (!rowss || ss_cols <= 0 || ss_cols % 64 || ss_cols > N || ss_cols > sigmoid_from || ld_rowss < ss_cols / 64)
    return LTX_ERR_INVALID_ARG;
  if (((uintptr_t)rowss & 3u) != 0) return LTX_ERR_ALIGNMENT;
  if (M > 0 && ld_rowss > (INT64_MAX / M)) return LTX_ERR_UNSUPPORTED;
  if (wformat == 1 && !w_scale) return LTX_ERR_INVALID_ARG;
  if (wformat == 2) {
    if (!w_scale || ld_scale < K / 32) return LTX_ERR_INVALID_ARG;
    if (ld_scale % 4 || ((uintptr_t)w_scale & 3u)) return LTX_ERR_ALIGNMENT;
  }
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  GemmArgs p = make_args(A, lda, W, ldw, wformat == 0 ? nullptr : w_scale, wformat == 2 ? ld_scale : 0, bias, C,
                         ldc, M, N, K, nullptr, 0, nullptr, sigmoid_from);
  p.rowss = rowss;
  p.ld_rowss = ld_rowss;
  p.ss_cols = (int)ss_cols;
  if (wformat == 0) return launch_kind<B_BF16>(p, epilogue, (hipStream_t)stream);
  if (wformat == 1) return launch_kind<B_INT8>(p, epilogue, (hipStream_t)stream);
  return launch_kind<B_MXFP8>(p, epilogue, (hipStream_t)stream);
}

// ---- split-K entry points ------------------------------------------------------
// MXFP8 activations x MXFP8 weights on the scaled fp8 MFMA (opt-in; no
// counterpart in the reference, whose MXFP8 path dequantises the weights and
// multiplies bf16 activations).  A: E4M3 codes (M, K) with row stride lda
// bytes and E8M0 scales (M, K/32) with row stride ld_ascale, as written by
// ltx_quantize_mxfp8_bf16 on the activation rows; W, w_scale as
// ltx_gemm_mxfp8_bf16.  Same epilogues and quantised-linear rounding flag.
extern "C" int ltx_gemm_mx_bf16(const uint8_t* A, int64_t lda, const uint8_t* a_scale, int64_t ld_ascale,
                                const uint8_t* Wq, int64_t ldw, const uint8_t* w_scale, int64_t ld_scale,
                                const float* bias, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K,
                                int epilogue, const void* residual, int64_t ldr, const float* gate,
                                int64_t sigmoid_from, void* stream) {
  if (!A || !a_scale || !Wq || !w_scale || !C || M < 0 || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2) return LTX_ERR_UNSUPPORTED;
  const int epi = epilogue & 0xff;
  if (epilogue & ~(0xfff | LTX_GEMM_ROUND_THEN_BIAS)) return LTX_ERR_INVALID_ARG;
  if (epi > LTX_GEMM_EPI_SIGMOID2) return LTX_ERR_INVALID_ARG;
  if ((epi == LTX_GEMM_EPI_RESIDUAL || epi == LTX_GEMM_EPI_RESIDUAL_ROUND) && (!residual || !gate || ldr < N))
    return LTX_ERR_INVALID_ARG;
  if (lda < K || ldw < K || ldc < N || ld_ascale < K / 32 || ld_scale < K / 32) return LTX_ERR_INVALID_ARG;
  if (K % 512 != 0 || N % 8 != 0) return LTX_ERR_UNSUPPORTED;
  if (!al16(A) || !al16(Wq) || !al16(C) || !al16(a_scale) || !al16(w_scale) || lda % 16 || ldw % 16 ||
      ldc % 8 || ld_ascale % 16 || ld_scale % 16 || (residual && (!al16(residual) || ldr % 8)))
    return LTX_ERR_ALIGNMENT;
  if (M == 0 || N == 0) return LTX_OK;
  GemmArgs p = make_args(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, residual, ldr, gate,
                         sigmoid_from);
  p.ascale = a_scale;
  p.ld_ascale = ld_ascale;
  return launch_kind<B_MX>(p, epilogue, (hipStream_t)stream);
}

// The MX path's feed-forward up-projection: GELU epilogue whose bf16 result
// is written as MXFP8 rows -- codes (M, N) with row stride ldcq bytes, E8M0
// scales (M, N/32) -- the quantised input of the down-projection, bit for bit
// what ltx_quantize_mxfp8_bf16 makes of the bf16 GELU output.
extern "C" int ltx_gemm_mx_gelu_mxfp8(const uint8_t* A, int64_t lda, const uint8_t* a_scale, int64_t ld_ascale,
                                      const uint8_t* Wq, int64_t ldw, const uint8_t* w_scale, int64_t ld_scale,
                                      const float* bias, uint8_t* Cq, int64_t ldcq, uint8_t* c_scale,
                                      int64_t ld_cscale, int64_t M, int64_t N, int64_t K, int flags,
                                      void* stream) {
  if (!A || !a_scale || !Wq || !w_scale || !Cq || !c_scale || M < 0 || N < 0 || K < 0)
    return LTX_ERR_INVALID_ARG;
  if (M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2) return LTX_ERR_UNSUPPORTED;
  if (flags & ~LTX_GEMM_ROUND_THEN_BIAS) return LTX_ERR_INVALID_ARG;
  if (lda < K || ldw < K || ldcq < N || ld_ascale < K / 32 || ld_scale < K / 32 || ld_cscale < N / 32)
    return LTX_ERR_INVALID_ARG;
  if (K % 512 != 0 || N % 32 != 0) return LTX_ERR_UNSUPPORTED;
  if (!al16(A) || !al16(Wq) || !al16(Cq) || !al16(a_scale) || !al16(w_scale) || lda % 16 || ldw % 16 ||
      ldcq % 8 || ld_ascale % 16 || ld_scale % 16)
    return LTX_ERR_ALIGNMENT;
  if (M == 0 || N == 0) return LTX_OK;
  GemmArgs p = make_args(A, lda, Wq, ldw, w_scale, ld_scale, bias, Cq, ldcq, M, N, K, nullptr, 0, nullptr, N);
  p.ascale = a_scale;
  p.ld_ascale = ld_ascale;
  p.cscale = c_scale;
  p.ld_cscale = ld_cscale;
  return launch_kind<B_MX>(p, kEpiGeluMx | flags, (hipStream_t)stream);
}

// Split-K factor that the library would choose for a product (wformat 0:
// bf16, 1: int8, 2: MXFP8): the count that models fastest, of those that leave
// whole units of K per split (at least 256 k: bf16 8 x 1024 -> 2048 9.9 us in 8
// splits of one unit, 7.3 in one pass) and fit one round of the 256 CUs.  All
// divisors count, not the powers of two alone: bf16 77 x 188160 -> 2048 161 us
// in 14 splits, 567 in 2 (a quarter of that depth is no whole number of units);
// int8 68 x 8448 -> 248 34 us in 2, 16 in 11.  A split must
// model 15 % faster than the single pass (it adds a launch and a workspace)
// and 10 % faster than a smaller count: over 213 measured products of 26-1024
// rows the choice is on average 1.1 % from the fastest count (15 % at every
// step: 1.8 %, 384 x 16384 -> 4096 bf16 2 splits 88 us for 4 splits 69).
// Depths that the mid-size kernel does not take (K / splits no multiple of its
// unit) split on 128x128 tiles, few rows only, up to 80 workgroups: MXFP8 68 x
// 3840 -> 4096 27 us in 2 splits against 40 in one pass, 68 x 1280 -> 2048 12.4
// in 5 against 16.5.
extern "C" int ltx_gemm_auto_splits(int64_t M, int64_t N, int64_t K, int wformat) {
  if (M <= 0 || N <= 0 || K <= 0 || wformat < 0 || wformat > 2 || M > INT32_MAX / 2 || N > INT32_MAX / 2 ||
      K > INT32_MAX / 2)
    return 1;
  if (((M + 255) / 256) * ((N + 255) / 256) >= 100) return 1;
  const int64_t ld_scale = wformat == B_MXFP8 ? K / 32 : 0;
  const int64_t tiles128 = ((M + 127) / 128) * ((N + 127) / 128), unit128 = wformat == B_MXFP8 ? 128 : 64;
  double single = tile128_time(M, N, K, 1);
  if (kg_ok(wformat, M, N, K, K, K, ld_scale)) kg_rows(wformat, M, N, K, 1, &single);
  double best = single;
  int splits = 1;
  for (int s = 2; s <= 16; ++s) {
    if (K % s || K / s < 256) continue;
    double us;
    if (kg_ok(wformat, M, N, K / s, K, K, ld_scale)) {
      const int bm = kg_rows(wformat, M, N, K, s, &us);
      if (((M + bm - 1) / bm) * ((N + 127) / 128) * s > 256) continue;
    } else if (M <= 256 && K / s % unit128 == 0 && tiles128 * s <= 80) {
      us = tile128_time(M, N, K, s);
    } else {
      continue;
    }
    if (us < 0.85 * single && us < 0.9 * best) {
      best = us;
      splits = s;
    }
  }
  return splits;
}

// Tile height (64, 128, 192) of an automatic launch of `splits` K ranges on the
// mid-size kernel, 0 where it takes another kernel; dense operands.
extern "C" int ltx_gemm_auto_rows(int64_t M, int64_t N, int64_t K, int wformat, int splits) {
  if (M <= 0 || N <= 0 || K <= 0 || wformat < 0 || wformat > 2 || M > INT32_MAX / 2 || N > INT32_MAX / 2 ||
      K > INT32_MAX / 2 || splits < 1 || splits > 64 || K % splits)
    return 0;
  const int64_t ld_scale = wformat == B_MXFP8 ? K / 32 : 0;
  const bool kg = splits == 1 ? kg_auto(wformat, M, N, K, K, K, ld_scale)
                              : kg_ok(wformat, M, N, K / splits, K, K, ld_scale);
  return kg ? kg_rows(wformat, M, N, K, splits, nullptr) : 0;
}

extern "C" int64_t ltx_gemm_splitk_workspace_bytes(int64_t M, int64_t N, int64_t splits) {
  if (M < 0 || N < 0 || splits < 1) return -1;
  return splits * M * N * 4;
}

static int splitk_check(int64_t M, int64_t N, int64_t K, int splits, const float* workspace,
                        int64_t workspace_bytes) {
  if (splits < 1 || splits > 64) return LTX_ERR_INVALID_ARG;
  if (K % (64 * (int64_t)splits)) return LTX_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < ltx_gemm_splitk_workspace_bytes(M, N, splits)) return LTX_ERR_INVALID_ARG;
  if (!al16(workspace)) return LTX_ERR_ALIGNMENT;
  return LTX_OK;
}

extern "C" int ltx_gemm_splitk_bf16(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias,
                                    void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue,
                                    const void* residual, int64_t ldr, const float* gate, int64_t sigmoid_from,
                                    int splits, float* workspace, int64_t workspace_bytes, void* stream) {
  int st = gemm_check(A, lda, W, ldw, C, ldc, M, N, K, epilogue, residual, ldr, gate, 2);
  if (st != LTX_OK) return st;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  if ((st = splitk_check(M, N, K, splits, workspace, workspace_bytes)) != LTX_OK) return st;
  GemmArgs p = make_args(A, lda, W, ldw, nullptr, 0, bias, C, ldc, M, N, K, residual, ldr, gate, sigmoid_from);
  return launch_splitk<B_BF16>(p, epilogue, splits, workspace, (hipStream_t)stream);
}

extern "C" int ltx_gemm_splitk_w8a16_bf16(const void* A, int64_t lda, const int8_t* Wq, int64_t ldw,
                                          const float* w_scale, const float* bias, void* C, int64_t ldc,
                                          int64_t M, int64_t N, int64_t K, int epilogue, const void* residual,
                                          int64_t ldr, const float* gate, int64_t sigmoid_from, int splits,
                                          float* workspace, int64_t workspace_bytes, void* stream) {
  int st = gemm_check(A, lda, Wq, ldw, C, ldc, M, N, K, epilogue, residual, ldr, gate, 1);
  if (st != LTX_OK) return st;
  if (!w_scale) return LTX_ERR_INVALID_ARG;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  if ((st = splitk_check(M, N, K, splits, workspace, workspace_bytes)) != LTX_OK) return st;
  GemmArgs p = make_args(A, lda, Wq, ldw, w_scale, 0, bias, C, ldc, M, N, K, residual, ldr, gate, sigmoid_from);
  return launch_splitk<B_INT8>(p, epilogue, splits, workspace, (hipStream_t)stream);
}

extern "C" int ltx_gemm_splitk_mxfp8_bf16(const void* A, int64_t lda, const uint8_t* Wq, int64_t ldw,
                                          const uint8_t* w_scale, int64_t ld_scale, const float* bias, void* C,
                                          int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue,
                                          const void* residual, int64_t ldr, const float* gate,
                                          int64_t sigmoid_from, int splits, float* workspace,
                                          int64_t workspace_bytes, void* stream) {
  int st = gemm_check(A, lda, Wq, ldw, C, ldc, M, N, K, epilogue, residual, ldr, gate, 1);
  if (st != LTX_OK) return st;
  if (!w_scale || ld_scale < K / 32) return LTX_ERR_INVALID_ARG;
  if (ld_scale % 4 || ((uintptr_t)w_scale & 3u)) return LTX_ERR_ALIGNMENT;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  if ((st = splitk_check(M, N, K, splits, workspace, workspace_bytes)) != LTX_OK) return st;
  if (K % (128 * (int64_t)splits)) return LTX_ERR_UNSUPPORTED;  // each split's scale words stay 4-byte aligned
  GemmArgs p = make_args(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, residual, ldr, gate,
                         sigmoid_from);
  return launch_splitk<B_MXFP8>(p, epilogue, splits, workspace, (hipStream_t)stream);
}
