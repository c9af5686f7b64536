// Projection GEMMs of MXFP4 rows and MXFP4 weights on the scaled FP4 MFMA
// (v_mfma_scale_f32_16x16x128_f8f6f4):
//
//   C[m, n] = epilogue( sum_k a[m, k] w[n, k] + bias[n] ),
//   a = e2m1(A) 2^(XA), w = e2m1(W) 2^(XW), a scale per 32 k on both sides.
//
// Operand storage: gemm_fp4.h.
//
// A workgroup of 4 waves (2 x 2) computes a BM x BN tile.  A stage is 256 k:
// rows of 128 code bytes, one line each, and two scale words per row; stages
// reach LDS by direct loads into a ring of NST.  A stage has two k-steps of 128;
// lane (row r16, quarter q) of a fragment holds the 16 bytes of its row's block
// q, and its scale operand that block's byte.  The fragments of the next
// k-step are read while the MFMAs of the current one run, also across the
// one barrier per stage.
#include "gemm_fp4.h"

namespace ltx {

constexpr int kM4Threads = 256;

template <int BM_, int BN_>
struct M4Cfg {
  static constexpr int BM = BM_, BN = BN_, WM = BM / 2, WN = BN / 2, AM = WM / 16, AN = WN / 16;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128;
  // two scale words per row; at least one direct-load instruction (1 KiB)
  static constexpr int SA_BYTES = BM * 8 < 1024 ? 1024 : BM * 8, SB_BYTES = BN * 8 < 1024 ? 1024 : BN * 8;
  static constexpr int B_OFF = A_BYTES, SA_OFF = B_OFF + B_BYTES, SB_OFF = SA_OFF + SA_BYTES;
  static constexpr int STAGE = SB_OFF + SB_BYTES;
  static constexpr int NST = BM * BN >= 256 * 256 ? 2 : 3;
  // direct loads of a wave per stage: code rows, and a share of the scales'
  static constexpr int A_DMA = BM / 32, B_DMA = BN / 32;
  static constexpr int SA_DMA = SA_BYTES / 1024, SB_DMA = SB_BYTES / 1024;
  // scale instructions go to the waves in turn: S_DMA per wave, the same count
  // for each (a wave without one of its own repeats one)
  static constexpr int S_DMA = (SA_DMA + SB_DMA + 3) / 4;
  static constexpr int DMA = A_DMA + B_DMA + S_DMA;
  static constexpr int EPI_ROWB = WN * 2, EPI_WAVE = WM * EPI_ROWB;
  static constexpr int RING = NST * STAGE, EPI = 4 * EPI_WAVE;
  static constexpr int LDS_BYTES = RING > EPI ? RING : EPI;
  static_assert(LDS_BYTES <= 160 * 1024 && (NST - 1) * DMA < 60, "LDS, vmcnt range");
};

template <int BM_, int BN_, int EPI>
__global__ __launch_bounds__(kM4Threads, 1) void gemm_mx4_kernel(GemmArgs p, int k_split) {
  using Cfg = M4Cfg<BM_, BN_>;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, WM = Cfg::WM, WN = Cfg::WN, AM = Cfg::AM, AN = Cfg::AN;
  constexpr int NST = Cfg::NST, A_DMA = Cfg::A_DMA, B_DMA = Cfg::B_DMA;
  constexpr bool RESID = EPI == LTX_GEMM_EPI_RESIDUAL || EPI == LTX_GEMM_EPI_RESIDUAL_ROUND;
  __shared__ __attribute__((aligned(1024))) char lds[Cfg::LDS_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int r16 = lane & 15, q = lane >> 4;
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
  const int chunk = pair_chunk(lane);
  const int back = (chunk & 4) * 16;
  uint32_t a_src[A_DMA], b_src[B_DMA];
#pragma unroll
  for (int d = 0; d < A_DMA; ++d) {
    int gm = m0 + 8 * (4 * d + wave) + (lane >> 3);
    gm = gm < p.M ? gm : p.M - 1;
    a_src[d] = (uint32_t)((int64_t)gm * p.lda + k0 / 2) + chunk * 16;
  }
#pragma unroll
  for (int d = 0; d < B_DMA; ++d) {
    int gn = n0 + 8 * (4 * d + wave) + (lane >> 3);
    gn = gn < p.N ? gn : p.N - 1;
    b_src[d] = (uint32_t)((int64_t)gn * p.ldb + k0 / 2) + chunk * 16;
  }
  // Scales: 16 bytes (4 rows' words) per lane.  Piece i of an operand's stage
  // (BM or BN words for each of the two k-steps) is words 4 i .. 4 i + 3.  Rows
  // past the padded count and k-steps past the last re-read the last.
  const int words = p.K / 128;
  auto scale_src = [&](int piece, int rows, int row0, int64_t ld, int t) __attribute__((always_inline)) {
    int kw = k0 / 128 + 2 * t + (piece * 4) / rows;
    int row = row0 + (piece * 4) % rows;
    kw = kw < words ? kw : words - 1;
    row = row + 4 <= (int)ld ? row : (int)ld - 4;
    return (uint32_t)(((int64_t)kw * ld + row) * 4);
  };
  const int sa_records = (int)((int64_t)words * p.ld_ascale * 4), sb_records = (int)((int64_t)words * p.ld_scale * 4);
  auto load_stage = [&](int t, int slot) __attribute__((always_inline)) {
    t = t < T ? t : T - 1;
    char* S = lds + slot * Cfg::STAGE;
    const uint32_t bk = half && t == T - 1 ? back : 0;
#pragma unroll
    for (int d = 0; d < A_DMA; ++d)
      buffer_dma16(p.A, a_records, a_src[d] - bk, t * 128, S + (4 * d + wave) * 1024);
#pragma unroll
    for (int d = 0; d < B_DMA; ++d)
      buffer_dma16(p.B, b_records, b_src[d] - bk, t * 128, S + Cfg::B_OFF + (4 * d + wave) * 1024);
#pragma unroll
    for (int d = 0; d < Cfg::S_DMA; ++d) {
      int i = 4 * d + wave;  // scale instruction: the activations', then the weights'
      i = i < Cfg::SA_DMA + Cfg::SB_DMA ? i : i % (Cfg::SA_DMA + Cfg::SB_DMA);
      if (i < Cfg::SA_DMA)
        buffer_dma16(p.ascale, sa_records, scale_src(i * 64 + lane, BM, m0, p.ld_ascale, t), 0,
                     S + Cfg::SA_OFF + i * 1024);
      else
        buffer_dma16(p.bscale, sb_records, scale_src((i - Cfg::SA_DMA) * 64 + lane, BN, n0, p.ld_scale, t), 0,
                     S + Cfg::SB_OFF + (i - Cfg::SA_DMA) * 1024);
    }
  };

  // ---- fragments
  struct Frag {
    u32x4 a[AM], b[AN];
    uint32_t sa[AM], sb[AN];
  };
  int c_off[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) c_off[ks] = ((4 * ks + q) ^ swz_pair(r16)) * 16;
  const int a_rd = (wm * WM + r16) * 128, b_rd = Cfg::B_OFF + (wn * WN + r16) * 128;
  const int sa_rd = Cfg::SA_OFF + (wm * WM + r16) * 4 + q, sb_rd = Cfg::SB_OFF + (wn * WN + r16) * 4 + q;
  auto read_a = [&](Frag& f, int slot, int ks, int i) __attribute__((always_inline)) {
    const char* S = lds + slot * Cfg::STAGE;
    f.a[i] = *reinterpret_cast<const u32x4*>(S + a_rd + c_off[ks] + i * 2048);
    f.sa[i] = *reinterpret_cast<const uint8_t*>(S + sa_rd + ks * BM * 4 + i * 64);
  };
  auto read_b = [&](Frag& f, int slot, int ks, int j) __attribute__((always_inline)) {
    const char* S = lds + slot * Cfg::STAGE;
    f.b[j] = *reinterpret_cast<const u32x4*>(S + b_rd + c_off[ks] + j * 2048);
    f.sb[j] = *reinterpret_cast<const uint8_t*>(S + sb_rd + ks * BN * 4 + j * 64);
  };

  f32x4 acc[AM][AN];
#pragma unroll
  for (int i = 0; i < AM; ++i)
#pragma unroll
    for (int j = 0; j < AN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto wide = [](u32x4 v) __attribute__((always_inline)) {
    const i32x4 x = __builtin_bit_cast(i32x4, v);
    return __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  };
  // the MFMAs of weight fragment j (weights as the MFMA's first operand: a
  // lane then holds four consecutive output columns)
  auto multiply = [&](const Frag& f, int j) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AM; ++i)
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(f.b[j]), wide(f.a[i]), acc[i][j], 4, 4, 0,
                                                                   (int)f.sb[j], 0, (int)f.sa[i]);
  };
  // a k-step's MFMAs, the reads of the next one spread over them
  constexpr int RPJ = (AM + AN + AN - 1) / AN;  // reads per group
  auto step = [&](const Frag& f, Frag& nx, int slot, int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < AN; ++j) {
#pragma unroll
      for (int r = j * RPJ; r < (j + 1) * RPJ && r < AM + AN; ++r) {
        if (r < AN) read_b(nx, slot, ks, r < AN ? r : 0);
        else read_a(nx, slot, ks, r >= AN ? r - AN : 0);
      }
      multiply(f, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // ---- prologue: the ring filled, stage 0 landed
  static_for<0, NST>([&](auto ic) { load_stage(decltype(ic)::value, decltype(ic)::value); });
  wait_vmcnt<(NST - 1) * Cfg::DMA>();
  barrier_nofence();
  Frag f0, f1;
#pragma unroll
  for (int j = 0; j < AN; ++j) read_b(f0, 0, 0, j);
#pragma unroll
  for (int i = 0; i < AM; ++i) read_a(f0, 0, 0, i);

  // Stage t: k-step 0 while k-step 1's fragments arrive; then, with every read
  // of the stage done and stage t + 1 landed, the barrier, the loads of stage
  // t + NST into this slot, and k-step 1 while the next stage's first
  // fragments arrive.  Past the last stage the loads repeat it.
  int slot = 0;
  for (int t = 0; t < depth / 256; ++t) {
    step(f0, f1, slot, 1);
    wait_lgkmcnt0();
    wait_vmcnt<(NST - 2) * Cfg::DMA>();
    barrier_nofence();
    load_stage(t + NST, slot);
    slot = slot + 1 < NST ? slot + 1 : 0;
    step(f1, f0, slot, 0);
  }
  if (half)
#pragma unroll
    for (int j = 0; j < AN; ++j) multiply(f0, j);
  wait_vmcnt<0>();
  if constexpr (EPI == kEpiPartial) {
    float* P = p.partial + (int64_t)kz * p.M * p.N;
#pragma unroll
    for (int i = 0; i < AM; ++i) {
      const int gm = m0 + wm * WM + i * 16 + r16;
#pragma unroll
      for (int j = 0; j < AN; ++j) {
        const int gn = n0 + wn * WN + j * 16 + 4 * q;  // N % 8 == 0: four columns inside or outside
        if (gm < p.M && gn < p.N) *reinterpret_cast<f32x4*>(P + (int64_t)gm * p.N + gn) = acc[i][j];
      }
    }
    return;
  } else {
    // ---- epilogue: bf16 tile through LDS, 16-byte chunks XORed by the row so
    // that both the 8-byte writes and the 16-byte reads spread over the banks
    __syncthreads();
    constexpr int CH = WN / 8, RPI = 64 / CH, ITS = WM / RPI;
    auto swz = [](int row) { return CH == 16 ? row & 15 : (row >> 1) & 7; };
    char* E = lds + wave * Cfg::EPI_WAVE;
#pragma unroll
    for (int j = 0; j < AN; ++j) {
      const int gn = n0 + wn * WN + j * 16 + 4 * q;
      f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
      if (p.bias && gn < p.N)
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = p.bias[gn + e];
#pragma unroll
      for (int i = 0; i < AM; ++i) {
        const int row = i * 16 + r16;
        *reinterpret_cast<bf16x4*>(E + row * Cfg::EPI_ROWB + ((2 * j + (q >> 1)) ^ swz(row)) * 16 + (q & 1) * 8) =
            fp4_branch4<EPI>(p, acc[i][j], bias, gn);
      }
    }
    // a wave reads back only what it wrote itself
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
    const int ch = lane % CH, rsub = lane / CH;
    const int gn = n0 + wn * WN + ch * 8;
    if (gn >= p.N) return;
    float g8[8];
    if constexpr (RESID)
#pragma unroll
      for (int e = 0; e < 8; ++e) g8[e] = p.gate[gn + e];
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
      const int row = it * RPI + rsub, gm = m0 + wm * WM + row;
      if (gm >= p.M) break;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(E + row * Cfg::EPI_ROWB + (ch ^ swz(row)) * 16);
      if constexpr (RESID) {
        const bf16x8 r = *reinterpret_cast<const bf16x8*>(p.R + (int64_t)gm * p.ldr + gn);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fp4_residual<EPI>(v[e], r[e], g8[e]);
      }
      *reinterpret_cast<bf16x8*>(p.C + (int64_t)gm * p.ldc + gn) = v;
    }
  }
}

struct Mx4Plan {
  int bm, bn, splits, k_split;
};
static Mx4Plan mx4_plan(int64_t M, int64_t N, int64_t K) {
  Mx4Plan pl;
  const int64_t big = ((M + 255) / 256) * ((N + 255) / 256);
  pl.bm = big >= 160 ? 256 : (M <= 64 ? 64 : 128);
  pl.bn = big >= 160 ? 256 : 128;
  const int64_t tiles = ((M + pl.bm - 1) / pl.bm) * ((N + pl.bn - 1) / pl.bn);
  const int64_t units = (K + 255) / 256;
  int64_t s = 256 / tiles;
  if (s > units / 2) s = units / 2;
  if (s > 32) s = 32;
  if (s < 1) s = 1;
  const int64_t per = (units + s - 1) / s;
  pl.k_split = (int)(per * 256);
  pl.splits = (int)((units + per - 1) / per);
  return pl;
}

template <int EPI>
static void mx4_launch(const GemmArgs& p, const Mx4Plan& pl, hipStream_t s) {
  GemmArgs a = p;
  a.tiles_m = (p.M + pl.bm - 1) / pl.bm;
  a.tiles_n = (p.N + pl.bn - 1) / pl.bn;
  const int blocks = a.tiles_m * a.tiles_n * pl.splits;
  if (pl.bm == 256) gemm_mx4_kernel<256, 256, EPI><<<blocks, kM4Threads, 0, s>>>(a, pl.k_split);
  else if (pl.bm == 128) gemm_mx4_kernel<128, 128, EPI><<<blocks, kM4Threads, 0, s>>>(a, pl.k_split);
  else gemm_mx4_kernel<64, 128, EPI><<<blocks, kM4Threads, 0, s>>>(a, pl.k_split);
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
