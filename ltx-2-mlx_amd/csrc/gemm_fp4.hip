// Projection GEMMs with MXFP4 weights and bf16 activations:
//
//   C[m, n] = epilogue( sum_k A[m, k] * e2m1(W[n, k]) 2^(X[n, k / 32]) + bias[n] )
//
// Operand storage: gemm_fp4.h.  The weights are decoded to bf16 (exact) in
// registers and multiplied on v_mfma_f32_16x16x32_bf16, fp32 accumulation.
#include "gemm8.h"
#include "gemm_fp4.h"

namespace ltx {

// ---- few-row tiles ---------------------------------------------------------
// A workgroup computes MB * 16 rows x 128 columns over one K range; its 8
// waves take 16 columns each.  A lane (column r16, quarter q) loads the 16
// code bytes of its k block of 32 straight from memory: one block, one scale,
// four MFMA k-steps; the quarter's k run 32 q + 8 j in k-step j, for both
// operands.  The activation rows go through LDS, KC of k at a time, where all
// waves read them.  Takes every size that the products allow: what the other
// kernels do not (few rows of a depth that ends inside a scale word, operands of
// 2 GiB).  Bound by its own serial phases (256 x 4096 -> 8192 55 us, the mid-size
// kernel 21).
constexpr int kFrThreads = 512, kFrBN = 128;

template <int MB>
struct FrCfg {
  static constexpr int BM = MB * 16;
  static constexpr int KC = 512;
  // LDS row: KC bf16 and 32 bytes, so that the 16 rows x 16 bytes that a
  // fragment read's lane octets fetch together start in 16-byte pieces two
  // apart; rows 8-15 use the pieces between (their chunks XOR 1)
  static constexpr int ROWB = KC * 2 + 32;
  static constexpr int LDS_BYTES = BM * ROWB;
};

template <int MB, int EPI>
__global__ __launch_bounds__(kFrThreads) void fp4_rows_kernel(GemmArgs p, int k_split) {
  using Cfg = FrCfg<MB>;
  constexpr int KC = Cfg::KC, KB = KC / 128, ROWB = Cfg::ROWB, BM = Cfg::BM;
  __shared__ __attribute__((aligned(16))) char lds[Cfg::LDS_BYTES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r16 = lane & 15, q = lane >> 4;
  const int tiles = p.tiles_m * p.tiles_n;
  const int kz = (int)blockIdx.x / tiles, tile = (int)blockIdx.x % tiles;
  const int m0 = tile % p.tiles_m * BM, n0 = tile / p.tiles_m * kFrBN + wave * 16;
  const int k_begin = kz * k_split, k_end = k_begin + k_split < p.K ? k_begin + k_split : p.K;

  // columns past N re-read the last one, rows past M the last row
  int gn = n0 + r16;
  gn = gn < p.N ? gn : p.N - 1;
  const uint8_t* wrow = (const uint8_t*)p.B + (int64_t)gn * p.ldb;
  const uint32_t* srow = (const uint32_t*)p.bscale + gn;

  f32x4 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (int kc = k_begin; kc < k_end; kc += KC) {
    u32x4 w[KB];
    uint32_t sc[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      // a block past the end of the range: any block of the row, its
      // activations are zeros and its scale 1
      const int k = kc + b * 128 + q * 32;
      const bool in = k < k_end;
      w[b] = *reinterpret_cast<const u32x4*>(wrow + (in ? k : k_begin) / 2);
      const uint32_t word = srow[(int64_t)((in ? k : k_begin) / 128) * p.ld_scale];
      sc[b] = in ? (word >> (8 * q)) & 0xffu : 127u;
    }
    if (kc != k_begin) __syncthreads();
#pragma unroll 4
    for (int i = tid; i < BM * (KC / 8); i += kFrThreads) {
      const int r = i / (KC / 8), c = i % (KC / 8);
      int gm = m0 + r;
      gm = gm < p.M ? gm : p.M - 1;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (kc + c * 8 < k_end) v = *reinterpret_cast<const u32x4*>(p.A + (int64_t)gm * p.lda + kc + c * 8);
      *reinterpret_cast<u32x4*>(lds + r * ROWB + (c ^ ((r >> 3) & 1)) * 16) = v;
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const float s = e8m0_to_f32_valu(sc[b]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 wf = fp4x8_bf16(w[b][j], s);
        const int c = b * 16 + q * 4 + j;
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const bf16x8 x =
              *reinterpret_cast<const bf16x8*>(lds + (i * 16 + r16) * ROWB + (c ^ ((r16 >> 3) & 1)) * 16);
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, x, acc[i], 0, 0, 0);
        }
      }
    }
  }
  const int n = n0 + 4 * q;  // N % 8 == 0: four columns inside or outside
  if (n >= p.N) return;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int m = m0 + i * 16 + r16;
    if (m >= p.M) continue;
    if constexpr (EPI == kEpiPartial)
      *reinterpret_cast<f32x4*>(p.partial + ((int64_t)kz * p.M + m) * p.N + n) = acc[i];
    else
      fp4_store4<EPI>(p, acc[i], m, n);
  }
}

// ---- one to 16 rows ----------------------------------------------------------
// Bound by latency and the weight bytes: one launch, no workspace, a wave's
// loads of up to 512 k issued before their first use.  A workgroup computes NB *
// 16 columns; its waves split K, each streaming its range of the codes (and the
// activations, which the L2 holds) straight to registers, and meet once through
// LDS, in wave order.  NB = 2 halves the reads of the activations, where that
// leaves workgroups for every CU.  Weights from HBM: 1 x 4096 -> 4096 6.0 us (10.8
// in 8 K ranges and a combining launch of the few-row tiles, 11.2 in 4 of the
// mid-size kernel; a launch that does next to nothing takes 4.0), 1 x 4096 ->
// 16384 12.5, 16 x 4096 -> 4096 8.7.  Holding the next 512 k in flight as well
// cost more in occupancy than it gave (1 x 4096 -> 16384, one fragment of columns:
// 16.9 against 13.8); 16 waves are no faster.
constexpr int kSkWaves = 8;

template <int NB, int EPI>
__global__ __launch_bounds__(kSkWaves * 64) void fp4_skinny_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(16))) f32x4 part[kSkWaves][NB][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int n0 = (int)blockIdx.x * (16 * NB);
  const uint8_t* wrow[NB];
  const uint32_t* srow[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c) {
    int gn = n0 + c * 16 + r16;  // columns past N re-read the last one, rows past M the last row
    gn = gn < p.N ? gn : p.N - 1;
    wrow[c] = (const uint8_t*)p.B + (int64_t)gn * p.ldb + q * 16;
    srow[c] = (const uint32_t*)p.bscale + gn;
  }
  const bf16* xrow = p.A + (int64_t)(r16 < p.M ? r16 : p.M - 1) * p.lda + q * 32;
  f32x4 acc[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c) acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // U units of 128 k from unit u on.  HALF: only the first 64 k of one exist; the
  // upper quarters take the lower ones' codes, with scale 1, and zeros for x
  auto run = [&](int u, auto uc, auto hc) __attribute__((always_inline)) {
    constexpr int U = decltype(uc)::value;
    constexpr bool HALF = decltype(hc)::value;
    const bool out = HALF && q >= 2;
    const int back = out ? 64 : 0;  // in k
    u32x4 w[U][NB];
    uint32_t sc[U][NB];
#pragma unroll
    for (int b = 0; b < U; ++b)
#pragma unroll
      for (int c = 0; c < NB; ++c) {
        w[b][c] = *reinterpret_cast<const u32x4*>(wrow[c] + (u + b) * 64 - back / 2);
        sc[b][c] = srow[c][(int64_t)(u + b) * p.ld_scale];
      }
    bf16x8 x[U][4];
#pragma unroll
    for (int b = 0; b < U; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[b][j] = *reinterpret_cast<const bf16x8*>(xrow + (u + b) * 128 - back + j * 8);
        if (out) x[b][j] = bf16x8{};
      }
#pragma unroll
    for (int b = 0; b < U; ++b)
#pragma unroll
      for (int c = 0; c < NB; ++c) {
        const float s = out ? 1.0f : e8m0_to_f32_valu((sc[b][c] >> (8 * q)) & 0xffu);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4x8_bf16(w[b][c][j], s), x[b][j], acc[c], 0, 0, 0);
      }
  };
  const int units = p.K >> 7;
  int u = units * wave / kSkWaves;
  const int end = units * (wave + 1) / kSkWaves;
  constexpr std::integral_constant<int, 4> c4;
  constexpr std::integral_constant<int, 2> c2;
  constexpr std::integral_constant<int, 1> c1;
  constexpr std::false_type whole;
  for (; u + 4 <= end; u += 4) run(u, c4, whole);
  if (u + 2 <= end) {
    run(u, c2, whole);
    u += 2;
  }
  if (u < end) run(u, c1, whole);
  if ((p.K & 64) && wave == kSkWaves - 1) run(units, c1, std::true_type{});

#pragma unroll
  for (int c = 0; c < NB; ++c) part[wave][c][lane] = acc[c];
  __syncthreads();
  if (wave >= NB) return;
  const int n = n0 + wave * 16 + 4 * q;  // N % 8 == 0: four columns inside or outside
  f32x4 a = part[0][wave][lane];
#pragma unroll
  for (int z = 1; z < kSkWaves; ++z) {
    const f32x4 b = part[z][wave][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] += b[e];
  }
  if (r16 < p.M && n < p.N) fp4_store4<EPI>(p, a, r16, n);
}

// sum of the partial products in split order, then the epilogue
template <int EPI>
__global__ __launch_bounds__(256) void fp4_combine_kernel(GemmArgs p, int splits) {
  const int per_row = p.N / 4;
  const int64_t total = (int64_t)p.M * per_row, plane = (int64_t)p.M * p.N;
  for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < total; idx += (int64_t)gridDim.x * 256) {
    const int m = (int)(idx / per_row), n = (int)(idx % per_row) * 4;
    const float* P = p.partial + (int64_t)m * p.N + n;
    f32x4 a = *reinterpret_cast<const f32x4*>(P);
    for (int z = 1; z < splits; ++z) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(P + z * plane);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] += b[e];
    }
    fp4_store4<EPI>(p, a, m, n);
  }
}

int fp4_combine(const GemmArgs& p, int epi, int splits, hipStream_t s) {
  const int64_t total = (int64_t)p.M * (p.N / 4);
  const int blocks = (int)((total + 255) / 256 < 4096 ? (total + 255) / 256 : 4096);
  if (!fp4_epilogue(epi, [&](auto e) { fp4_combine_kernel<decltype(e)::value><<<blocks, 256, 0, s>>>(p, splits); }))
    return LTX_ERR_INVALID_ARG;
  return ltx_launch_status();
}

// ---- which kernel ------------------------------------------------------------
// kFp4Skinny, kFp4Rows: above.  kFp4Mid: the mid-size kernel (gemm_kg.hip), tiles
// of 64, 128 or 192 x 128, whole units of 128 k.  kFp4Large: the 8-wave kernel
// (gemm8.h), 128 x 256.  Before it, rows [0, head) on the 8-wave kernel's 256 x 256
// tiles: where those make whole rounds of the CUs and another kernel takes the
// rows left over for less than one more round.
enum Fp4Kernel { kFp4Skinny, kFp4Rows, kFp4Mid, kFp4Large };
struct Fp4Plan {
  int64_t head;  // a multiple of 256, or M: all rows
  int kernel;    // of the rows from head on
  int bm;        // rows of its tiles (kFp4Skinny: columns of a workgroup)
  int splits;    // its K ranges (1 with a head)
  int k_split;   // k of one (a multiple of 128)
};

// Modelled times (us) of one launch.  Mid-size: a round of one workgroup per CU
// costs `unit` us per 128 k, the L2s deliver 13 TB/s of tile operands at most, 4 us
// of launch, first loads and epilogue, a split's second launch and its partials.
// Against measured: 1296 x 4096 -> 4096 tiles of 192 / 128 / 64 rows 39 / 53 / 57
// against 40 / 56 / 56, 68 x 2048 -> 8192 64 rows 13 / 12, 68 x 8192 -> 2048 in 8
// splits 64 rows 14 / 16, 256 x 4096 -> 8192 22 / 21.
static inline int64_t fp4_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
static double fp4_mid_time(int64_t M, int64_t N, int64_t K, int bm, int splits) {
  const double unit = bm == 64 ? 0.55 : (bm == 128 ? 0.77 : 1.08);
  const int64_t wgs = fp4_up(M, bm) * fp4_up(N, 128) * splits;
  const double units = (double)(K / 128) / splits;
  double t = (double)fp4_up(wgs, 256) * units * unit;
  const double bytes = (double)wgs * units * 128 * (2.0 * bm + 64);
  if (bytes / 13e6 > t) t = bytes / 13e6;
  t += 4.0;
  if (splits > 1) t += 3.5 + (double)(M * N) * splits * 8 / 3.5e6;
  return t;
}
// 8-wave: a round of 256-row tiles 2.3 us per 128 k, of 128-row tiles 1.5 (3456 x
// 4096 -> 4096 in one round 79; 3456 x 16384 -> 4096 287; 1296 x 4096 -> 4096 in
// 128-row tiles 50).
static double fp4_large_time(int64_t M, int64_t N, int64_t K, int bm) {
  return 4.0 + (double)(fp4_up(fp4_up(M, bm) * fp4_up(N, 256), 256) * fp4_up(K, 128)) * (bm == 256 ? 2.3 : 1.5);
}
// Up to 16 rows: every workgroup reads all activations; 32 columns each where
// that leaves one for every CU (16 / 32 columns: 16 x 4096 -> 12320 22.5 / 15.3 us,
// 4 x 4096 -> 16384 15.9 / 13.4, 1 x 2048 -> 8192 5.9 / 5.9, 16 x 4096 -> 4096 8.7 / 9.4,
// 1 x 16384 -> 4096 14.8 / 19.9).
static int fp4_skinny_cols(int64_t N) { return N >= 32 * 256 ? 32 : 16; }
static double fp4_skinny_time(int64_t M, int64_t N, int64_t K) {
  const double weights = (double)(N * K) * 0.53 / 3.6e6, rows = (double)N / 256 / fp4_skinny_cols(N) * (double)(M * K) * 2 / 47e3;
  return 4.0 + (weights > rows ? weights + 0.5 * rows : rows + 0.5 * weights);
}

// The fastest single launch (or, where `split`, K ranges and a combining one)
static double fp4_one(int64_t M, int64_t N, int64_t K, bool split, Fp4Plan* pl) {
  const int whole = (int)((K + 127) / 128 * 128);
  double best = fp4_large_time(M, N, K, 128);
  *pl = {0, kFp4Large, 128, 1, whole};
  if (M <= 16) {
    const double t = fp4_skinny_time(M, N, K);
    if (t < best) {
      best = t;
      *pl = {0, kFp4Skinny, fp4_skinny_cols(N), 1, whole};
    }
  }
  const int64_t units = fp4_up(K, 128);
  if (K % 128 != 0) {
    // half a scale word past the last unit: not the mid-size kernel's.  Few-row
    // tiles in any K ranges of at least 512 k (a round of 256 workgroups 1.6 us
    // per 128 k: 256 x 4096 -> 8192 55, 68 x 8192 -> 2048 in 8 ranges 21)
    const int bm = M <= 32 ? 32 : 64;
    const int64_t tiles = fp4_up(M, bm) * fp4_up(N, kFrBN);
    for (int s = 1; s <= (split ? 32 : 1); ++s) {
      if (s > 1 && (tiles * s > 512 || units / s < 4)) break;
      const int64_t per = fp4_up(units, s), n = fp4_up(units, per);
      double t = 4.0 + (double)(fp4_up(tiles * n, 256) * per) * 1.6;
      if (n > 1) t += 3.5 + (double)(M * N * n) * 8 / 3.5e6;
      if (t < best * (n > 1 ? 0.9 : 1.0)) {
        best = t;
        *pl = {0, kFp4Rows, bm, (int)n, (int)(per * 128)};
      }
    }
    return best;
  }
  for (int bm = 64; bm <= 192; bm += 64) {
    const int64_t tiles = ((M + bm - 1) / bm) * ((N + 127) / 128);
    for (int s = 1; s <= (split ? 16 : 1); ++s) {
      // splits: whole units, at least 256 k each, within one round of the CUs,
      // and 10 % faster (a launch and a workspace more)
      if (s > 1 && (tiles * s > 256 || units / s < 2)) break;
      if (units % s) continue;
      const double t = fp4_mid_time(M, N, K, bm, s);
      if (t < best * (s > 1 ? 0.9 : 1.0)) {
        best = t;
        *pl = {0, kFp4Mid, bm, s, (int)(K / s)};
      }
    }
  }
  return best;
}

static Fp4Plan fp4_plan(int64_t M, int64_t N, int64_t K) {
  Fp4Plan pl;
  if (M <= 16 && M * K <= 16384) return {0, kFp4Skinny, fp4_skinny_cols(N), 1, (int)K};  // a few rows: the launch, not the choice, counts
  double best = fp4_one(M, N, K, true, &pl);
  if (M <= 128) return pl;
  const double all = fp4_large_time(M, N, K, 256);
  if (all < best) {
    best = all;
    pl = {M, kFp4Large, 128, 1, (int)((K + 127) / 128 * 128)};
  }
  for (int64_t b = (M - 1) / 256, tries = 0; b >= 1 && tries < 16; --b, ++tries) {
    Fp4Plan rest;
    const double t = fp4_large_time(256 * b, N, K, 256) + fp4_one(M - 256 * b, N, K, false, &rest);
    if (t < 0.97 * best) {
      best = t;
      pl = rest;
      pl.head = 256 * b;
    }
  }
  return pl;
}

template <int EPI>
static void fp4_launch_rows(const GemmArgs& p, int bm, int splits, int k_split, hipStream_t s) {
  GemmArgs a = p;
  a.tiles_m = (p.M + bm - 1) / bm;
  a.tiles_n = (p.N + kFrBN - 1) / kFrBN;
  const int blocks = a.tiles_m * a.tiles_n * splits;
  if (bm == 32) fp4_rows_kernel<2, EPI><<<blocks, kFrThreads, 0, s>>>(a, k_split);
  else fp4_rows_kernel<4, EPI><<<blocks, kFrThreads, 0, s>>>(a, k_split);
}

// one launch of the plan's kernel (EPI kEpiPartial: its K ranges)
template <int EPI>
static void fp4_launch(const GemmArgs& p, const Fp4Plan& pl, hipStream_t s) {
  if (pl.kernel == kFp4Rows) {
    fp4_launch_rows<EPI>(p, pl.bm, pl.splits, pl.k_split, s);
  } else if (pl.kernel == kFp4Mid) {
    GemmArgs a = p;
    if (EPI == kEpiPartial) {
      a.K = pl.k_split;
      a.ldc = p.N;
    }
    kg_launch(B_MXFP4, a, EPI, pl.bm, pl.splits, s);
  } else if constexpr (EPI != kEpiPartial) {
    if (pl.kernel == kFp4Skinny && pl.bm == 32) fp4_skinny_kernel<2, EPI><<<(p.N + 31) / 32, kSkWaves * 64, 0, s>>>(p);
    else if (pl.kernel == kFp4Skinny) fp4_skinny_kernel<1, EPI><<<(p.N + 15) / 16, kSkWaves * 64, 0, s>>>(p);
    else launch_g8<B_MXFP4, EPI, 128>(p, s);
  }
}

// Rows of activations that one launch of the mid-size or the 8-wave kernel takes: their
// operands' byte offsets have 31 bits.  All rows, or fewer in whole tiles (of 64, 128,
// 192 or 256 rows); 0: those kernels do not take the product (weights, scale words or a
// single tile's rows of 2 GiB), the few-row tiles do.
static int64_t fp4_rows_per_launch(const GemmArgs& p, int64_t rows) {
  const int64_t lim = ((int64_t)1 << 31) - 1, most = lim / (p.lda * 2);
  if (p.N > lim / p.ldb || p.ld_scale > lim / 4 / ((p.K + 127) / 128)) return 0;
  return rows <= most ? rows : most / 768 * 768;
}

}  // namespace ltx

using namespace ltx;

extern "C" int64_t ltx_gemm_mxfp4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return -1;
  if (M == 0 || N == 0 || K == 0 || M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2) return 0;
  const Fp4Plan pl = fp4_plan(M, N, K);
  return pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0;
}

extern "C" int ltx_gemm_mxfp4_bf16(const void* A, int64_t lda, const uint8_t* Wq, int64_t ldw,
                                   const uint32_t* w_scale, int64_t ld_scale, const float* bias, void* C,
                                   int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue,
                                   const void* residual, int64_t ldr, const float* gate, int64_t sigmoid_from,
                                   float* workspace, int64_t workspace_bytes, void* stream) {
  const int st = fp4_check(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, epilogue, residual, ldr, gate,
                           K, 8);
  if (st != LTX_OK) return st;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  Fp4Plan pl = fp4_plan(M, N, K);
  const int64_t need = pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return LTX_ERR_INVALID_ARG;
  if (need > 0 && ((uintptr_t)workspace & 15u)) return LTX_ERR_ALIGNMENT;
  GemmArgs p = fp4_args(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, epilogue, residual, ldr, gate,
                        sigmoid_from);
  hipStream_t s = (hipStream_t)stream;
  const int epi = epilogue & 0xff;
  if (pl.splits > 1) {
    if (pl.kernel == kFp4Mid && fp4_rows_per_launch(p, M) < M) {
      pl.kernel = kFp4Rows;
      pl.bm = 64;
    }
    p.partial = workspace;
    fp4_launch<kEpiPartial>(p, pl, s);
    const int e = ltx_launch_status();
    return e != LTX_OK ? e : fp4_combine(p, epi, pl.splits, s);
  }
  // rows [r0, r1) on a kernel: the mid-size and 8-wave kernels in pieces of as many
  // as a launch takes; what they do not take on the few-row tiles
  auto run = [&](int64_t r0, int64_t r1, bool head) {
    int64_t piece = r1 - r0;
    Fp4Plan q = pl;
    bool large = head;
    if (head || q.kernel == kFp4Mid || q.kernel == kFp4Large) {
      piece = fp4_rows_per_launch(p, r1 - r0);
      if (piece == 0) {
        piece = r1 - r0;
        q.kernel = kFp4Rows;
        q.bm = 64;
        q.splits = 1;
        q.k_split = (int)((K + 127) / 128 * 128);
        large = false;
      }
    }
    for (; r0 < r1; r0 += piece) {
      GemmArgs part = rows_from(p, r0);
      part.M = (int)(r1 - r0 < piece ? r1 - r0 : piece);
      fp4_epilogue(epi, [&](auto e) {
        if (large) launch_g8<B_MXFP4, decltype(e)::value>(part, s);
        else fp4_launch<decltype(e)::value>(part, q, s);
      });
      const int e = ltx_launch_status();
      if (e != LTX_OK) return e;
    }
    return LTX_OK;
  };
  if (pl.head > 0) {
    const int e = run(0, pl.head, true);
    if (e != LTX_OK || pl.head >= M) return e;
  }
  return run(pl.head, M, false);
}
