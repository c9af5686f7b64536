// Projection GEMMs with MXFP4 weights and bf16 activations:
//
//   C[m, n] = epilogue( sum_k A[m, k] * e2m1(W[n, k]) 2^(X[n, k / 32]) + bias[n] )
//
// Operand storage: gemm_fp4.h.  The weights are decoded to bf16 (exact) in
// registers and multiplied on v_mfma_f32_16x16x32_bf16, fp32 accumulation.
#include "gemm_fp4.h"

namespace ltx {

// ---- few-row tiles ---------------------------------------------------------
// A workgroup computes MB * 16 rows x 128 columns over one K range; its 8
// waves take 16 columns each.  A lane (column r16, quarter q) loads the 16
// code bytes of its k block of 32 straight from memory: one block, one scale,
// four MFMA k-steps; the quarter's k run 32 q + 8 j in k-step j, for both
// operands.  The activation rows go through LDS, KC of k at a time, where all
// waves read them.  Takes every size that the products allow.
constexpr int kFrThreads = 512, kFrBN = 128;

template <int MB>
struct FrCfg {
  static constexpr int BM = MB * 16;
  static constexpr int KC = MB <= 4 ? 512 : 256;
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

// How a product runs: rows per tile and K ranges.
struct Fp4Plan {
  int mb;       // 16-row blocks of a tile
  int splits;   // K ranges
  int k_split;  // k of one (a multiple of 128)
};

static Fp4Plan fp4_plan(int64_t M, int64_t N, int64_t K) {
  Fp4Plan pl;
  pl.mb = M <= 16 ? 1 : (M <= 32 ? 2 : 4);
  const int64_t tiles = ((M + pl.mb * 16 - 1) / (pl.mb * 16)) * ((N + kFrBN - 1) / kFrBN);
  const int64_t units = (K + 127) / 128;
  int64_t s = 512 / tiles;
  if (s > units / 4) s = units / 4;
  if (s > 32) s = 32;
  if (s < 1) s = 1;
  const int64_t per = (units + s - 1) / s;
  pl.k_split = (int)(per * 128);
  pl.splits = (int)((units + per - 1) / per);
  return pl;
}

template <int EPI>
static void fp4_launch_rows(const GemmArgs& p, const Fp4Plan& pl, hipStream_t s) {
  GemmArgs a = p;
  a.tiles_m = (p.M + pl.mb * 16 - 1) / (pl.mb * 16);
  a.tiles_n = (p.N + kFrBN - 1) / kFrBN;
  const int blocks = a.tiles_m * a.tiles_n * pl.splits;
  if (pl.mb == 1) fp4_rows_kernel<1, EPI><<<blocks, kFrThreads, 0, s>>>(a, pl.k_split);
  else if (pl.mb == 2) fp4_rows_kernel<2, EPI><<<blocks, kFrThreads, 0, s>>>(a, pl.k_split);
  else fp4_rows_kernel<4, EPI><<<blocks, kFrThreads, 0, s>>>(a, pl.k_split);
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
  const Fp4Plan pl = fp4_plan(M, N, K);
  const int64_t need = pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return LTX_ERR_INVALID_ARG;
  if (need > 0 && ((uintptr_t)workspace & 15u)) return LTX_ERR_ALIGNMENT;
  GemmArgs p = fp4_args(A, lda, Wq, ldw, w_scale, ld_scale, bias, C, ldc, M, N, K, epilogue, residual, ldr, gate,
                        sigmoid_from);
  hipStream_t s = (hipStream_t)stream;
  const int epi = epilogue & 0xff;
  if (pl.splits > 1) {
    p.partial = workspace;
    fp4_launch_rows<kEpiPartial>(p, pl, s);
    const int e = ltx_launch_status();
    return e != LTX_OK ? e : fp4_combine(p, epi, pl.splits, s);
  }
  fp4_epilogue(epi, [&](auto e) { fp4_launch_rows<decltype(e)::value>(p, pl, s); });
  return ltx_launch_status();
}
