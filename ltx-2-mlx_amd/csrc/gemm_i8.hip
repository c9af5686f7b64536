// Projection GEMMs of int8 rows and int8 weights on the int8 MFMA
// (v_mfma_i32_16x16x64_i8):
//
//   C[m, n] = epilogue( (sum_k a[m, k] w[n, k]) sa[m] sw[n] + bias[n] ),
//
// a scale per row and per output channel.  The sum is exact in int32, so however
// the work is split the results are the same bits; scales, bias and epilogue are
// fp32 (the MXFP4 products' epilogue: gemm_fp4.h).
#include "gemm_fp4.h"

namespace ltx {

__device__ __forceinline__ const int8_t* i8_rows(const GemmArgs& p) { return (const int8_t*)p.A; }
__device__ __forceinline__ const int8_t* i8_weights(const GemmArgs& p) { return (const int8_t*)p.B; }
__device__ __forceinline__ const float* i8_row_scale(const GemmArgs& p) { return (const float*)p.ascale; }
__device__ __forceinline__ const float* i8_col_scale(const GemmArgs& p) { return (const float*)p.bscale; }

// Four columns of a row from their sums.  Products that are never fused with the
// bias: the same bits in every kernel.
__device__ __forceinline__ f32x4 i8_value(i32x4 a, float sa, f32x4 sw) {
  f32x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = mul_rn(mul_rn((float)a[e], sa), sw[e]);
  return y;
}
// (scales need no 16-byte alignment)
__device__ __forceinline__ f32x4 i8_four(const float* v) { return f32x4{v[0], v[1], v[2], v[3]}; }

__device__ __forceinline__ void i8_store4(const GemmArgs& p, int epi, i32x4 a, int m, int n) {
  const f32x4 y = i8_value(a, i8_row_scale(p)[m], i8_four(i8_col_scale(p) + n));
  if (epi == LTX_GEMM_EPI_BIAS) fp4_store4<LTX_GEMM_EPI_BIAS>(p, y, m, n);
  else if (epi == LTX_GEMM_EPI_GELU) fp4_store4<LTX_GEMM_EPI_GELU>(p, y, m, n);
  else if (epi == LTX_GEMM_EPI_RESIDUAL) fp4_store4<LTX_GEMM_EPI_RESIDUAL>(p, y, m, n);
  else if (epi == LTX_GEMM_EPI_RESIDUAL_ROUND) fp4_store4<LTX_GEMM_EPI_RESIDUAL_ROUND>(p, y, m, n);
  else fp4_store4<LTX_GEMM_EPI_SIGMOID2>(p, y, m, n);
}

// ---- few rows ------------------------------------------------------------------
// A workgroup computes MB * 16 rows x NB * 16 columns; its eight waves split K, each
// streaming its range of both operands straight to registers (lane (r16, q): row
// r16, bytes 16 q of 64 k), and meet once through LDS.
constexpr int kI8Waves = 8;

template <int MB, int NB>
__global__ __launch_bounds__(kI8Waves * 64) void i8_rows_kernel(GemmArgs p, int epi) {
  __shared__ __attribute__((aligned(16))) i32x4 part[kI8Waves][MB * NB][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int n0 = (int)blockIdx.x % p.tiles_n * (16 * NB), m0 = (int)blockIdx.x / p.tiles_n * (16 * MB);
  const int8_t *wrow[NB], *xrow[MB];
#pragma unroll
  for (int c = 0; c < NB; ++c) {  // columns past N re-read the last one, rows past M the last row
    const int gn = n0 + c * 16 + r16;
    wrow[c] = i8_weights(p) + (int64_t)(gn < p.N ? gn : p.N - 1) * p.ldb + q * 16;
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int gm = m0 + i * 16 + r16;
    xrow[i] = i8_rows(p) + (int64_t)(gm < p.M ? gm : p.M - 1) * p.lda + q * 16;
  }
  i32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int c = 0; c < NB; ++c) acc[i][c] = i32x4{0, 0, 0, 0};
  auto run = [&](int u, auto uc) __attribute__((always_inline)) {  // units of 64 k from u on
    constexpr int U = decltype(uc)::value;
    i32x4 w[U][NB], x[U][MB];
#pragma unroll
    for (int b = 0; b < U; ++b) {
#pragma unroll
      for (int c = 0; c < NB; ++c) w[b][c] = *reinterpret_cast<const i32x4*>(wrow[c] + (u + b) * 64);
#pragma unroll
      for (int i = 0; i < MB; ++i) x[b][i] = *reinterpret_cast<const i32x4*>(xrow[i] + (u + b) * 64);
    }
#pragma unroll
    for (int b = 0; b < U; ++b)
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[i][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[b][c], x[b][i], acc[i][c], 0, 0, 0);
  };
  const int units = p.K >> 6;
  int u = (int)((int64_t)units * wave / kI8Waves);
  const int end = (int)((int64_t)units * (wave + 1) / kI8Waves);
  constexpr int U = MB + NB <= 4 ? 8 : (MB + NB <= 8 ? 4 : 2);
  for (; u + U <= end; u += U) run(u, std::integral_constant<int, U>{});
  if constexpr (U > 4)
    if (u + 4 <= end) {
      run(u, std::integral_constant<int, 4>{});
      u += 4;
    }
  for (; u < end; ++u) run(u, std::integral_constant<int, 1>{});
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int c = 0; c < NB; ++c) part[wave][i * NB + c][lane] = acc[i][c];
  __syncthreads();
  for (int f = wave; f < MB * NB; f += kI8Waves) {
    i32x4 a = part[0][f][lane];
#pragma unroll
    for (int z = 1; z < kI8Waves; ++z) a += part[z][f][lane];
    const int m = m0 + f / NB * 16 + r16, n = n0 + f % NB * 16 + 4 * q;  // N % 8 == 0: four columns inside or outside
    if (m < p.M && n < p.N) i8_store4(p, epi, a, m, n);
  }
}

template <int MB, int NB>
static void i8_launch_rows(GemmArgs p, int epi, hipStream_t s) {
  p.tiles_n = (p.N + 16 * NB - 1) / (16 * NB);
  p.tiles_m = (p.M + 16 * MB - 1) / (16 * MB);
  i8_rows_kernel<MB, NB><<<p.tiles_m * p.tiles_n, kI8Waves * 64, 0, s>>>(p, epi);
}

static inline int i8_check(const void* A, int64_t lda, const float* a_scale, const void* W, int64_t ldw,
                           const float* w_scale, const float* bias, const void* C, int64_t ldc, int64_t M, int64_t N,
                           int64_t K, int epilogue, const void* R, int64_t ldr, const float* gate) {
  auto al = [](const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; };
  if (!A || !a_scale || !W || !w_scale || !C || M < 0 || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  const int64_t size = 1 << 27, stride = (int64_t)1 << 40;
  if (M > size || N > size || M * N > (int64_t)1 << 34) return LTX_ERR_UNSUPPORTED;
  if (lda > stride || ldw > stride || ldc > stride || ldr > stride) return LTX_ERR_UNSUPPORTED;
  const int epi = epilogue & 0xff;
  if (epilogue & ~(0xff | LTX_GEMM_ROUND_THEN_BIAS) || epi > LTX_GEMM_EPI_SIGMOID2) return LTX_ERR_INVALID_ARG;
  const bool resid = epi == LTX_GEMM_EPI_RESIDUAL || epi == LTX_GEMM_EPI_RESIDUAL_ROUND;
  if (resid && (!R || !gate || ldr < N)) return LTX_ERR_INVALID_ARG;
  if (K % 64 != 0 || N % 8 != 0 || K >= 1 << 17) return LTX_ERR_UNSUPPORTED;  // 128 * 128 * K < 2^31
  if (lda < K || ldw < K || ldc < N) return LTX_ERR_INVALID_ARG;
  if (!al(A, 16) || !al(W, 16) || !al(C, 16) || !al(a_scale, 4) || !al(w_scale, 4) || !al(bias, 4) || !al(gate, 4) ||
      lda % 16 || ldw % 16 || ldc % 8 || (resid && (!al(R, 16) || ldr % 8)))
    return LTX_ERR_ALIGNMENT;
  return LTX_OK;
}

}  // namespace ltx

using namespace ltx;

extern "C" int64_t ltx_gemm_i8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return -1;
  return 0;
}

extern "C" int ltx_gemm_i8_bf16(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* Wq, int64_t ldw,
                                const float* w_scale, const float* bias, void* C, int64_t ldc, int64_t M, int64_t N,
                                int64_t K, int epilogue, const void* residual, int64_t ldr, const float* gate,
                                int64_t sigmoid_from, void* workspace, int64_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  const int st = i8_check(A, lda, a_scale, Wq, ldw, w_scale, bias, C, ldc, M, N, K, epilogue, residual, ldr, gate);
  if (st != LTX_OK) return st;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  GemmArgs p = {};
  p.A = (const bf16*)A;
  p.lda = lda;
  p.ascale = (const uint8_t*)a_scale;
  p.B = Wq;
  p.ldb = ldw;
  p.bscale = w_scale;
  p.bias = bias;
  p.C = (bf16*)C;
  p.ldc = ldc;
  p.R = (const bf16*)residual;
  p.ldr = ldr;
  p.gate = gate;
  p.sig_from = (int)(sigmoid_from < N ? (sigmoid_from < 0 ? 0 : sigmoid_from) : N);
  p.round_then_bias = (epilogue & LTX_GEMM_ROUND_THEN_BIAS) != 0;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  hipStream_t s = (hipStream_t)stream;
  const int epi = epilogue & 0xff;
  if (M <= 16) i8_launch_rows<1, 1>(p, epi, s);
  else i8_launch_rows<4, 2>(p, epi, s);
  return ltx_launch_status();
}
