// MXFP4 operands of the projection GEMMs (gemm_fp4.hip: bf16 rows x MXFP4
// weights; gemm_mx4.hip: MXFP4 rows x MXFP4 weights) and their epilogue.
//
// Storage: E2M1 codes (rows, K / 2 bytes), the even k in the low nibble, and
// the E8M0 scales of 32-element blocks as words (ceil(K / 128), ld): word
// [k / 128][row] holds the four blocks of those 128 k, the first in its low
// byte.  The words of neighbouring rows are neighbours, so the scales of a
// tile's rows for 128 k are one contiguous piece (a (rows, K / 32) array gives
// every row's few bytes a line of its own: beside 4-bit codes those lines
// would be a third of all requests).  Bytes past K hold no block and are not
// used.
#pragma once

#include "gemm_common.h"

namespace ltx {

// Four consecutive columns n .. n + 3 of an output row from their fp32 sums, up
// to the residual.  MXFP4 products reproduce no reference arithmetic, so GELU, the
// head gate and the gated residual act on the fp32 value, without the other
// formats' bf16 rounding before them (EPI_RESIDUAL_ROUND is the form that rounds).
// SIG: columns from sig_from on may be among these; RTB: round_then_bias.
template <int EPI, bool SIG, bool RTB>
__device__ __forceinline__ f32x4 fp4_branch4(const GemmArgs& p, f32x4 a, f32x4 bias, int n) {
  float y[4] = {a[0], a[1], a[2], a[3]};
  if (RTB) {
    round_bf2(y[0], y[1]);
    round_bf2(y[2], y[3]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] += bias[e];
    if (EPI == LTX_GEMM_EPI_GELU) y[e] = gelu_tanh(y[e]);
    if (EPI == LTX_GEMM_EPI_SIGMOID2) y[e] = sigmoid2_bf(y[e]);
    if (SIG) {  // both, then a choice: not a branch per value
      float g = sigmoid2_bf(y[e]);
      asm("" : "+v"(g));
      y[e] = n + e >= p.sig_from ? g : y[e];
    }
  }
  return f32x4{y[0], y[1], y[2], y[3]};
}
__device__ __forceinline__ bf16x4 fp4_bf16(f32x4 y) { return bf16x4{(bf16)y[0], (bf16)y[1], (bf16)y[2], (bf16)y[3]}; }
template <int EPI>
__device__ __forceinline__ bf16 fp4_residual(float y, bf16 r, float g) {
  return (bf16)(EPI == LTX_GEMM_EPI_RESIDUAL ? fmaf(g, y, (float)r) : round_bf(round_bf(y) * g) + (float)r);
}
template <int EPI>
__device__ __forceinline__ void fp4_store4(const GemmArgs& p, f32x4 a, int m, int n) {
  f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.bias)
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = p.bias[n + e];
  constexpr bool SIG = EPI == LTX_GEMM_EPI_BIAS;
  const f32x4 y = p.round_then_bias ? fp4_branch4<EPI, SIG, true>(p, a, bias, n) : fp4_branch4<EPI, SIG, false>(p, a, bias, n);
  bf16x4 v = fp4_bf16(y);
  if constexpr (EPI == LTX_GEMM_EPI_RESIDUAL || EPI == LTX_GEMM_EPI_RESIDUAL_ROUND) {
    const bf16x4 r = *reinterpret_cast<const bf16x4*>(p.R + (int64_t)m * p.ldr + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fp4_residual<EPI>(y[e], r[e], p.gate[n + e]);
  }
  *reinterpret_cast<bf16x4*>(p.C + (int64_t)m * p.ldc + n) = v;
}

// Residual epilogue of a wave that holds NB x 4 accumulator blocks of 16 x 16 (lane
// (r16, q): row r16, columns 4 q .. 4 q + 3), rows row0 on and columns col0 on; acc(i,
// j) is block (i, j), bias and gate the wave's 64 columns.  The branch stays fp32: PASS
// row blocks at a time go through PASS * 4 KiB of LDS, which only this wave uses, in
// rows of 256 bytes with their 16-byte chunks XORed by the row, and come back as rows of
// eight columns per lane.  All residual rows are read before the first is written.
template <int EPI, int NB, int PASS, class Acc>
__device__ __forceinline__ void fp4_residual_rows(const GemmArgs& p, char* E, const float* bias, const float* gate,
                                                  int row0, int col0, int lane, Acc acc) {
  static_assert(NB % PASS == 0, "whole passes");
  const int r16 = lane & 15, q = lane >> 4, ch = lane & 7, rsub = lane >> 3;
  const int gn = col0 + ch * 8;
  const bool ok = gn < p.N;  // N % 8 == 0
  bf16x8 res[NB * 2];
  float g8[8];
  auto stage = [&](int i0, auto rtb) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(bias + j * 16 + 4 * q);
#pragma unroll
      for (int i = 0; i < PASS; ++i) {
        const int row = i * 16 + r16;
        *reinterpret_cast<f32x4*>(E + row * 256 + (((4 * j + q) ^ row) & 15) * 16) =
            fp4_branch4<EPI, false, decltype(rtb)::value>(p, acc(i0 + i, j), b, 0);
      }
    }
  };
#pragma unroll
  for (int i0 = 0; i0 < NB; i0 += PASS) {
    if (p.round_then_bias) stage(i0, std::true_type{});
    else stage(i0, std::false_type{});
    if (i0 == 0) {  // (after the first accumulators are in LDS: fewer live registers)
#pragma unroll
      for (int it = 0; it < NB * 2; ++it) {
        int gm = row0 + it * 8 + rsub;
        gm = gm < p.M ? gm : p.M - 1;
        res[it] = *reinterpret_cast<const bf16x8*>(p.R + (int64_t)gm * p.ldr + (ok ? gn : 0));
      }
      const f32x4 ga = *reinterpret_cast<const f32x4*>(gate + ch * 8), gb = *reinterpret_cast<const f32x4*>(gate + ch * 8 + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) g8[e] = e < 4 ? ga[e & 3] : gb[e & 3];
    }
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < PASS * 2; ++it) {
      const int ml = it * 8 + rsub, gm = row0 + i0 * 16 + ml;
      const f32x4 a = *reinterpret_cast<const f32x4*>(E + ml * 256 + (((2 * ch) ^ ml) & 15) * 16);
      const f32x4 b = *reinterpret_cast<const f32x4*>(E + ml * 256 + (((2 * ch + 1) ^ ml) & 15) * 16);
      bf16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fp4_residual<EPI>(e < 4 ? a[e & 3] : b[e & 3], res[2 * i0 + it][e], g8[e]);
      if (gm < p.M && ok) *reinterpret_cast<bf16x8*>(p.C + (int64_t)gm * p.ldc + gn) = v;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// sum of `splits` partial products (fp32, split order) and the epilogue
int fp4_combine(const GemmArgs& p, int epi, int splits, hipStream_t s);

// f<EPI>() of an epilogue code; false for an unknown one
template <class F>
static bool fp4_epilogue(int epi, F&& f) {
  switch (epi) {
    case LTX_GEMM_EPI_BIAS: f(std::integral_constant<int, LTX_GEMM_EPI_BIAS>{}); return true;
    case LTX_GEMM_EPI_GELU: f(std::integral_constant<int, LTX_GEMM_EPI_GELU>{}); return true;
    case LTX_GEMM_EPI_RESIDUAL: f(std::integral_constant<int, LTX_GEMM_EPI_RESIDUAL>{}); return true;
    case LTX_GEMM_EPI_RESIDUAL_ROUND: f(std::integral_constant<int, LTX_GEMM_EPI_RESIDUAL_ROUND>{}); return true;
    case LTX_GEMM_EPI_SIGMOID2: f(std::integral_constant<int, LTX_GEMM_EPI_SIGMOID2>{}); return true;
  }
  return false;
}

// Checks shared by the two products; `a_bytes` bytes per row of K activations.
static inline int fp4_check(const void* A, int64_t lda, const void* W, int64_t ldw, const void* w_scale,
                            int64_t ld_scale, const float* bias, const void* C, int64_t ldc, int64_t M, int64_t N,
                            int64_t K, int epilogue, const void* R, int64_t ldr, const float* gate, int64_t lda_min,
                            int64_t lda_unit) {
  auto al = [](const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; };
  if (!A || !W || !w_scale || !C || M < 0 || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  // a launch has fewer than 2^32 threads: 512 for a tile of at least 32 x 128
  // outputs, or for 32 columns of a few rows
  const int64_t size = 1 << 27, stride = (int64_t)1 << 40;
  if (M > size || N > size || K > INT32_MAX / 2 || M * N > (int64_t)1 << 34) return LTX_ERR_UNSUPPORTED;
  if (lda > stride || ldw > stride || ldc > stride || ldr > stride || ld_scale > stride) return LTX_ERR_UNSUPPORTED;
  const int epi = epilogue & 0xff;
  if (epilogue & ~(0xff | LTX_GEMM_ROUND_THEN_BIAS) || epi > LTX_GEMM_EPI_SIGMOID2) return LTX_ERR_INVALID_ARG;
  const bool resid = epi == LTX_GEMM_EPI_RESIDUAL || epi == LTX_GEMM_EPI_RESIDUAL_ROUND;
  if (resid && (!R || !gate || ldr < N)) return LTX_ERR_INVALID_ARG;
  if (K % 64 != 0 || N % 8 != 0) return LTX_ERR_UNSUPPORTED;
  if (lda < lda_min || ldw < K / 2 || ldc < N || ld_scale < N) return LTX_ERR_INVALID_ARG;
  if (!al(A, 16) || !al(W, 16) || !al(C, 16) || !al(w_scale, 16) || !al(bias, 4) || !al(gate, 4) ||
      lda % lda_unit || ldw % 16 || ldc % 8 || ld_scale % 4 || (resid && (!al(R, 16) || ldr % 8)))
    return LTX_ERR_ALIGNMENT;
  return LTX_OK;
}

static inline GemmArgs fp4_args(const void* A, int64_t lda, const void* W, int64_t ldw, const uint32_t* w_scale,
                                int64_t ld_scale, const float* bias, void* C, int64_t ldc, int64_t M, int64_t N,
                                int64_t K, int epilogue, const void* R, int64_t ldr, const float* gate,
                                int64_t sigmoid_from) {
  GemmArgs p = {};
  p.A = (const bf16*)A;
  p.lda = lda;
  p.B = W;
  p.ldb = ldw;
  p.bscale = w_scale;
  p.ld_scale = ld_scale;
  p.bias = bias;
  p.C = (bf16*)C;
  p.ldc = ldc;
  p.R = (const bf16*)R;
  p.ldr = ldr;
  p.gate = gate;
  p.sig_from = (int)(sigmoid_from < N ? (sigmoid_from < 0 ? 0 : sigmoid_from) : N);
  p.round_then_bias = (epilogue & LTX_GEMM_ROUND_THEN_BIAS) != 0;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  return p;
}

}  // namespace ltx
