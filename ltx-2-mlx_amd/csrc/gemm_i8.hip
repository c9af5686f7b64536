// Projection GEMMs of int8 rows and int8 weights on the int8 MFMA
// (v_mfma_i32_16x16x64_i8):
//
//   C[m, n] = epilogue( (sum_k a[m, k] w[n, k]) sa[m] sw[n] + bias[n] ),
//
// a scale per row and per output channel.  The sum is exact in int32, so however
// the work is split the results are the same bits; scales, bias and epilogue are
// fp32 (the MXFP4 products' epilogue: gemm_fp4.h).
#include "gemm_fp4.h"
#include "gemm_i8_plan.h"

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

// ---- tiles -----------------------------------------------------------------------
// A workgroup computes BM x BN tiles, one after another.  A stage is 128 k: rows of 128
// bytes, one line each, which reach LDS by direct loads into a ring of stages per operand, one
// stream over all its tiles (the next tile's first stages travel during the last
// stages and the epilogue of this one).  A stage has two k-steps of 64, each in two halves of the
// wave's rows: while the MFMAs of one half run, the fragments of the next are read, also
// across the one barrier per stage, so that only a quarter of a wave's activations and two
// k-steps of its weights are in registers beside the sums.
//
// The rings: LDS holds two stages of 256 x 256 tiles and one operand's third.  The weights have it:
// their loads leave two stages ahead, and they are what comes from HBM (every row tile of a
// round reads the same activations from the L2s).  With eight sets of operands in turn 3456 x 16384 ->
// 4096 takes 192 us, 208 with two stages each, 180 with one set; 6144 x 4096 -> 16384 333 / 344 / 322 (one
// card; others take up to 8 % more: 208 / 191 and 350 / 337 in turn / with one set).
// More stages of the smaller tiles: 0 to 4 % slower (their first loads are as many more).
//
// What bounds it: the chip's power.  A stage of 256 x 256 tiles takes 1.4 us with every CU
// busy, 3.0 PO/s (6144 x 4096 -> 16384 without its epilogues 275 us), 1.08 us on zeros; a loop
// of nothing but these MFMAs on such codes reaches 4.1 (32 x 32 x 32: 3.5); the stage without its
// loads takes 1.19 us, without its fragment reads 1.21, without MFMAs 0.99.  With its epilogues that
// product takes 312 us with bias and 330 with GELU (one set of operands).  Measured beside it, one set each: four waves of 128 x 128, sums
// in AGPRs (a third less LDS traffic), 152 against 148 us (4096 x 12288 -> 4096); 224-row tiles, which
// give each CU one at 3456 x 16384 -> 4096, 178 against 181; loads in one half step, all
// fragment reads in the first group, fewer vector instructions in the loop: no change; two
// workgroups per CU of 128 x 128: 459.
template <int BM_, int BN_, int WAVES_M_, int WAVES_N_, int NA_, int NB_>
struct I8Tile {
  static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
  static constexpr int WAVES = WAVES_M * WAVES_N, THREADS = WAVES * 64;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
  static constexpr int TM = WM / 16, TN = WN / 16;
  // fragments of rows of the halves of a k-step: the first's, and the second's
  static constexpr int HM = (TM + 1) / 2;
  static constexpr int half(int h) { return h == 0 ? HM : TM - HM; }
  // direct loads of a wave per stage, 8 rows each (of the activations' last some may repeat a row)
  static constexpr int A_DMA = (BM + 8 * WAVES - 1) / (8 * WAVES), B_DMA = BN / 8 / WAVES;
  // rings of NA stages of activations and NB of weights
  static constexpr int NA = NA_, NB = NB_, A_BYTES = A_DMA * 8 * WAVES * 128, B_BYTES = BN * 128;
  static constexpr int B_OFF = NA * A_BYTES;
  // loads that may be outstanding when the next stage has to be in LDS: those issued after its
  // activations, and after its weights (see the kernel)
  static constexpr int A_LEFT = (NA - 1) * B_DMA + (NA - 2) * A_DMA, B_LEFT = (NB - 2) * (A_DMA + B_DMA);
  static constexpr int LEFT = A_LEFT < B_LEFT ? A_LEFT : B_LEFT;
  static constexpr int LDS_BYTES = B_OFF + NB * B_BYTES;
  static_assert(WM % 16 == 0 && BN % (8 * WAVES) == 0, "whole fragments, whole direct-load instructions per wave");
  static_assert(TM >= 2 && TN % 2 == 0, "two halves, pairs of weight fragments");
  static_assert(NB >= NA && LDS_BYTES <= 160 * 1024, "LDS");
  static_assert(NA * A_DMA + (NB - 1) * B_DMA < 60, "vmcnt range");
};

template <class Cfg, int EPI>
__global__ __launch_bounds__(Cfg::THREADS, 1) void gemm_i8_kernel(GemmArgs p, int k_split) {
  constexpr int BM = Cfg::BM, BN = Cfg::BN, WM = Cfg::WM, WN = Cfg::WN, TM = Cfg::TM, TN = Cfg::TN, HM = Cfg::HM;
  constexpr int NA = Cfg::NA, NB = Cfg::NB, A_DMA = Cfg::A_DMA, B_DMA = Cfg::B_DMA, WAVES = Cfg::WAVES;
  constexpr bool RESID = EPI == LTX_GEMM_EPI_RESIDUAL || EPI == LTX_GEMM_EPI_RESIDUAL_ROUND;
  __shared__ __attribute__((aligned(1024))) char lds[Cfg::LDS_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % Cfg::WAVES_M, wn = wave / Cfg::WAVES_M;
  const int r16 = lane & 15, q = lane >> 4;
  const int tiles = p.tiles_m * p.tiles_n, total = tiles * (EPI == kEpiPartial ? (p.K + k_split - 1) / k_split : 1);
  // tile `id`: its first row and column, and its K range
  auto locate = [&](int id, int& m0, int& n0, int& k0, int& depth) __attribute__((always_inline)) {
    const int kz = EPI == kEpiPartial ? id / tiles : 0;
    int tm, tn;
    tile_coords(id - kz * tiles, tiles, p.tiles_m, p.tiles_n, tm, tn);
    m0 = tm * BM;
    n0 = tn * BN;
    k0 = kz * k_split;
    depth = p.K - k0 < k_split ? p.K - k0 : k_split;  // a multiple of 64
  };

  // ---- direct-load sources (bytes from the operand's start).  Instruction d of a
  // wave fills 8 LDS rows of 128 bytes, lane j the 16-byte slot j & 7 of row j >> 3
  // (the chunk that the row's swizzle puts there).  Rows past M / N re-read the last
  // one.  A k-step takes every other chunk (the reads' pattern for which g8_swz128 leaves
  // no bank conflicts), so a last half stage's four chunks go to the even places.
  const int a_records = (int)((int64_t)(p.M - 1) * p.lda + p.K);
  const int b_records = (int)((int64_t)(p.N - 1) * p.ldb + p.K);
  // Weight fragments j and j + 1 (j even) of a wave hold its columns 16 j + 8 (r16 / 4) +
  // r16 % 4 and the ones 4 further on, so that a lane's sums of the two are eight
  // neighbouring columns; their rows' swizzle takes bit 3 where the activations' takes bit 2.
  const int chunk = (lane & 7) ^ g8_swz128(lane >> 3, true);  // (8 rows on, the swizzle repeats)
  const int b_chunk = (lane & 7) ^ g8_swz128(((lane >> 3) & 3) | (wave & 1) << 2, true);
  const int back = (chunk - (chunk >> 1)) * 16, b_back = (b_chunk - (b_chunk >> 1)) * 16;
  uint32_t a_src[A_DMA], b_src[B_DMA];
  // the stage that an operand's loads are at: its tile, its number there, and the tile's stages
  struct Place {
    int tile, t, stages;
    bool half;  // whether the last stage is a half
  } pa, pb;
  pa.tile = pb.tile = (int)blockIdx.x;
  auto aim = [&](Place& l, bool of_a) __attribute__((always_inline)) {
    int m0, n0, k0, depth;
    locate(l.tile, m0, n0, k0, depth);
    l.t = 0;
    l.stages = (depth + 127) / 128;
    l.half = (depth & 64) != 0;
    if (of_a) {
#pragma unroll
      for (int d = 0; d < A_DMA; ++d) {
        int row = 8 * (WAVES * d + wave) + (lane >> 3);
        if (BM % (8 * WAVES) != 0) row = row < BM ? row : BM - 1;
        const int gm = m0 + row < p.M ? m0 + row : p.M - 1;
        a_src[d] = (uint32_t)((int64_t)gm * p.lda + k0) + chunk * 16;
      }
    } else {
#pragma unroll
      for (int d = 0; d < B_DMA; ++d) {
        int gn = n0 + 8 * (WAVES * d + wave) + (lane >> 3);
        gn = gn < p.N ? gn : p.N - 1;
        b_src[d] = (uint32_t)((int64_t)gn * p.ldb + k0) + b_chunk * 16;
      }
    }
  };
  // load instruction l of the operand's stage, and the step to the stage behind it (past the
  // last tile's: that one again)
  auto load_a = [&](int slot, int l) __attribute__((always_inline)) {
    const bool last = pa.half && pa.t == pa.stages - 1;
    buffer_dma16(p.A, a_records, a_src[l] - (last ? back : 0), pa.t * 128,
                 lds + slot * Cfg::A_BYTES + (WAVES * l + wave) * 1024);
  };
  auto load_b = [&](int slot, int l) __attribute__((always_inline)) {
    const bool last = pb.half && pb.t == pb.stages - 1;
    buffer_dma16(p.B, b_records, b_src[l] - (last ? b_back : 0), pb.t * 128,
                 lds + Cfg::B_OFF + slot * Cfg::B_BYTES + (WAVES * l + wave) * 1024);
  };
  auto advance = [&](Place& l, bool of_a) __attribute__((always_inline)) {
    if (++l.t < l.stages) return;
    if (l.tile + (int)gridDim.x < total) {
      l.tile += (int)gridDim.x;
      aim(l, of_a);
    } else {
      l.t = l.stages - 1;
    }
  };

  // ---- fragments of a k-step: lane (row r16, quarter q) holds the 16 bytes of chunk 2 q + ks
  i32x4 a[2][HM], w[2][TN];
  int c_off[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) c_off[ks] = ((2 * q + ks) ^ g8_swz128(r16, true)) * 16;
  const int a_rd = (wm * WM + r16) * 128, w_rd = Cfg::B_OFF + (wn * WN + 8 * (r16 >> 2) + (r16 & 3)) * 128;
  int slot_a = 0, slot_b = 0;  // of the stage at work
  auto read_a = [&](i32x4& f, int ks, int i) __attribute__((always_inline)) {
    f = *reinterpret_cast<const i32x4*>(lds + slot_a * Cfg::A_BYTES + a_rd + c_off[ks] + i * 2048);
  };
  auto read_w = [&](i32x4& f, int ks, int j) __attribute__((always_inline)) {
    f = *reinterpret_cast<const i32x4*>(lds + slot_b * Cfg::B_BYTES + w_rd + c_off[ks] + (j >> 1) * 4096 + (j & 1) * 512);
  };
  // share j of TN of the reads of half h of k-step ks (of its weights too, where `weights`)
  auto read_share = [&](int ks, int h, bool weights, int j) __attribute__((always_inline)) {
    if (weights) read_w(w[ks][j], ks, j);
#pragma unroll
    for (int i = 0; i < Cfg::half(h); ++i)
      if (i * TN / HM == j) read_a(a[h][i], ks, h * HM + i);
  };
  i32x4 acc[TM][TN];
  // the MFMAs of half h of k-step ks in groups of one weight fragment (weights as the
  // MFMA's first operand: a lane then holds four consecutive output columns); f(j) issues
  // what goes beside group j
  auto step = [&](auto kc, auto hc, auto f) __attribute__((always_inline)) {
    constexpr int KS = decltype(kc)::value, H = decltype(hc)::value;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      f(j);
#pragma unroll
      for (int i = 0; i < Cfg::half(H); ++i)
        acc[H * HM + i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[KS][j], a[H][i], acc[H * HM + i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::integral_constant<int, 0> c0;
  constexpr std::integral_constant<int, 1> c1;

  // ---- prologue: stages 0 to NA - 1 of the activations and to NB - 2 of the weights, the first landed
  aim(pa, true);
  aim(pb, false);
#pragma unroll 1
  for (int t = 0; t < NB - 1; ++t) {
    if (t < NA) {
#pragma unroll
      for (int l = 0; l < A_DMA; ++l) load_a(t, l);
      advance(pa, true);
    }
#pragma unroll
    for (int l = 0; l < B_DMA; ++l) load_b(t, l);
    advance(pb, false);
  }
  if constexpr (NA == NB) {
#pragma unroll
    for (int l = 0; l < A_DMA; ++l) load_a(NA - 1, l);
    advance(pa, true);
  }
  wait_vmcnt<(NA - 1) * A_DMA + (NB - 2) * B_DMA>();
  barrier_nofence();
#pragma unroll
  for (int j = 0; j < TN; ++j) read_share(0, 0, true, j);

  // The stages of all the workgroup's tiles are one stream.  A stage t: the weights of stage t + NB -
  // 1 are loaded into the slot that stage t - 1 left.  Before its last half step, with every
  // read of it done and the next stage landed, the barrier, after which the activations of
  // stage t + NA are loaded into its slot.  (So after the activations of stage t + 1 those of NA - 2
  // stages and the weights of NA - 1 have been issued, after its weights NB - 2 of both.)
  int free_a = 0, free_b = NB - 1;
  auto late = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int l = 0; l < B_DMA; ++l)
      if (l * TN / B_DMA == j) load_b(free_b, l);
  };
  auto early = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int l = 0; l < A_DMA; ++l)
      if (l * TN / A_DMA == j) load_a(free_a, l);
  };
  auto turn = [&]() __attribute__((always_inline)) {
    wait_lgkmcnt0();
    wait_vmcnt<Cfg::LEFT>();
    barrier_nofence();
    free_a = slot_a;
    free_b = slot_b;
    slot_a = slot_a + 1 < NA ? slot_a + 1 : 0;
    slot_b = slot_b + 1 < NB ? slot_b + 1 : 0;
  };
  for (int id = (int)blockIdx.x; id < total; id += (int)gridDim.x) {
    int m0, n0, k0, depth;
    locate(id, m0, n0, k0, depth);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    for (int t = 0; t < depth / 128; ++t) {
      step(c0, c0, [&](int j) __attribute__((always_inline)) {
        read_share(0, 1, false, j);
        late(j);
      });
      advance(pb, false);
      step(c0, c1, [&](int j) __attribute__((always_inline)) { read_share(1, 0, true, j); });
      step(c1, c0, [&](int j) __attribute__((always_inline)) { read_share(1, 1, false, j); });
      turn();
      step(c1, c1, [&](int j) __attribute__((always_inline)) {
        read_share(0, 0, true, j);
        early(j);
      });
      advance(pa, true);
    }
    if ((depth & 64) != 0) {  // the last stage has one k-step
      step(c0, c0, [&](int j) __attribute__((always_inline)) {
        read_share(0, 1, false, j);
        late(j);
      });
      advance(pb, false);
      turn();
      step(c0, c1, early);
      advance(pa, true);
#pragma unroll
      for (int j = 0; j < TN; ++j) read_share(0, 0, true, j);
    }
    // ---- epilogue: from registers, 16 bytes per lane and row, 64 side by side.  Everything
    // that is loaded is loaded before the first store: loads wait for the stores before them.
    int er = r16, eq = q;
    asm volatile("" : "+v"(er), "+v"(eq));  // (keeps what depends on them out of the registers of the stages)
    if constexpr (EPI == kEpiPartial) {
      int32_t* P = (int32_t*)p.partial + (int64_t)(id / tiles) * p.M * p.N;
#pragma unroll
      for (int h = 0; h < TN / 2; ++h) {
        const int n = n0 + wn * WN + 32 * h + 8 * eq;
        if (n >= p.N) continue;  // N % 8 == 0: eight columns inside or outside
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int m = m0 + wm * WM + i * 16 + er;
          if (m >= p.M) continue;
          *reinterpret_cast<i32x4*>(P + (int64_t)m * p.N + n) = acc[i][2 * h];
          *reinterpret_cast<i32x4*>(P + (int64_t)m * p.N + n + 4) = acc[i][2 * h + 1];
        }
      }
    } else {
      float sa[TM];
      f32x4 sw[TN], bias[TN], gate[TN];
      auto columns = [&](int j) __attribute__((always_inline)) {
        int n = n0 + wn * WN + 32 * (j >> 1) + 8 * eq;
        n = (n < p.N ? n : 0) + 4 * (j & 1);
        sw[j] = i8_four(i8_col_scale(p) + n);
        bias[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (p.bias) bias[j] = i8_four(p.bias + n);
        if constexpr (RESID) gate[j] = i8_four(p.gate + n);
      };
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int m = m0 + wm * WM + i * 16 + er;
        sa[i] = i8_row_scale(p)[m < p.M ? m : p.M - 1];
      }
      auto store = [&](int i, int h, bf16x8 v) __attribute__((always_inline)) {
        const int m = m0 + wm * WM + i * 16 + er, n = n0 + wn * WN + 32 * h + 8 * eq;
        if (m < p.M && n < p.N) *reinterpret_cast<bf16x8*>(p.C + (int64_t)m * p.ldc + n) = v;  // N % 8 == 0
      };
      auto rows = [&](auto sig_tag, auto rtb_tag) __attribute__((always_inline)) {
        auto eight = [&](int i, int h, auto finish) __attribute__((always_inline)) {
          const int n = n0 + wn * WN + 32 * h + 8 * eq;
          bf16x8 v;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const f32x4 y = fp4_branch4<EPI, decltype(sig_tag)::value, decltype(rtb_tag)::value>(
                p, i8_value(acc[i][2 * h + c], sa[i], sw[2 * h + c]), bias[2 * h + c], n + 4 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * c + e] = finish(y[e], c, e);
          }
          store(i, h, v);
        };
        if constexpr (RESID) {
          // 32 columns at a time (all at once do not fit the registers)
#pragma unroll
          for (int h = 0; h < TN / 2; ++h) {
            columns(2 * h);
            columns(2 * h + 1);
            bf16x8 res[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
              int m = m0 + wm * WM + i * 16 + er;
              m = m < p.M ? m : p.M - 1;
              const int n = n0 + wn * WN + 32 * h + 8 * eq;
              res[i] = *reinterpret_cast<const bf16x8*>(p.R + (int64_t)m * p.ldr + (n < p.N ? n : 0));
            }
            __builtin_amdgcn_sched_barrier(0);
            wait_vmcnt<0>();  // (for the compiler too: no register waits for a load past here)
#pragma unroll
            for (int i = 0; i < TM; ++i) {
              eight(i, h, [&](float y, int c, int e) {
                return fp4_residual<EPI>(y, res[i][4 * c + e], gate[2 * h + c][e]);
              });
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < TN; ++j) columns(j);
          wait_vmcnt<0>();  // (likewise)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int h = 0; h < TN / 2; ++h) eight(i, h, [](float y, int, int) { return (bf16)y; });
        }
      };
      const bool sig = EPI == LTX_GEMM_EPI_BIAS && n0 + wn * WN + WN > p.sig_from;
      if (p.round_then_bias) {
        if (sig) rows(std::true_type{}, std::true_type{});
        else rows(std::false_type{}, std::true_type{});
      } else {
        if (sig) rows(std::true_type{}, std::false_type{});
        else rows(std::false_type{}, std::false_type{});
      }
    }
    // the next tile's first fragments again: the epilogue had their registers
#pragma unroll
    for (int j = 0; j < TN; ++j) read_share(0, 0, true, j);
  }
  wait_vmcnt<0>();  // (the loads past the last stage: LDS is theirs until then)
}

// 288 rows: where they make one round of the CUs less than 256 (below); the third stage of weights has no room
// beside them.  The residual epilogues spill: at 256 x 256 19 to 21 registers, which stay in the epilogue, at 288
// rows 67 to 69, whose reloads make the stages wait for part of their loads.  The choice does not know the epilogue; 288 rows
// against the best other tiles, x 16384 -> 4096, sets of operands in turn (us): 4608 rows 229 / 249 with bias, 270 / 269
// with residual, 9216 rows 453 / 476 and 517 / 494, 13824 rows 674 / 695 and 774 / 725.
using I8Huge = I8Tile<288, 256, 2, 4, 2, 2>;
using I8Large = I8Tile<256, 256, 2, 4, 2, 3>;
using I8Tall = I8Tile<256, 128, 4, 2, 3, 3>;
using I8Mid = I8Tile<128, 128, 2, 4, 4, 4>;
using I8Small = I8Tile<64, 128, 2, 4, 4, 4>;

// sum of the K ranges' partial products, then the epilogue
__global__ __launch_bounds__(256) void i8_combine_kernel(GemmArgs p, int epi, int splits) {
  const int per_row = p.N / 4;
  const int64_t total = (int64_t)p.M * per_row, plane = (int64_t)p.M * p.N;
  for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < total; idx += (int64_t)gridDim.x * 256) {
    const int m = (int)(idx / per_row), n = (int)(idx % per_row) * 4;
    const int32_t* P = (const int32_t*)p.partial + (int64_t)m * p.N + n;
    i32x4 a = *reinterpret_cast<const i32x4*>(P);
    for (int z = 1; z < splits; ++z) a += *reinterpret_cast<const i32x4*>(P + z * plane);
    i8_store4(p, epi, a, m, n);
  }
}

template <int EPI>
static void i8_launch_tiles(GemmArgs p, const I8Plan& pl, hipStream_t s) {
  p.tiles_m = (p.M + pl.bm - 1) / pl.bm;
  p.tiles_n = (p.N + pl.bn - 1) / pl.bn;
  const int all = p.tiles_m * p.tiles_n * pl.splits, blocks = all < 256 ? all : 256;
  auto go = [&](auto t) {
    using T = decltype(t);
    gemm_i8_kernel<T, EPI><<<blocks, T::THREADS, 0, s>>>(p, pl.k_split);
  };
  if (pl.bm == 256 && pl.bn == 256) go(I8Large{});
  else if (pl.bm == 288) go(I8Huge{});
  else if (pl.bm == 256) go(I8Tall{});
  else if (pl.bm == 128) go(I8Mid{});
  else go(I8Small{});
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
  if (M == 0 || N == 0 || K == 0 || M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2) return 0;
  const I8Plan pl = i8_plan(M, N, K);
  return pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0;
}

extern "C" int ltx_gemm_i8_bf16(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* Wq, int64_t ldw,
                                const float* w_scale, const float* bias, void* C, int64_t ldc, int64_t M, int64_t N,
                                int64_t K, int epilogue, const void* residual, int64_t ldr, const float* gate,
                                int64_t sigmoid_from, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = i8_check(A, lda, a_scale, Wq, ldw, w_scale, bias, C, ldc, M, N, K, epilogue, residual, ldr, gate);
  if (st != LTX_OK) return st;
  if (M == 0 || N == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  const I8Plan pl = i8_plan(M, N, K);
  const int64_t need = pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return LTX_ERR_INVALID_ARG;
  if (need > 0 && ((uintptr_t)workspace & 15u)) return LTX_ERR_ALIGNMENT;
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
  p.N = (int)N;
  p.K = (int)K;
  hipStream_t s = (hipStream_t)stream;
  const int epi = epilogue & 0xff;
  // rows [r0, r1) by a plan's kernel in one pass over K
  auto run = [&](int64_t r0, int64_t r1, int bm, int bn) {
    const I8Plan whole = {0, 0, bm, bn, 1, (int)((K + 127) / 128 * 128)};
    // Rows that one launch of the tile kernel takes: its operands' byte offsets have 31 bits.
    // None where a tile's rows, or the weights, are past them: then the few-row kernel, whose
    // addresses have 64 bits
    const int64_t lim = ((int64_t)1 << 31) - 1;
    int64_t piece = r1 - r0;
    if (bn > 0) {
      if (N > lim / ldw) piece = 0;
      else if (lim / lda < piece) piece = lim / lda / 256 * 256;
      if (piece == 0) {
        piece = r1 - r0;
        bm = 64;
        bn = -2;
      }
    }
    if (bn < 0) {  // (a launch has fewer than 2^32 threads)
      const int64_t most = (((int64_t)1 << 23) - 1) / ((N - 16 * bn - 1) / (-16 * bn)) * bm;
      piece = most < piece ? most : piece;
    }
    for (; r0 < r1; r0 += piece) {
      GemmArgs part = p;
      part.A = (const bf16*)(A + r0 * lda);
      part.ascale = (const uint8_t*)(a_scale + r0);
      part.C = p.C + r0 * ldc;
      if (p.R) part.R = p.R + r0 * ldr;
      part.M = (int)(r1 - r0 < piece ? r1 - r0 : piece);
      if (bn > 0) fp4_epilogue(epi, [&](auto e) { i8_launch_tiles<decltype(e)::value>(part, whole, s); });
      else if (bm == 16 && bn == -1) i8_launch_rows<1, 1>(part, epi, s);
      else if (bm == 16) i8_launch_rows<1, 2>(part, epi, s);
      else if (bm == 32 && bn == -1) i8_launch_rows<2, 1>(part, epi, s);
      else if (bm == 32) i8_launch_rows<2, 2>(part, epi, s);
      else if (bn == -1) i8_launch_rows<4, 1>(part, epi, s);
      else i8_launch_rows<4, 2>(part, epi, s);
      const int e = ltx_launch_status();
      if (e != LTX_OK) return e;
    }
    return LTX_OK;
  };
  const int64_t lim = ((int64_t)1 << 31) - 1;
  if (pl.splits > 1 && N <= lim / ldw && M <= lim / lda) {
    p.M = (int)M;
    p.partial = (float*)workspace;
    i8_launch_tiles<kEpiPartial>(p, pl, s);
    const int e = ltx_launch_status();
    if (e != LTX_OK) return e;
    const int64_t total = M * (N / 4);
    i8_combine_kernel<<<(int)(total + 255 < 4096 * 256 ? (total + 255) / 256 : 4096), 256, 0, s>>>(p, epi, pl.splits);
    return ltx_launch_status();
  }
  if (pl.head > 0) {
    const int e = run(0, pl.head, 256, pl.head_bn);
    if (e != LTX_OK) return e;
  }
  return run(pl.head, M, pl.bm, pl.bn);
}
