// Weight formats of the quantised projections: encoders and bf16 decoders.
//
// MXFP8 (OCP Microscaling v1.0, element E4M3, block 32 along K, scale E8M0):
//   the storage of LTX_2_MLX's `mx.quantize(W, 32, 8, mode="mxfp8")`
//   (loader/transformer_cache.py:1255-1267): codes (N, K) uint8 -- the same
//   bytes as the reference's (N, K/4) uint32 words -- and scales (N, K/32).
//   The reference's encoder is MLX-internal; this one follows the OCP rule:
//     X = floor(log2(max|w|)) - 8 (8 = E4M3 emax), clamped to [-127, 127],
//     scale byte = X + 127, code = E4M3(w / 2^X) rounded to nearest-even and
//     saturated to +-448.  An all-zero block gets X = -127.
// FP8 checkpoints (loader/transformer_cache.py:658-708): E4M3 codes with an
//   optional per-tensor fp32 weight_scale, dequantised at load time as
//   from_fp8(w) * scale in fp32 and rounded once to the cache dtype.
// int8 W8A16 (per output channel, symmetric):
//     s[n] = max_k |w[n,k]| / 127 (fp32), q = clamp(rint(w / s), -127, 127);
//     a zero row has s = 0 and q = 0.  Decode: w' = bf16(fp32(q) * s).
//   Activation rows (int8 x int8 products) by the same rule; a row with a NaN or an
//   infinity has s = NaN and q = 0.
// MXFP4 (OCP Microscaling v1.0, element E2M1, block 32 along K, scale E8M0):
//     X = floor(log2(max|v|)) - 2 (2 = E2M1 emax), clamped to [-127, 127],
//     scale byte = X + 127, code = E2M1(v / 2^X) rounded to nearest-even and
//     saturated to +-6, the sign kept on zeros.  An all-zero block gets X = -127.
//     E2M1 has no NaN: a block with a NaN or an infinity gets scale byte 255
//     (NaN) and codes 0, and decodes to NaN throughout.
//     Codes two to a byte, the even k low; scale words as gemm_fp4.h lays out.
#include <type_traits>

#include "gemm_fp4.h"

namespace ltx {

// Rows of 32-element blocks: one wave per 512-element chunk of a row, lane l
// holding elements 8l..8l+7 (one 16-byte load), lanes 4b..4b+3 forming block
// b; the block maximum takes two lane exchanges, the codes leave as one
// 8-byte store per lane (512 contiguous bytes per wave) and lane 4b writes the
// block's scale byte.  Chunks past K (K % 512 != 0) leave their lanes idle.
// Used for weights (at load) and for activation rows (the opt-in MX path).
__global__ __launch_bounds__(256) void mxfp8_quantize_kernel(const bf16* __restrict__ W, int64_t ldw, int64_t N,
                                                             int64_t K, uint8_t* __restrict__ q, int64_t ldq,
                                                             uint8_t* __restrict__ sc, int64_t lds) {
  const int lane = threadIdx.x & 63;
  const int64_t chunks = (K + 511) / 512;
  const int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (task >= N * chunks) return;  // whole waves: the exchanges below see all 64 lanes
  const int64_t n = task / chunks;
  const int64_t col = (task % chunks) * 512 + lane * 8;
  const bool in = col < K;  // K % 32 == 0: a block's four lanes agree
  float v[8];
  float amax = 0.0f;
  if (in) {
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(W + n * ldw + col);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = (float)x[e];
      amax = fmaxf(amax, fabsf(v[e]));
    }
  }
  amax = fmaxf(amax, __shfl_xor(amax, 1, 64));
  amax = fmaxf(amax, __shfl_xor(amax, 2, 64));
  if (!in) return;
  const int X = mxfp8_block_exponent(amax);
  if ((lane & 3) == 0) sc[n * lds + col / 32] = (uint8_t)(X + 127);
  const float s = ldexpf(1.0f, X), lim = 448.0f * s;
  const uint32_t w0 = e4m3x4_ocp(v[0], v[1], v[2], v[3], s, lim);
  const uint32_t w1 = e4m3x4_ocp(v[4], v[5], v[6], v[7], s, lim);
  *reinterpret_cast<u32x2*>(q + n * ldq + col) = u32x2{w0, w1};
}

__global__ void mxfp8_dequantize_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                        const uint8_t* __restrict__ sc, int64_t lds, int64_t N,
                                        int64_t K, bf16* __restrict__ out, int64_t ldo) {
  const int64_t per_row = K / 8;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= N * per_row) return;
  const int64_t n = idx / per_row, c = idx % per_row;
  const u32x2 raw = *reinterpret_cast<const u32x2*>(q + n * ldq + c * 8);
  const uint32_t s = sc[n * lds + (c * 8) / 32];
  const float scale = s == 0xffu ? __uint_as_float(0x7fc00000u)
                                 : (s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23));
  uint32_t o[4];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    o[2 * d] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d], scale, false));
    o[2 * d + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d], scale, true));
  }
  *reinterpret_cast<u32x4*>(out + n * ldo + c * 8) = u32x4{o[0], o[1], o[2], o[3]};
}

// ---- MXFP4 -------------------------------------------------------------------
// Row loads of eight elements as fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (std::is_same_v<T, float>) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
    typedef T t8 __attribute__((ext_vector_type(8)));
    const t8 x = *reinterpret_cast<const t8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
  }
}

// A workgroup encodes 16 rows x 512 k, a wave a row at a time (lane l elements
// 8 l .. 8 l + 7, lanes 4 b .. 4 b + 3 forming block b).  The scale words of a
// k range are contiguous over rows, so they meet in LDS and leave as 64-byte
// pieces.  Bound by HBM: 14640 x 4096 bf16 25 us (6.0 TB/s), the decoder 24 (6.6);
// 68 x 2048 4.1 and 2.6, a launch.
constexpr int kQ4Rows = 16;
constexpr int64_t kQ4Blocks = (1 << 24) - 1;  // of 256 threads: a launch has fewer than 2^32
constexpr int64_t kI8Rows = (1 << 24) - 1;    // (up to a workgroup of 256 threads each)
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                             int64_t K, uint8_t* __restrict__ q, int64_t ldq,
                                                             uint32_t* __restrict__ sc, int64_t lds) {
  __shared__ uint8_t scale[4][kQ4Rows][4];  // [128 k][row][block]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t chunks = (K + 511) / 512;
  const int64_t r0 = (int64_t)blockIdx.x / chunks * kQ4Rows, k0 = (int64_t)blockIdx.x % chunks * 512;
  const int64_t col = k0 + lane * 8;
  const bool in = col < K;  // K % 32 == 0: a block's four lanes agree
#pragma unroll
  for (int i = 0; i < kQ4Rows / 4; ++i) {
    const int lr = i * 4 + wave;
    const int64_t r = r0 + lr;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (in && r < rows) load8(x + r * ldx + col, v);
    // the block's largest magnitude, as bits: those of a NaN or an infinity
    // are above every finite one's
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = __float_as_uint(v[e]) & 0x7fffffffu;
      top = b > top ? b : top;
    }
    const uint32_t t1 = __shfl_xor(top, 1, 64);
    top = t1 > top ? t1 : top;
    const uint32_t t2 = __shfl_xor(top, 2, 64);
    top = t2 > top ? t2 : top;
    const bool bad = top >= 0x7f800000u;
    // floor(log2): the exponent field; below 2^-126 (and 0) X is -127 anyway
    int X = (int)(top >> 23) - 127 - 2;
    X = X < -127 ? -127 : X;
    if ((lane & 3) == 0) scale[lane >> 4][lr][(lane >> 2) & 3] = !in ? 0 : (bad ? 255 : (uint8_t)(X + 127));
    if (!in || r >= rows) continue;
    const float s = ldexpf(1.0f, X), lim = 6.0f * s;  // lim: X <= 125
    uint32_t w = 0;
    auto cl = [lim](float f) { return fabsf(f) >= lim ? __builtin_copysignf(lim, f) : f; };
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, cl(v[0]), cl(v[1]), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, cl(v[2]), cl(v[3]), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, cl(v[4]), cl(v[5]), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, cl(v[6]), cl(v[7]), s, 3);
    *reinterpret_cast<uint32_t*>(q + r * ldq + col / 2) = bad ? 0u : w;
  }
  __syncthreads();
  const int64_t words = (K + 127) / 128;
  const int t = threadIdx.x;
  if (t < 4 * kQ4Rows) {
    const int64_t w = k0 / 128 + t / kQ4Rows, r = r0 + t % kQ4Rows;
    if (w < words && r < rows)
      sc[w * lds + r] = *reinterpret_cast<const uint32_t*>(scale[t / kQ4Rows][t % kQ4Rows]);
  }
}

// Eight codes per lane (4 bytes in, 16 out).
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                               const uint32_t* __restrict__ sc, int64_t lds,
                                                               int64_t rows, int64_t K, bf16* __restrict__ out,
                                                               int64_t ldo) {
  const int64_t per_row = K / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= rows * per_row) return;
  const int64_t r = idx / per_row, c = idx % per_row * 8;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(q + r * ldq + c / 2);
  const uint32_t e = (sc[c / 128 * lds + r] >> (c / 32 % 4 * 8)) & 0xffu;
  *reinterpret_cast<bf16x8*>(out + r * ldo + c) = fp4x8_bf16(w, e8m0_to_f32(e));
}

// One wave per row.
__global__ __launch_bounds__(256) void w8_quantize_kernel(const bf16* __restrict__ W, int64_t ldw,
                                                          int64_t N, int64_t K,
                                                          int8_t* __restrict__ q, int64_t ldq,
                                                          float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  const bf16* row = W + n * ldw;
  float amax = 0.0f;
  for (int64_t k = lane * 8; k < K; k += 512) {
    bf16x8 x = *reinterpret_cast<const bf16x8*>(row + k);
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf((float)x[e]));
  }
  amax = wave_max(amax);
  const float s = __fdiv_rn(amax, 127.0f);
  if (lane == 0) scale[n] = s;
  int8_t* qrow = q + n * ldq;
  for (int64_t k = lane * 8; k < K; k += 512) {
    bf16x8 x = *reinterpret_cast<const bf16x8*>(row + k);
    uint32_t w0 = 0, w1 = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float r = s > 0.0f ? rintf(__fdiv_rn((float)x[e], s)) : 0.0f;
      r = fminf(fmaxf(r, -127.0f), 127.0f);
      const uint32_t b = (uint32_t)((int32_t)r & 0xff);
      if (e < 4) w0 |= b << (8 * e); else w1 |= b << (8 * (e - 4));
    }
    *reinterpret_cast<u32x2*>(qrow + k) = u32x2{w0, w1};
  }
}

// C codes (8 or 16) per thread.
template <int C>
__global__ __launch_bounds__(256) void w8_dequantize_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                     const float* __restrict__ scale, int64_t N, int64_t K,
                                     bf16* __restrict__ out, int64_t ldo) {
  const int64_t per_row = K / C;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= N * per_row) return;
  const int64_t n = idx / per_row, c = idx % per_row;
  typedef uint32_t words __attribute__((ext_vector_type(C / 4)));
  const words raw = *reinterpret_cast<const words*>(q + n * ldq + c * C);
  const float s = scale[n];
#pragma unroll
  for (int h = 0; h < C; h += 8) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int32_t v = (int32_t)(int8_t)((raw[(h + e) / 4] >> (8 * (e % 4))) & 0xffu);
      o[e] = (bf16)mul_rn((float)v, s);
    }
    *reinterpret_cast<bf16x8*>(out + n * ldo + c * C + h) = o;
  }
}

// ---- int8 rows -----------------------------------------------------------------
// The code of the rule, rint(fp32(v / s)), of eight values.  v (1 / s) is within 2^-16.4 of the
// fp32 quotient (|v / s| < 128: 2^-17 by the reciprocal's rounding, 2^-18 by the quotient's), so its
// nearest integer is the code's unless it lies that close to a half; then the divisions are made.
// The sum with 1.5 * 2^23 has the integer in its low byte.
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x04000c0cu);
  return lo | hi;
}
__device__ __forceinline__ u32x2 int8_codes8(const float (&v)[8], float s, float inv) {
  constexpr float kMagic = 12582912.0f;
  float t[8];
  bool near = !(s >= 0x1p-126f);  // a subnormal scale's reciprocal may not be finite
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    t[e] = fmaf(v[e], inv, kMagic);
    near |= fabsf(fmaf(v[e], inv, -(t[e] - kMagic))) > 0.5f - 0x1p-15f;
  }
  if (near) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = s > 0.0f ? rintf(__fdiv_rn(v[e], s)) : 0.0f;
      t[e] = fminf(fmaxf(c, -127.0f), 127.0f) + kMagic;  // (a subnormal scale may be off by more than a step)
    }
  }
  return u32x2{low_bytes(t[0], t[1], t[2], t[3]), low_bytes(t[4], t[5], t[6], t[7])};
}

// The magnitude bits of eight elements: those of a NaN or an infinity are above every
// finite one's, in each type's own bits.
template <typename T>
struct Bits8 {
  typedef T t8 __attribute__((ext_vector_type(8), aligned(16)));  // (eight fp32 are two loads of 16 bytes)
  static_assert(alignof(t8) == 16, "rows are at multiples of 16 bytes");
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kInf =
      std::is_same_v<T, float> ? 0x7f800000u : (std::is_same_v<T, bf16> ? 0x7f80u : 0x7c00u);
  t8 x;
  // largest so far of the even and the odd elements (fp32: one value)
  __device__ __forceinline__ uint32_t top(uint32_t t) const {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
        t = b > t ? b : t;
      }
      return t;
    } else {
      const u32x4 w = __builtin_bit_cast(u32x4, x);
      u16x2 m = __builtin_bit_cast(u16x2, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
      return __builtin_bit_cast(uint32_t, m);
    }
  }
  static __device__ __forceinline__ uint32_t one(uint32_t t) {
    if constexpr (std::is_same_v<T, float>) return t;
    else return (t >> 16) > (t & 0xffffu) ? t >> 16 : t & 0xffffu;
  }
  static __device__ __forceinline__ float value(uint32_t bits) {
    if constexpr (std::is_same_v<T, float>) return __uint_as_float(bits);
    else return (float)__builtin_bit_cast(T, (uint16_t)bits);
  }
};

// A row stays in the registers of WPR waves between its maximum and its codes: NC pieces of
// 512 * WPR elements, eight per lane.  Bound by HBM: from memory that no cache holds 14640 x 4096 bf16 37 us (4.8
// TB/s; read twice, with a division per element, 52), fp32 53 (5.7), 3456 x 16384 bf16 37 (4.6), 68 x 2048 3.1, a
// launch; the decoder 14640 x 4096 32 (5.6).  The same rows again, partly in the last-level cache: 29 and 29.
template <typename T, int WPR, int NC>
__global__ __launch_bounds__(256) void int8_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t K,
                                                        int8_t* __restrict__ q, int64_t ldq,
                                                        float* __restrict__ scale) {
  __shared__ uint32_t tops[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = WPR == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
  if (r >= rows) return;  // (WPR 4: no workgroup is past them)
  const int64_t first = (WPR == 1 ? lane : (int)threadIdx.x) * 8;
  Bits8<T> v[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t k = first + c * (512 * WPR);
    // (past K: the last ones)
    v[c].x = *reinterpret_cast<const typename Bits8<T>::t8*>(x + r * ldx + (k < K ? k : K - 8));
  }
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) top = v[c].top(top);
  top = Bits8<T>::one(top);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t t = __shfl_xor(top, off, 64);
    top = t > top ? t : top;
  }
  if constexpr (WPR == 4) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) top = tops[w] > top ? tops[w] : top;
  }
  const bool bad = top >= Bits8<T>::kInf;
  const float s = bad ? 0.0f : __fdiv_rn(Bits8<T>::value(top), 127.0f), inv = __fdiv_rn(1.0f, s);
  if (lane == 0 && (WPR == 1 || wave == 0)) scale[r] = bad ? __uint_as_float(0x7fc00000u) : s;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t k = first + c * (512 * WPR);
    if (k >= K) break;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)v[c].x[e];
    *reinterpret_cast<u32x2*>(q + r * ldq + k) = int8_codes8(f, s, inv);
  }
}

// Rows of more than 16384: a workgroup each, read twice.
template <typename T>
__global__ __launch_bounds__(256) void int8_long_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t K,
                                                             int8_t* __restrict__ q, int64_t ldq,
                                                             float* __restrict__ scale) {
  __shared__ uint32_t tops[4];
  const int64_t r = blockIdx.x;
  uint32_t top = 0;
  for (int64_t k = threadIdx.x * 8; k < K; k += 2048)
    top = Bits8<T>{*reinterpret_cast<const typename Bits8<T>::t8*>(x + r * ldx + k)}.top(top);
  top = Bits8<T>::one(top);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t t = __shfl_xor(top, off, 64);
    top = t > top ? t : top;
  }
  if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) top = tops[w] > top ? tops[w] : top;
  const bool bad = top >= Bits8<T>::kInf;
  const float s = bad ? 0.0f : __fdiv_rn(Bits8<T>::value(top), 127.0f), inv = __fdiv_rn(1.0f, s);
  if (threadIdx.x == 0) scale[r] = bad ? __uint_as_float(0x7fc00000u) : s;
  for (int64_t k = threadIdx.x * 8; k < K; k += 2048) {
    float f[8];
    load8(x + r * ldx + k, f);
    *reinterpret_cast<u32x2*>(q + r * ldq + k) = int8_codes8(f, s, inv);
  }
}

// One wave per row for many short ones, four otherwise: one / four 30000 x 512 fp16 11 / 21 us,
// 14640 x 1024 bf16 12 / 16, x 2048 22 / 23, x 4096 42 / 35, 3456 x 4096 16 / 12.
template <typename T>
static void int8_rows_launch(const T* x, int64_t ldx, int64_t rows, int64_t K, int8_t* q, int64_t ldq, float* scale,
                             hipStream_t s) {
  const bool one = K <= 2048 && rows >= 2048;
  const int64_t pieces = (K + (one ? 511 : 2047)) / (one ? 512 : 2048);
  auto go = [&](auto wpr, auto nc) {
    constexpr int W = decltype(wpr)::value, N = decltype(nc)::value;
    int8_rows_kernel<T, W, N><<<(int)(W == 1 ? (rows + 3) / 4 : rows), 256, 0, s>>>(x, ldx, rows, K, q, ldq, scale);
  };
  auto pick = [&](auto wpr) {
    if (pieces <= 1) go(wpr, std::integral_constant<int, 1>{});
    else if (pieces <= 2) go(wpr, std::integral_constant<int, 2>{});
    else if (decltype(wpr)::value == 1 || pieces <= 4) go(wpr, std::integral_constant<int, 4>{});
    else if constexpr (decltype(wpr)::value == 4) go(wpr, std::integral_constant<int, 8>{});  // (one wave: at most 2048)
  };
  if (pieces > 8) int8_long_rows_kernel<<<(int)rows, 256, 0, s>>>(x, ldx, K, q, ldq, scale);
  else if (one) pick(std::integral_constant<int, 1>{});
  else pick(std::integral_constant<int, 4>{});
}

// E4M3 code -> float, exact: (-1)^s 2^(e-7) (1 + m/8), subnormals (e = 0)
// m 2^-9, 0x7F / 0xFF NaN, no infinities.  The subnormals are formed from
// the integer m rather than an fp32 denormal, so the decode does not depend on
// the denormal mode.
__device__ __forceinline__ float e4m3_to_f32(uint32_t c) {
  const uint32_t e = (c >> 3) & 0xFu, m = c & 7u;
  const float mag = e == 0u ? (float)m * 0.001953125f : __uint_as_float(((e + 120u) << 23) | (m << 20));
  const float v = (c & 0x7Fu) == 0x7Fu ? __builtin_nanf("") : mag;
  return (c & 0x80u) ? -v : v;
}

// FP8 checkpoint dequantisation: out[i] = OUT(e4m3(codes[i]) * scale) with the
// product in fp32 (scale = 1 without a weight_scale: exact).  16 codes per
// thread; the tail (n % 16) one code per thread.
template <typename OUT>
__global__ __launch_bounds__(256) void fp8_dequant_kernel(const uint8_t* __restrict__ codes, int64_t n,
                                                          const float* __restrict__ scale,
                                                          OUT* __restrict__ out) {
  const float sc = scale ? *scale : 1.0f;
  const int64_t groups = n / 16;
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (t < groups) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(codes + t * 16);
    float v[16];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int b = 0; b < 4; ++b) v[4 * q + b] = e4m3_to_f32((w[q] >> (8 * b)) & 0xFFu) * sc;
    if constexpr (std::is_same_v<OUT, bf16>) {
      bf16x8 o0, o1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o0[e] = (bf16)v[e];
        o1[e] = (bf16)v[8 + e];
      }
      *reinterpret_cast<bf16x8*>(out + t * 16) = o0;
      *reinterpret_cast<bf16x8*>(out + t * 16 + 8) = o1;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(out + t * 16 + 4 * e) = f32x4{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
    }
  } else if (t < groups + n % 16) {
    const int64_t i = groups * 16 + (t - groups);
    out[i] = (OUT)(e4m3_to_f32(codes[i]) * sc);
  }
}

}  // namespace ltx

using namespace ltx;

static inline bool a16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

extern "C" int ltx_quantize_mxfp8_bf16(const void* W, int64_t ldw, int64_t N, int64_t K,
                                       uint8_t* q, int64_t ldq, uint8_t* scales, int64_t ld_scale,
                                       void* stream) {
  if (!W || !q || !scales || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (K % 32) return LTX_ERR_UNSUPPORTED;
  if (ldw < K || ldq < K || ld_scale < K / 32) return LTX_ERR_INVALID_ARG;
  if (!a16(W) || !a16(q) || ldw % 8 || ldq % 8) return LTX_ERR_ALIGNMENT;
  const int64_t tasks = N * ((K + 511) / 512);  // one wave each, four per workgroup
  if (tasks == 0) return LTX_OK;
  if ((tasks + 3) / 4 > INT32_MAX) return LTX_ERR_UNSUPPORTED;
  mxfp8_quantize_kernel<<<(int)((tasks + 3) / 4), 256, 0, (hipStream_t)stream>>>(
      (const bf16*)W, ldw, N, K, q, ldq, scales, ld_scale);
  return ltx_launch_status();
}

extern "C" int ltx_dequantize_mxfp8_bf16(const uint8_t* q, int64_t ldq, const uint8_t* scales,
                                         int64_t ld_scale, int64_t N, int64_t K, void* out,
                                         int64_t ldo, void* stream) {
  if (!q || !scales || !out || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (K % 32) return LTX_ERR_UNSUPPORTED;
  if (ldq < K || ldo < K || ld_scale < K / 32) return LTX_ERR_INVALID_ARG;
  if (!a16(out) || (uintptr_t)q % 8 || ldq % 8 || ldo % 8) return LTX_ERR_ALIGNMENT;
  const int64_t total = N * (K / 8);
  if (total == 0) return LTX_OK;
  mxfp8_dequantize_kernel<<<(int)((total + 255) / 256), 256, 0, (hipStream_t)stream>>>(
      q, ldq, scales, ld_scale, N, K, (bf16*)out, ldo);
  return ltx_launch_status();
}

extern "C" int ltx_quantize_w8_bf16(const void* W, int64_t ldw, int64_t N, int64_t K, int8_t* q,
                                    int64_t ldq, float* scale, void* stream) {
  if (!W || !q || !scale || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (K % 8) return LTX_ERR_UNSUPPORTED;
  if (ldw < K || ldq < K) return LTX_ERR_INVALID_ARG;
  if (!a16(W) || (uintptr_t)q % 8 || ldw % 8 || ldq % 8) return LTX_ERR_ALIGNMENT;
  if (N == 0) return LTX_OK;
  w8_quantize_kernel<<<(int)((N + 3) / 4), 256, 0, (hipStream_t)stream>>>((const bf16*)W, ldw, N,
                                                                        K, q, ldq, scale);
  return ltx_launch_status();
}

extern "C" int ltx_dequantize_w8_bf16(const int8_t* q, int64_t ldq, const float* scale, int64_t N,
                                      int64_t K, void* out, int64_t ldo, void* stream) {
  if (!q || !scale || !out || N < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (K % 8) return LTX_ERR_UNSUPPORTED;
  if (ldq < K || ldo < K) return LTX_ERR_INVALID_ARG;
  if (!a16(out) || (uintptr_t)q % 8 || ldq % 8 || ldo % 8) return LTX_ERR_ALIGNMENT;
  if (N == 0 || K == 0) return LTX_OK;
  if (K / 8 > kQ4Blocks * 256 / N) return LTX_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  if (K % 16 == 0 && ldq % 16 == 0 && (uintptr_t)q % 16 == 0)
    w8_dequantize_kernel<16><<<(int)((N * (K / 16) + 255) / 256), 256, 0, st>>>(q, ldq, scale, N, K, (bf16*)out, ldo);
  else
    w8_dequantize_kernel<8><<<(int)((N * (K / 8) + 255) / 256), 256, 0, st>>>(q, ldq, scale, N, K, (bf16*)out, ldo);
  return ltx_launch_status();
}

extern "C" int ltx_quantize_int8(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t K, int8_t* q,
                                 int64_t ldq, float* scale, void* stream) {
  if (!x || !q || !scale || rows < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > 2 || K % 16) return LTX_ERR_UNSUPPORTED;
  if (ldx < K || ldq < K) return LTX_ERR_INVALID_ARG;
  if (!a16(x) || !a16(q) || (uintptr_t)scale % 4 || ldx % (dtype == 2 ? 4 : 8) || ldq % 16) return LTX_ERR_ALIGNMENT;
  if (rows > kI8Rows) return LTX_ERR_UNSUPPORTED;
  if (rows == 0) return LTX_OK;
  if (K == 0) return LTX_ERR_UNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == 0) int8_rows_launch((const bf16*)x, ldx, rows, K, q, ldq, scale, s);
  else if (dtype == 1) int8_rows_launch((const _Float16*)x, ldx, rows, K, q, ldq, scale, s);
  else int8_rows_launch((const float*)x, ldx, rows, K, q, ldq, scale, s);
  return ltx_launch_status();
}

extern "C" int ltx_quantize_mxfp4(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t K, uint8_t* q,
                                  int64_t ldq, uint32_t* scales, int64_t ld_scale, void* stream) {
  if (!x || !q || !scales || rows < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > 2 || K % 32) return LTX_ERR_UNSUPPORTED;
  if (ldx < K || ldq < K / 2 || ld_scale < rows) return LTX_ERR_INVALID_ARG;
  if (!a16(x) || !a16(q) || !a16(scales) || ldx % (dtype == 2 ? 4 : 8) || ldq % 16 || ld_scale % 4)
    return LTX_ERR_ALIGNMENT;
  if (rows == 0 || K == 0) return LTX_OK;
  const int64_t chunks = (K + 511) / 512, groups = (rows + kQ4Rows - 1) / kQ4Rows;
  if (chunks > kQ4Blocks / groups) return LTX_ERR_UNSUPPORTED;
  const int blocks = (int)(chunks * groups);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == 0)
    mxfp4_quantize_kernel<<<blocks, 256, 0, s>>>((const bf16*)x, ldx, rows, K, q, ldq, scales, ld_scale);
  else if (dtype == 1)
    mxfp4_quantize_kernel<<<blocks, 256, 0, s>>>((const _Float16*)x, ldx, rows, K, q, ldq, scales, ld_scale);
  else
    mxfp4_quantize_kernel<<<blocks, 256, 0, s>>>((const float*)x, ldx, rows, K, q, ldq, scales, ld_scale);
  return ltx_launch_status();
}

extern "C" int ltx_dequantize_mxfp4_bf16(const uint8_t* q, int64_t ldq, const uint32_t* scales, int64_t ld_scale,
                                         int64_t rows, int64_t K, void* out, int64_t ldo, void* stream) {
  if (!q || !scales || !out || rows < 0 || K < 0) return LTX_ERR_INVALID_ARG;
  if (K % 32) return LTX_ERR_UNSUPPORTED;
  if (ldq < K / 2 || ldo < K || ld_scale < rows) return LTX_ERR_INVALID_ARG;
  if (!a16(out) || !a16(q) || !a16(scales) || ldq % 16 || ldo % 8 || ld_scale % 4) return LTX_ERR_ALIGNMENT;
  if (rows == 0 || K == 0) return LTX_OK;
  if (K / 8 > kQ4Blocks * 256 / rows) return LTX_ERR_UNSUPPORTED;
  const int64_t total = rows * (K / 8);
  mxfp4_dequantize_kernel<<<(int)((total + 255) / 256), 256, 0, (hipStream_t)stream>>>(
      q, ldq, scales, ld_scale, rows, K, (bf16*)out, ldo);
  return ltx_launch_status();
}

// FP8 E4M3 checkpoint tensor -> bf16 (out_dtype 0) or fp32 (out_dtype 1).
extern "C" int ltx_dequantize_fp8_e4m3(const uint8_t* codes, int64_t n, const float* scale, void* out,
                                       int out_dtype, void* stream) {
  if (!codes || !out || n < 0) return LTX_ERR_INVALID_ARG;
  if (out_dtype != 0 && out_dtype != 1) return LTX_ERR_UNSUPPORTED;
  if (!a16(codes) || !a16(out) || ((uintptr_t)scale & 3u)) return LTX_ERR_ALIGNMENT;
  const int64_t threads = n / 16 + n % 16;
  if (threads == 0) return LTX_OK;
  if ((threads + 255) / 256 > INT32_MAX) return LTX_ERR_UNSUPPORTED;
  const int blocks = (int)((threads + 255) / 256);
  if (out_dtype == 0)
    fp8_dequant_kernel<bf16><<<blocks, 256, 0, (hipStream_t)stream>>>(codes, n, scale, (bf16*)out);
  else
    fp8_dequant_kernel<float><<<blocks, 256, 0, (hipStream_t)stream>>>(codes, n, scale, (float*)out);
  return ltx_launch_status();
}
