// Rotary positions of queries and keys:
//
//   a' = f (a cos t - b sin t),  b' = f (b cos t + a sin t),  t = position * inv_freq[i]
//
// for the pairs (a, b) of the first `rotary` channels of every head: channels
// (i, i + rotary / 2) or (2 i, 2 i + 1); the other channels are copied.  With
// the angle negated it is the transposed map, which takes the gradient of the
// outputs to that of the inputs (f included).
//
// Bound by memory: every element is read and written once.  An angle is needed
// by all heads of a token, so a workgroup takes a few tokens, computes their
// cosines and sines once into LDS (one pair per thread) and then streams the
// heads.  The angle is formed and reduced to a fraction of a turn in fp64: at
// position 10^6 an fp32 angle has lost 0.06 of a radian.
#include <type_traits>

#include "ltx_common.h"

namespace ltx {

constexpr int kRotThreads = 256, kRotTokens = 4, kRotMaxDim = 512;

struct RotArgs {
  ltx_rotary_rows side[2];
  int64_t batch, tokens;
  int head_dim, rotary;
  const void* positions;
  int64_t pos_batch;
  int pos_type;
  const double* inv_freq;
  float factor;
  int transpose;
  int per_block;  // tokens of a workgroup
};

__device__ __forceinline__ double rot_position(const RotArgs& p, int64_t i) {
  switch (p.pos_type) {
    case 0: return (double)((const int32_t*)p.positions)[i];
    case 1: return (double)((const int64_t*)p.positions)[i];
    case 2: return (double)((const float*)p.positions)[i];
    default: return ((const double*)p.positions)[i];
  }
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
  T v[VEC];
};

// VEC elements per load and store: the largest power of two up to 16 bytes
// that divides the extents, strides and addresses.
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs p) {
  using V = RotVec<T, VEC>;
  __shared__ __attribute__((aligned(16))) float cs[kRotTokens][kRotMaxDim / 2];
  __shared__ __attribute__((aligned(16))) float sn[kRotTokens][kRotMaxDim / 2];
  const int pairs = p.rotary / 2;
  const int64_t all = p.batch * p.tokens;
  const int64_t first = (int64_t)blockIdx.x * p.per_block;
  const int count = (int)(all - first < p.per_block ? all - first : p.per_block);
  for (int i = threadIdx.x; i < count * pairs; i += kRotThreads) {
    const int t = i / pairs, j = i % pairs;
    const int64_t row = first + t;
    const double pos = rot_position(p, row / p.tokens * p.pos_batch + row % p.tokens);
    double turns = pos * p.inv_freq[j] * 0.15915494309189533576888;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    cs[t][j] = c * p.factor;
    sn[t][j] = (p.transpose ? -s : s) * p.factor;
  }
  __syncthreads();

  // items of a head: vectors of pairs (half layout: two loads), then vectors of
  // the channels that are only copied.  A thread keeps its item over the heads.
  constexpr bool NEIGHBOURS = INTERLEAVED && VEC > 1;  // a vector holds whole pairs
  const int rot_items = NEIGHBOURS ? p.rotary / VEC : pairs / VEC;
  const int all_items = rot_items + (p.head_dim - p.rotary) / VEC;
  const int lanes = all_items < kRotThreads ? all_items : kRotThreads;
  const int step = kRotThreads / lanes;
  const int i0 = threadIdx.x % lanes, h0 = threadIdx.x / lanes;
  if (h0 >= step) return;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const ltx_rotary_rows& r = p.side[side];
    if (r.heads == 0) continue;
    const bool in_place = r.x == r.out && r.x_batch == r.out_batch && r.x_token == r.out_token && r.x_head == r.out_head;
    const int items = in_place ? rot_items : all_items;
    for (int t = 0; t < count; ++t) {
      const int64_t row = first + t, b = row / p.tokens, tok = row % p.tokens;
      const T* x = (const T*)r.x + b * r.x_batch + tok * r.x_token;
      T* out = (T*)r.out + b * r.out_batch + tok * r.out_token;
      for (int i = i0; i < items; i += lanes) {
        if (i >= rot_items) {
          const int c = p.rotary + (i - rot_items) * VEC;
#pragma unroll 2
          for (int64_t h = h0; h < r.heads; h += step)
            *reinterpret_cast<V*>(out + h * r.out_head + c) = *reinterpret_cast<const V*>(x + h * r.x_head + c);
          continue;
        }
        if constexpr (NEIGHBOURS) {
          const int c = i * VEC;
          float ca[VEC / 2], sa[VEC / 2];
#pragma unroll
          for (int e = 0; e < VEC / 2; ++e) {
            ca[e] = cs[t][c / 2 + e];
            sa[e] = sn[t][c / 2 + e];
          }
#pragma unroll 2
          for (int64_t h = h0; h < r.heads; h += step) {
            V v = *reinterpret_cast<const V*>(x + h * r.x_head + c);
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
              const float u = (float)v.v[2 * e], w = (float)v.v[2 * e + 1];
              v.v[2 * e] = (T)(u * ca[e] - w * sa[e]);
              v.v[2 * e + 1] = (T)(w * ca[e] + u * sa[e]);
            }
            *reinterpret_cast<V*>(out + h * r.out_head + c) = v;
          }
        } else {
          const int c = i * VEC, c0 = INTERLEAVED ? 2 * c : c, c1 = INTERLEAVED ? 2 * c + 1 : c + pairs;
          float ca[VEC], sa[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            ca[e] = cs[t][c + e];
            sa[e] = sn[t][c + e];
          }
#pragma unroll 2
          for (int64_t h = h0; h < r.heads; h += step) {
            const V u = *reinterpret_cast<const V*>(x + h * r.x_head + c0);
            const V w = *reinterpret_cast<const V*>(x + h * r.x_head + c1);
            V o, n;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float a = (float)u.v[e], d = (float)w.v[e];
              o.v[e] = (T)(a * ca[e] - d * sa[e]);
              n.v[e] = (T)(d * ca[e] + a * sa[e]);
            }
            *reinterpret_cast<V*>(out + h * r.out_head + c0) = o;
            *reinterpret_cast<V*>(out + h * r.out_head + c1) = n;
          }
        }
      }
    }
  }
}

template <typename T, int VEC>
static void rotary_launch(const RotArgs& p, bool interleaved, int blocks, hipStream_t s) {
  if (interleaved) rotary_kernel<T, VEC, true><<<blocks, kRotThreads, 0, s>>>(p);
  else rotary_kernel<T, VEC, false><<<blocks, kRotThreads, 0, s>>>(p);
}
template <typename T>
static void rotary_launch_vec(const RotArgs& p, int vec, bool interleaved, int blocks, hipStream_t s) {
  if (vec == 8) {
    if constexpr (sizeof(T) == 2) rotary_launch<T, 8>(p, interleaved, blocks, s);
  } else if (vec == 4) {
    rotary_launch<T, 4>(p, interleaved, blocks, s);
  } else if (vec == 2) {
    rotary_launch<T, 2>(p, interleaved, blocks, s);
  } else {
    rotary_launch<T, 1>(p, interleaved, blocks, s);
  }
}

}  // namespace ltx

using namespace ltx;

extern "C" int ltx_rotary(const ltx_rotary_rows* q, const ltx_rotary_rows* k, int dtype, int64_t batch,
                          int64_t tokens, int64_t head_dim, int64_t rotary_dim, const void* positions, int pos_type,
                          int64_t pos_batch, const double* inv_freq, double factor, int flags, void* stream) {
  if (!q || batch < 0 || tokens < 0 || head_dim < 1 || rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
    return LTX_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > 2 || pos_type < 0 || pos_type > 3) return LTX_ERR_UNSUPPORTED;
  if (flags & ~(LTX_ROTARY_INTERLEAVED | LTX_ROTARY_TRANSPOSE)) return LTX_ERR_INVALID_ARG;
  if (head_dim > kRotMaxDim) return LTX_ERR_UNSUPPORTED;
  if (!positions || !inv_freq || pos_batch < 0) return LTX_ERR_INVALID_ARG;
  const uintptr_t pos_size = pos_type == 1 || pos_type == 3 ? 8 : 4, size = dtype == 2 ? 4 : 2;
  if ((uintptr_t)positions % pos_size || (uintptr_t)inv_freq % 8) return LTX_ERR_ALIGNMENT;
  RotArgs p = {};
  p.side[0] = *q;
  if (k) p.side[1] = *k;
  const bool interleaved = (flags & LTX_ROTARY_INTERLEAVED) != 0;
  // the widest vector that divides every extent, stride and address
  int64_t bits = interleaved ? rotary_dim : rotary_dim / 2;
  bits |= head_dim - rotary_dim;
  for (const ltx_rotary_rows& r : p.side) {
    if (r.heads < 0 || r.heads > INT32_MAX) return LTX_ERR_INVALID_ARG;
    if (r.heads == 0) continue;
    if (!r.x || !r.out) return LTX_ERR_INVALID_ARG;
    if ((uintptr_t)r.x % size || (uintptr_t)r.out % size) return LTX_ERR_ALIGNMENT;
    bits |= (int64_t)((uintptr_t)r.x / size | (uintptr_t)r.out / size);
    // the stride of an axis of one entry is never used
    if (batch > 1) bits |= r.x_batch | r.out_batch;
    if (tokens > 1) bits |= r.x_token | r.out_token;
    if (r.heads > 1) bits |= r.x_head | r.out_head;
  }
  if (p.side[0].heads == 0 && p.side[1].heads == 0) return LTX_OK;
  if (batch == 0 || tokens == 0) return LTX_OK;
  if (tokens > INT64_MAX / 2 / batch) return LTX_ERR_UNSUPPORTED;
  int vec = (int)(16 / size);
  while (vec > 1 && (bits & (vec - 1))) vec >>= 1;
  p.batch = batch;
  p.tokens = tokens;
  p.head_dim = (int)head_dim;
  p.rotary = (int)rotary_dim;
  p.positions = positions;
  p.pos_type = pos_type;
  p.pos_batch = pos_batch;
  p.inv_freq = inv_freq;
  p.factor = (float)factor;
  p.transpose = (flags & LTX_ROTARY_TRANSPOSE) != 0;
  const int64_t all = batch * tokens;
  p.per_block = all >= 4096 ? kRotTokens : (all >= 2048 ? 2 : 1);
  const int64_t blocks = (all + p.per_block - 1) / p.per_block;
  if (blocks > INT32_MAX) return LTX_ERR_UNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == 0) rotary_launch_vec<bf16>(p, vec, interleaved, (int)blocks, s);
  else if (dtype == 1) rotary_launch_vec<_Float16>(p, vec, interleaved, (int)blocks, s);
  else rotary_launch_vec<float>(p, vec, interleaved, (int)blocks, s);
  return ltx_launch_status();
}
