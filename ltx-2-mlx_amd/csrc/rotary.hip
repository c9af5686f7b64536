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
// Measured: 3456 tokens x 64 heads of 128 bf16 22 us in either layout (5.2 TB/s), 14640 x 40 heads
// of 128 bf16 56-59 (5.1-5.3 TB/s), 14639 x 40 heads of 64 fp32 56 (5.3 TB/s), 14639 x
// 9 heads of 64 bf16 11 (3.1 TB/s), one token 4.
#include <type_traits>

#include "ltx_common.h"

namespace ltx {

constexpr int kRotThreads = 256, kRotTokens = 16, kRotMaxDim = 512;
constexpr int kRotTable = 2048;  // cosines (and sines) of a workgroup
constexpr int64_t kRotBlocks = (1 << 24) - 1;  // a launch has fewer than 2^32 threads
constexpr int64_t kRotHeads = 1 << 30;         // an item's head index runs up to kRotThreads + 1 past them

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
  int table;      // table entries of a token: its pairs, up to a multiple of 4
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
//
// An item is two vectors of a head: the two halves of VEC pairs, or two vectors
// of neighbouring pairs, or two that are only copied (the second may repeat the
// first at an odd end), the second half a range after the first, so that the
// lanes of a load lie side by side.  The items of the workgroup's tokens and heads form
// one list that the threads go through, kBatch items each at a time: as many
// loads in flight whatever the head layout (a loop over heads with a fixed item
// per thread left them idle where tokens have few heads: 14639 tokens x 40 heads
// of 64 fp32 99 us).
constexpr int kRotBatch = 4;
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs p) {
  using V = RotVec<T, VEC>;
  constexpr bool NEIGHBOURS = INTERLEAVED && VEC > 1;  // a vector holds whole pairs
  __shared__ __attribute__((aligned(16))) float cs[kRotTable], sn[kRotTable];
  __shared__ int64_t row_x[2][kRotTokens], row_out[2][kRotTokens];
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
    cs[t * p.table + j] = c * p.factor;
    sn[t * p.table + j] = (p.transpose ? -s : s) * p.factor;
  }
  if (threadIdx.x < 2 * kRotTokens) {
    const int side = threadIdx.x / kRotTokens, t = threadIdx.x % kRotTokens;
    const ltx_rotary_rows& r = p.side[side];
    const int64_t row = first + t, b = row / p.tokens, tok = row % p.tokens;
    row_x[side][t] = b * r.x_batch + tok * r.x_token;
    row_out[side][t] = b * r.out_batch + tok * r.out_token;
  }
  __syncthreads();

  const int rot_vecs = NEIGHBOURS ? p.rotary / VEC : 2 * (pairs / VEC), copy_vecs = (p.head_dim - p.rotary) / VEC;
  const int rot_items = (rot_vecs + 1) / 2, copy_items = (copy_vecs + 1) / 2, all_items = rot_items + copy_items;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const ltx_rotary_rows& r = p.side[side];
    const int heads = (int)r.heads;
    if (heads == 0) continue;
    const bool in_place = r.x == r.out && r.x_batch == r.out_batch && r.x_token == r.out_token && r.x_head == r.out_head;
    const int items = in_place ? rot_items : all_items;
    const T* x = (const T*)r.x;
    T* out = (T*)r.out;
    // (token, head, item) of this thread, and what kRotThreads items add to it
    int i = threadIdx.x % items, h = threadIdx.x / items % heads, t = threadIdx.x / items / heads;
    const int di = kRotThreads % items, dh = kRotThreads / items % heads, dt = kRotThreads / items / heads;
    while (t < count) {
      V a[kRotBatch], b[kRotBatch];
      T* dst[kRotBatch];
      int c0[kRotBatch], c1[kRotBatch], at[kRotBatch];
#pragma unroll
      for (int e = 0; e < kRotBatch; ++e) {
        at[e] = t;
        if (t < count) {
          const int j = i - rot_items;
          if (j >= 0) {
            c0[e] = p.rotary + j * VEC;
            c1[e] = p.rotary + (j + copy_items < copy_vecs ? j + copy_items : j) * VEC;
          } else if (NEIGHBOURS) {
            c0[e] = i * VEC;
            c1[e] = (i + rot_items < rot_vecs ? i + rot_items : i) * VEC;
          } else {
            c0[e] = INTERLEAVED ? 2 * i : i * VEC;
            c1[e] = INTERLEAVED ? 2 * i + 1 : i * VEC + pairs;
          }
          const T* src = x + row_x[side][t] + h * r.x_head;
          dst[e] = out + row_out[side][t] + h * r.out_head;
          a[e] = *reinterpret_cast<const V*>(src + c0[e]);
          b[e] = *reinterpret_cast<const V*>(src + c1[e]);
        }
        i += di;
        h += dh;
        t += dt;
        if (i >= items) {
          i -= items;
          ++h;
        }
        if (h >= heads) {
          h -= heads;
          ++t;
        }
      }
#pragma unroll
      for (int e = 0; e < kRotBatch; ++e) {
        if (at[e] >= count) break;
        if (c0[e] < p.rotary) {
          const float* cv = (const float*)__builtin_assume_aligned(cs + at[e] * p.table, 16);
          const float* sv = (const float*)__builtin_assume_aligned(sn + at[e] * p.table, 16);
          if constexpr (NEIGHBOURS) {
#pragma unroll
            for (int k = 0; k < VEC / 2; ++k) {
              const float ca = cv[c0[e] / 2 + k], sa = sv[c0[e] / 2 + k], u = (float)a[e].v[2 * k], w = (float)a[e].v[2 * k + 1];
              a[e].v[2 * k] = (T)(u * ca - w * sa);
              a[e].v[2 * k + 1] = (T)(w * ca + u * sa);
              const float cb = cv[c1[e] / 2 + k], sb = sv[c1[e] / 2 + k], y = (float)b[e].v[2 * k], z = (float)b[e].v[2 * k + 1];
              b[e].v[2 * k] = (T)(y * cb - z * sb);
              b[e].v[2 * k + 1] = (T)(z * cb + y * sb);
            }
          } else {
            const int j = INTERLEAVED ? c0[e] / 2 : c0[e];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              const float ca = cv[j + k], sa = sv[j + k], u = (float)a[e].v[k], w = (float)b[e].v[k];
              a[e].v[k] = (T)(u * ca - w * sa);
              b[e].v[k] = (T)(w * ca + u * sa);
            }
          }
        }
        *reinterpret_cast<V*>(dst[e] + c0[e]) = a[e];
        *reinterpret_cast<V*>(dst[e] + c1[e]) = b[e];
      }
    }
  }
}

// Tokens of a workgroup: a power of two, of up to 48 KiB of heads (fp32, with half
// the arithmetic per byte: 32), where 448 workgroups remain, 640 of more than 4 tokens.
// Fewer tokens wait for a table too often, more leave the CUs uneven.  1 / 2 / 4 / 16 tokens: 14639 x 64 heads
// of 128 bf16 100 / 90 / 91 us, x 9 heads of 64 bf16 45 / 26 / 17 / 11; 2 / 4 tokens: 14640 x
// 40 heads of 128 bf16 62 / 56, x 40 heads of 64 fp32 52 / 56, 4096 x 40 heads of 128
// bf16 18 / 16; 1 / 2: 256 x 64 heads of 128 bf16 5.6 / 6.5, 1000 x 64 heads 8.6 / 8.4;
// 8 / 16: 9000 x 16 heads of 80 fp16 12.4 / 14.0.
static int rot_tokens(int64_t all, int64_t token_bytes, int size, int table) {
  const int64_t most = size == 2 ? 49152 : 32768;
  int n = 1;
  while (2 * n <= kRotTokens && 2 * n * table <= kRotTable &&
         ((2 * n * token_bytes <= most && 2 * n <= all / (n < 4 ? 448 : 640)) || all / n > kRotBlocks))
    n *= 2;
  return n;
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
    if (r.heads < 0) return LTX_ERR_INVALID_ARG;
    if (r.heads > kRotHeads) return LTX_ERR_UNSUPPORTED;
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
  if (tokens > 4 * kRotBlocks / batch) return LTX_ERR_UNSUPPORTED;  // (4 tokens of any width fit a workgroup)
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
  p.table = (int)(rotary_dim / 2 + 3) / 4 * 4;
  p.per_block = rot_tokens(all, (p.side[0].heads + p.side[1].heads) * head_dim * (int64_t)size, (int)size, p.table);
  const int64_t blocks = (all + p.per_block - 1) / p.per_block;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == 0) rotary_launch_vec<bf16>(p, vec, interleaved, (int)blocks, s);
  else if (dtype == 1) rotary_launch_vec<_Float16>(p, vec, interleaved, (int)blocks, s);
  else rotary_launch_vec<float>(p, vec, interleaved, (int)blocks, s);
  return ltx_launch_status();
}
