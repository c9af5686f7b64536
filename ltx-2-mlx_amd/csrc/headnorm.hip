// RMS norm of every query and key head, its weights and rotary positions, and
// the gradient:
//
//   r = (mean x^2 + eps)^-1/2,  z = r x u,  u = offset + w,  y = f R(position) z
//   gz = f R(position)^T g,  gn = gz u,  k = mean(gn x) r
//   dx = r (gn - r x k),  dw = sum over tokens and heads of gz r x
//
// with R the rotation of rotary.hip (pairs (i, i + rotary / 2) or (2 i, 2 i + 1) of
// the first `rotary` channels, the others as they are; rotary 0: no rotation).
//
// Bound by memory: every element is read and written once.  A head lives in the
// registers of a group of lanes (a power of two of them, each with one item: the two
// halves of VEC pairs, or two vectors of neighbouring pairs or of plain channels), so
// the sums over its channels are a few lane exchanges.  A lane keeps its channels
// for all heads, and with them the norm weights and, in the gradient, its share of dw.
// Sums, r and dw are fp32, cosines and sines as in rotary.hip from fp64 angles; one
// rounding at the end.
#include <type_traits>

#include "ltx_common.h"

namespace ltx {

constexpr int kHnThreads = 256, kHnTokens = 16, kHnMaxDim = 512;
constexpr int kHnTable = 2048;  // cosines (and sines) of a workgroup
constexpr int64_t kHnBlocks = (1 << 24) - 1;  // a launch has fewer than 2^32 threads
constexpr int64_t kHnHeads = 1 << 30;
constexpr int kHnGradBlocks = 1024;  // workgroups of the gradient, each with a share of dw

struct HnArgs {
  ltx_headnorm_rows side[2];
  int64_t batch, tokens;
  int head_dim, rotary;
  const void* positions;
  int64_t pos_batch;
  int pos_type;
  const double* inv_freq;
  float factor, eps, offset;
  int lanes;      // of a head's group
  int per_block;  // tokens of a tile
  int table;      // table entries of a token: its pairs, up to a multiple of 4
  int64_t tiles;
  float* partial;  // gradient: dw of each workgroup, (blocks, 2, head_dim)
};

__device__ __forceinline__ double hn_position(const HnArgs& p, int64_t i) {
  switch (p.pos_type) {
    case 0: return (double)((const int32_t*)p.positions)[i];
    case 1: return (double)((const int64_t*)p.positions)[i];
    case 2: return (double)((const float*)p.positions)[i];
    default: return ((const double*)p.positions)[i];
  }
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) HnVec {
  T v[VEC];
};

// A lane's item of a head: vectors at channels c0 and c1.
struct HnItem {
  int c0, c1;
  int at;     // first table entry of c0's pairs
  int at1;    // (neighbouring pairs) of c1's
  bool have;  // not past the head's items
  bool two;   // c1 is not c0 again (an odd end)
  bool rot;
};
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ HnItem hn_item(int j, int head_dim, int rotary) {
  constexpr bool NEIGHBOURS = INTERLEAVED && VEC > 1;
  const int pairs = rotary / 2;
  const int rot_vecs = NEIGHBOURS ? rotary / VEC : 2 * (pairs / VEC), copy_vecs = (head_dim - rotary) / VEC;
  const int rot_items = (rot_vecs + 1) / 2, copy_items = (copy_vecs + 1) / 2;
  HnItem it;
  it.have = j < rot_items + copy_items;
  it.rot = j < rot_items;
  it.at = it.at1 = 0;
  if (!it.have) {
    it.c0 = it.c1 = 0;
    it.two = false;
  } else if (!it.rot) {
    j -= rot_items;
    it.two = j + copy_items < copy_vecs;
    it.c0 = rotary + j * VEC;
    it.c1 = it.two ? it.c0 + copy_items * VEC : it.c0;
  } else if (NEIGHBOURS) {
    it.two = j + rot_items < rot_vecs;
    it.c0 = j * VEC;
    it.c1 = it.two ? it.c0 + rot_items * VEC : it.c0;
    it.at = it.c0 / 2;
    it.at1 = it.c1 / 2;
  } else {
    it.two = true;
    it.c0 = INTERLEAVED ? 2 * j : j * VEC;
    it.c1 = INTERLEAVED ? 2 * j + 1 : j * VEC + pairs;
    it.at = it.at1 = INTERLEAVED ? j : j * VEC;
  }
  return it;
}
static int hn_items(int vec, bool interleaved, int head_dim, int rotary) {
  const int rot_vecs = interleaved && vec > 1 ? rotary / vec : 2 * (rotary / 2 / vec);
  return (rot_vecs + 1) / 2 + ((head_dim - rotary) / vec + 1) / 2;
}

// the rotation of an item's values (fp32), cosines and sines of its token at cv, sv
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ void hn_rotate(const HnItem& it, const float* cv, const float* sv, float (&a)[VEC],
                                          float (&b)[VEC]) {
  if (!it.rot) return;
  if constexpr (INTERLEAVED && VEC > 1) {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) {
      const float ca = cv[it.at + k / 2], sa = sv[it.at + k / 2], cb = cv[it.at1 + k / 2], sb = sv[it.at1 + k / 2];
      const float u = a[k], w = a[k + 1], y = b[k], z = b[k + 1];
      a[k] = u * ca - w * sa;
      a[k + 1] = w * ca + u * sa;
      b[k] = y * cb - z * sb;
      b[k + 1] = z * cb + y * sb;
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float c = cv[it.at + k], s = sv[it.at + k], u = a[k], w = b[k];
      a[k] = u * c - w * s;
      b[k] = w * c + u * s;
    }
  }
}

// IPL items per lane (more than one only where a head has more than 64); BATCH
// heads of a group in flight.
template <typename T, int VEC, bool INTERLEAVED, int IPL, bool GRAD>
__global__ __launch_bounds__(kHnThreads) void headnorm_kernel(HnArgs p) {
  using V = HnVec<T, VEC>;
  constexpr int BATCH = IPL > 1 ? 1 : (GRAD ? 2 : 4);
  __shared__ __attribute__((aligned(16))) float cs[kHnTable], sn[kHnTable];
  __shared__ int64_t row_x[2][kHnTokens], row_out[2][kHnTokens], row_g[2][GRAD ? kHnTokens : 1];
  const int pairs = p.rotary / 2;
  const int64_t all = p.batch * p.tokens;
  const int G = p.lanes, groups = kHnThreads / G;
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  HnItem it[IPL];
#pragma unroll
  for (int s = 0; s < IPL; ++s) it[s] = hn_item<VEC, INTERLEAVED>(lane + s * G, p.head_dim, p.rotary);
  float u0[2][IPL][VEC], u1[2][IPL][VEC], d0[2][IPL][VEC], d1[2][IPL][VEC];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int s = 0; s < IPL; ++s)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float* w = p.side[side].weight;
        u0[side][s][k] = w && it[s].have ? p.offset + w[it[s].c0 + k] : 1.0f;
        u1[side][s][k] = w && it[s].have ? p.offset + w[it[s].c1 + k] : 1.0f;
        d0[side][s][k] = d1[side][s][k] = 0.0f;
      }
  const float mean = 1.0f / (float)p.head_dim;

  for (int64_t tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
    const int64_t first = tile * p.per_block;
    const int count = (int)(all - first < p.per_block ? all - first : p.per_block);
    if (GRAD && tile != blockIdx.x) __syncthreads();
    for (int i = threadIdx.x; i < count * pairs; i += kHnThreads) {
      const int t = i / pairs, j = i % pairs;
      const int64_t row = first + t;
      const double pos = hn_position(p, row / p.tokens * p.pos_batch + row % p.tokens);
      double turns = pos * p.inv_freq[j] * 0.15915494309189533576888;  // 1 / (2 pi)
      turns -= rint(turns);
      float s, c;
      sincospif((float)(2.0 * turns), &s, &c);
      cs[t * p.table + j] = c * p.factor;
      sn[t * p.table + j] = (GRAD ? -s : s) * p.factor;
    }
    if (threadIdx.x < 2 * kHnTokens) {
      const int side = threadIdx.x / kHnTokens, t = threadIdx.x % kHnTokens;
      const ltx_headnorm_rows& r = p.side[side];
      const int64_t row = first + t, b = row / p.tokens, tok = row % p.tokens;
      row_x[side][t] = b * r.x_batch + tok * r.x_token;
      row_out[side][t] = b * r.out_batch + tok * r.out_token;
      if constexpr (GRAD) row_g[side][t] = b * r.g_batch + tok * r.g_token;
    }
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const ltx_headnorm_rows& r = p.side[side];
      const int heads = (int)r.heads;
      if (heads == 0) continue;
      const T* x = (const T*)r.x;
      const T* g = (const T*)r.g;
      T* out = (T*)r.out;
      // (token, head) of this group, and what `groups` heads add to it
      int h = group % heads, t = group / heads;
      const int dh = groups % heads, dt = groups / heads;
      while (t < count) {
        V xa[BATCH][IPL], xb[BATCH][IPL], ga[BATCH][IPL], gb[BATCH][IPL];
        int at[BATCH], ah[BATCH];
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
          at[e] = t;
          ah[e] = h;
#pragma unroll
          for (int s = 0; s < IPL; ++s) {
            xa[e][s] = xb[e][s] = V{};
            if constexpr (GRAD) ga[e][s] = gb[e][s] = V{};
            if (t < count && it[s].have) {
              const T* src = x + row_x[side][t] + h * r.x_head;
              xa[e][s] = *reinterpret_cast<const V*>(src + it[s].c0);
              xb[e][s] = *reinterpret_cast<const V*>(src + it[s].c1);
              if constexpr (GRAD) {
                const T* up = g + row_g[side][t] + h * r.g_head;
                ga[e][s] = *reinterpret_cast<const V*>(up + it[s].c0);
                gb[e][s] = *reinterpret_cast<const V*>(up + it[s].c1);
              }
            }
          }
          h += dh;
          t += dt;
          if (h >= heads) {
            h -= heads;
            ++t;
          }
        }
        float ss[BATCH], sg[BATCH];
        float za[BATCH][IPL][VEC], zb[BATCH][IPL][VEC];  // gz
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
          ss[e] = sg[e] = 0.0f;
#pragma unroll
          for (int s = 0; s < IPL; ++s) {
            if constexpr (GRAD) {
#pragma unroll
              for (int k = 0; k < VEC; ++k) {
                za[e][s][k] = (float)ga[e][s].v[k];
                zb[e][s][k] = (float)gb[e][s].v[k];
              }
              const int tt = at[e] < count ? at[e] : 0;
              hn_rotate<VEC, INTERLEAVED>(it[s], (const float*)__builtin_assume_aligned(cs + tt * p.table, 16),
                                          (const float*)__builtin_assume_aligned(sn + tt * p.table, 16), za[e][s],
                                          zb[e][s]);
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              const float va = (float)xa[e][s].v[k], vb = it[s].two ? (float)xb[e][s].v[k] : 0.0f;
              ss[e] += va * va + vb * vb;
              if constexpr (GRAD) sg[e] += va * za[e][s][k] * u0[side][s][k] + vb * zb[e][s][k] * u1[side][s][k];
            }
          }
        }
        for (int off = 1; off < G; off <<= 1)
#pragma unroll
          for (int e = 0; e < BATCH; ++e) {
            ss[e] += __shfl_xor(ss[e], off, kWave);
            if constexpr (GRAD) sg[e] += __shfl_xor(sg[e], off, kWave);
          }
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
          if (at[e] >= count) break;
          const float rn = rsqrt_rn(ss[e] * mean + p.eps);
          const float kk = sg[e] * mean * rn;
          T* dst = out + row_out[side][at[e]] + ah[e] * r.out_head;
          const float* cv = (const float*)__builtin_assume_aligned(cs + at[e] * p.table, 16);
          const float* sv = (const float*)__builtin_assume_aligned(sn + at[e] * p.table, 16);
#pragma unroll
          for (int s = 0; s < IPL; ++s) {
            if (!it[s].have) continue;
            float a[VEC], b[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              const float na = (float)xa[e][s].v[k] * rn, nb = (float)xb[e][s].v[k] * rn;
              if constexpr (GRAD) {
                d0[side][s][k] += za[e][s][k] * na;
                d1[side][s][k] += zb[e][s][k] * nb;
                a[k] = rn * (za[e][s][k] * u0[side][s][k] - na * kk);
                b[k] = rn * (zb[e][s][k] * u1[side][s][k] - nb * kk);
              } else {
                a[k] = na * u0[side][s][k];
                b[k] = nb * u1[side][s][k];
              }
            }
            if constexpr (!GRAD) hn_rotate<VEC, INTERLEAVED>(it[s], cv, sv, a, b);
            V oa, ob;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              oa.v[k] = (T)a[k];
              ob.v[k] = (T)b[k];
            }
            *reinterpret_cast<V*>(dst + it[s].c0) = oa;
            *reinterpret_cast<V*>(dst + it[s].c1) = ob;
          }
        }
      }
    }
  }
  if constexpr (GRAD) {
    // the workgroup's share of dw: the groups of a wave by lane exchanges, the waves through LDS
    // (the tables' place), in wave order
    static_assert(2 * kHnTable >= 4 * kHnMaxDim, "room for the waves' shares");
    const int wave = threadIdx.x / kWave;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      if (p.side[side].dweight == nullptr) continue;
      __syncthreads();
#pragma unroll
      for (int s = 0; s < IPL; ++s)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float a = d0[side][s][k], b = d1[side][s][k];
          for (int off = G; off < kWave; off <<= 1) {
            a += __shfl_xor(a, off, kWave);
            b += __shfl_xor(b, off, kWave);
          }
          if (threadIdx.x % kWave < G && it[s].have) {
            float* dst = (wave < 2 ? cs : sn) + (wave & 1) * kHnMaxDim;
            dst[it[s].c0 + k] = a;
            if (it[s].two) dst[it[s].c1 + k] = b;
          }
        }
      __syncthreads();
      for (int c = threadIdx.x; c < p.head_dim; c += kHnThreads)
        p.partial[((int64_t)blockIdx.x * 2 + side) * p.head_dim + c] =
            (cs[c] + cs[kHnMaxDim + c]) + (sn[c] + sn[kHnMaxDim + c]);
    }
  }
}

// dw from the workgroups' shares: eight channels per workgroup, 32 threads each
__global__ __launch_bounds__(256) void headnorm_dw_kernel(const float* __restrict__ partial, int blocks, int head_dim,
                                                          float* dwq, float* dwk) {
  const int side = blockIdx.y, c = blockIdx.x * 8 + threadIdx.x % 8, part = threadIdx.x / 8;
  float* dw = side == 0 ? dwq : dwk;
  if (dw == nullptr) return;
  __shared__ double sum[256];
  double a = 0.0;
  if (c < head_dim)
    for (int b = part; b < blocks; b += 32) a += (double)partial[((int64_t)b * 2 + side) * head_dim + c];
  sum[threadIdx.x] = a;
  __syncthreads();
  if (part == 0 && c < head_dim) {
    for (int i = 1; i < 32; ++i) a += sum[i * 8 + threadIdx.x];
    dw[c] = (float)a;
  }
}

static int hn_tokens(int64_t all, int64_t token_bytes, int table) {
  int n = 1;
  while (2 * n <= kHnTokens && 2 * n * table <= kHnTable &&
         ((2 * n * token_bytes <= 49152 && 2 * n <= all / (n < 4 ? 448 : 640)) || all / n > kHnBlocks))
    n *= 2;
  return n;
}

template <typename T, int VEC, bool GRAD>
static void hn_launch(const HnArgs& p, bool interleaved, int items, int blocks, hipStream_t s) {
  if (items <= kWave) {
    if (interleaved) headnorm_kernel<T, VEC, true, 1, GRAD><<<blocks, kHnThreads, 0, s>>>(p);
    else headnorm_kernel<T, VEC, false, 1, GRAD><<<blocks, kHnThreads, 0, s>>>(p);
  } else if constexpr (VEC <= 4) {  // (vectors of eight: at most 33 items)
    if (interleaved) headnorm_kernel<T, VEC, true, 4, GRAD><<<blocks, kHnThreads, 0, s>>>(p);
    else headnorm_kernel<T, VEC, false, 4, GRAD><<<blocks, kHnThreads, 0, s>>>(p);
  }
}
template <typename T, bool GRAD>
static void hn_launch_vec(const HnArgs& p, int vec, bool interleaved, int items, int blocks, hipStream_t s) {
  if (vec == 8) {
    if constexpr (sizeof(T) == 2) hn_launch<T, 8, GRAD>(p, interleaved, items, blocks, s);
  } else if (vec == 4) {
    hn_launch<T, 4, GRAD>(p, interleaved, items, blocks, s);
  } else if (vec == 2) {
    hn_launch<T, 2, GRAD>(p, interleaved, items, blocks, s);
  } else {
    hn_launch<T, 1, GRAD>(p, interleaved, items, blocks, s);
  }
}
template <bool GRAD>
static void hn_launch_type(const HnArgs& p, int dtype, int vec, bool interleaved, int items, int blocks, hipStream_t s) {
  if (dtype == 0) hn_launch_vec<bf16, GRAD>(p, vec, interleaved, items, blocks, s);
  else if (dtype == 1) hn_launch_vec<_Float16, GRAD>(p, vec, interleaved, items, blocks, s);
  else hn_launch_vec<float, GRAD>(p, vec, interleaved, items, blocks, s);
}

// Checks and arguments of both entry points; *vec and *items: the kernel's form.
// LTX_OK with p->tiles == 0: nothing to do.
static int hn_args(const ltx_headnorm_rows* q, const ltx_headnorm_rows* k, bool grad, int dtype, int64_t batch,
                   int64_t tokens, int64_t head_dim, int64_t rotary_dim, const void* positions, int pos_type,
                   int64_t pos_batch, const double* inv_freq, double factor, double eps, double offset, int flags,
                   HnArgs* p, int* vec, int* items) {
  if (!q || batch < 0 || tokens < 0 || head_dim < 1 || rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
    return LTX_ERR_INVALID_ARG;
  if (dtype < 0 || dtype > 2 || pos_type < 0 || pos_type > 3) return LTX_ERR_UNSUPPORTED;
  if (flags & ~LTX_ROTARY_INTERLEAVED || !(eps >= 0.0)) return LTX_ERR_INVALID_ARG;
  if (head_dim > kHnMaxDim) return LTX_ERR_UNSUPPORTED;
  const uintptr_t pos_size = pos_type == 1 || pos_type == 3 ? 8 : 4, size = dtype == 2 ? 4 : 2;
  const bool some = batch > 0 && tokens > 0;  // (tensors of no elements may have no address)
  if (rotary_dim > 0 && some) {
    if (!positions || !inv_freq || pos_batch < 0) return LTX_ERR_INVALID_ARG;
    if ((uintptr_t)positions % pos_size || (uintptr_t)inv_freq % 8) return LTX_ERR_ALIGNMENT;
  }
  *p = {};
  p->side[0] = *q;
  if (k) p->side[1] = *k;
  const bool interleaved = (flags & LTX_ROTARY_INTERLEAVED) != 0;
  // the widest vector that divides every extent, stride and address
  int64_t bits = interleaved ? rotary_dim : rotary_dim / 2;
  bits |= head_dim - rotary_dim;
  int64_t heads = 0;
  for (ltx_headnorm_rows& r : p->side) {
    if (!grad) r.dweight = nullptr;
    if (r.heads < 0 || (r.dweight && !r.weight)) return LTX_ERR_INVALID_ARG;
    if (r.heads > kHnHeads) return LTX_ERR_UNSUPPORTED;
    if ((uintptr_t)r.weight % 4 || (uintptr_t)r.dweight % 4) return LTX_ERR_ALIGNMENT;
    if (r.heads == 0 || !some) continue;
    heads += r.heads;
    if (!r.x || !r.out || (grad && !r.g)) return LTX_ERR_INVALID_ARG;
    if ((uintptr_t)r.x % size || (uintptr_t)r.out % size || (grad && (uintptr_t)r.g % size)) return LTX_ERR_ALIGNMENT;
    bits |= (int64_t)((uintptr_t)r.x / size | (uintptr_t)r.out / size | (grad ? (uintptr_t)r.g / size : 0));
    // the stride of an axis of one entry is never used
    if (batch > 1) bits |= r.x_batch | r.out_batch | (grad ? r.g_batch : 0);
    if (tokens > 1) bits |= r.x_token | r.out_token | (grad ? r.g_token : 0);
    if (r.heads > 1) bits |= r.x_head | r.out_head | (grad ? r.g_head : 0);
  }
  if (heads == 0) return LTX_OK;
  if (tokens > 4 * kHnBlocks / batch) return LTX_ERR_UNSUPPORTED;  // (4 tokens of any width fit a workgroup)
  *vec = (int)(16 / size);
  while (*vec > 1 && (bits & (*vec - 1))) *vec >>= 1;
  *items = hn_items(*vec, interleaved, (int)head_dim, (int)rotary_dim);
  p->lanes = 1;
  while (p->lanes < *items && p->lanes < kWave) p->lanes *= 2;
  p->batch = batch;
  p->tokens = tokens;
  p->head_dim = (int)head_dim;
  p->rotary = (int)rotary_dim;
  p->positions = positions;
  p->pos_type = pos_type;
  p->pos_batch = pos_batch;
  p->inv_freq = inv_freq;
  p->factor = (float)factor;
  p->eps = (float)eps;
  p->offset = (float)offset;
  p->table = (int)(rotary_dim / 2 + 3) / 4 * 4;
  const int64_t all = batch * tokens;
  p->per_block = hn_tokens(all, heads * head_dim * (int64_t)size, p->table);
  p->tiles = (all + p->per_block - 1) / p->per_block;
  return LTX_OK;
}

}  // namespace ltx

using namespace ltx;

extern "C" int ltx_headnorm_rotary(const ltx_headnorm_rows* q, const ltx_headnorm_rows* k, int dtype, int64_t batch,
                                   int64_t tokens, int64_t head_dim, int64_t rotary_dim, const void* positions,
                                   int pos_type, int64_t pos_batch, const double* inv_freq, double factor, double eps,
                                   double weight_offset, int flags, void* stream) {
  HnArgs p;
  int vec, items;
  const int st = hn_args(q, k, false, dtype, batch, tokens, head_dim, rotary_dim, positions, pos_type, pos_batch,
                         inv_freq, factor, eps, weight_offset, flags, &p, &vec, &items);
  if (st != LTX_OK || p.tiles == 0) return st;
  hn_launch_type<false>(p, dtype, vec, (flags & LTX_ROTARY_INTERLEAVED) != 0, items, (int)p.tiles, (hipStream_t)stream);
  return ltx_launch_status();
}

extern "C" int64_t ltx_headnorm_rotary_grad_workspace_bytes(int64_t head_dim) {
  return head_dim < 0 ? -1 : (int64_t)kHnGradBlocks * 2 * head_dim * 4;
}

extern "C" int ltx_headnorm_rotary_grad(const ltx_headnorm_rows* q, const ltx_headnorm_rows* k, int dtype,
                                        int64_t batch, int64_t tokens, int64_t head_dim, int64_t rotary_dim,
                                        const void* positions, int pos_type, int64_t pos_batch, const double* inv_freq,
                                        double factor, double eps, double weight_offset, int flags, float* workspace,
                                        int64_t workspace_bytes, void* stream) {
  HnArgs p;
  int vec, items;
  const int st = hn_args(q, k, true, dtype, batch, tokens, head_dim, rotary_dim, positions, pos_type, pos_batch,
                         inv_freq, factor, eps, weight_offset, flags, &p, &vec, &items);
  if (st != LTX_OK) return st;
  const bool sums = p.side[0].dweight || p.side[1].dweight;
  if (p.tiles > 0 && sums) {
    if (!workspace || workspace_bytes < ltx_headnorm_rotary_grad_workspace_bytes(head_dim)) return LTX_ERR_INVALID_ARG;
    if ((uintptr_t)workspace % 4) return LTX_ERR_ALIGNMENT;
  }
  hipStream_t s = (hipStream_t)stream;
  int blocks = 0;
  if (p.tiles > 0) {
    p.partial = workspace;
    blocks = (int)(p.tiles < kHnGradBlocks ? p.tiles : kHnGradBlocks);
    hn_launch_type<true>(p, dtype, vec, (flags & LTX_ROTARY_INTERLEAVED) != 0, items, blocks, s);
    const int e = ltx_launch_status();
    if (e != LTX_OK) return e;
  }
  if (!sums) return LTX_OK;
  headnorm_dw_kernel<<<dim3((unsigned)(head_dim + 7) / 8, 2), 256, 0, s>>>(workspace, blocks, (int)head_dim,
                                                                          p.side[0].dweight, p.side[1].dweight);
  return ltx_launch_status();
}
