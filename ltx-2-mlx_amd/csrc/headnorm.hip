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
// Bound by memory: every element is read and written once.  A workgroup takes the
// query heads or the key heads of a few tokens.  A head lives in the
// registers of a group of lanes (a power of two of them, each with one item: the two
// halves of VEC pairs, or two vectors of neighbouring pairs or of plain channels), so
// the sums over its channels are a few lane exchanges.  A lane keeps its channels
// for all heads, and with them the norm weights and, in the gradient, its share of dw.
// The first heads are on their way while the workgroup computes its tokens' cosines and
// sines, the next ones while it works on these.
// Sums and r are fp32, cosines and sines as in rotary.hip from fp64 angles; one
// rounding at the end.  A lane's share of dw is fp32 over kHnRun heads, then the workgroup's is added to
// in fp64: however long a call is, its chains of fp32 sums are not longer.
// Measured, inputs from HBM: 3456 tokens x 64 heads of 128 bf16 30 us (3.8 TB/s; 23 with part of them in a cache,
// the rotation alone 22), 14640 x 40
// heads of 128 bf16 66 (4.5 TB/s), 14639 x 40 heads of 64 fp32 62 (4.8 TB/s), one token 4.3, its gradient at
// 14640 x 40 heads of 128 bf16 94 (4.8 TB/s, 4 of them the second launch), 3456 x 64 heads 47 (39 with part of them
// in a cache).  Heads of 80 and 96 have five and six items in groups of eight lanes: 9000 x 16 of them in fp16 20 and 22
// us, the gradient 30 and 32, where a copy of as many bytes takes 9.0, 10.8, 13.5 and 16.2.  About
// 300 vector instructions per eight heads of 128 lie beside the loads.  Beside it: both sides in one
// workgroup 43, 88 and 127 us (3456 and 14640 tokens, gradient); two heads on their way and one at work
// (29, 70, 102); as many workgroups as the CUs hold, each with tiles of the same size (28, 70, 101); positions in
// batches of four, a pair per thread (29, 65, 109).
#include <type_traits>

#include "ltx_common.h"

namespace ltx {

constexpr int kHnThreads = 256, kHnTokens = 16, kHnMaxDim = 512;
constexpr int kHnTable = 2048;  // cosines (and sines) of a workgroup
constexpr int64_t kHnBlocks = (1 << 23) - 1;  // of a side: a launch has fewer than 2^32 threads
constexpr int64_t kHnHeads = 1 << 30;
// Workgroups of a side of the gradient, each with a share of dw and one tile after another.  384 /
// 512 / 1024, inputs from HBM: 14640 x 32 and 8 heads of 128 bf16 99 / 94 / 98 us, 3456 x 32 heads of each side
// 44 / 47 / 53, 9000 x 12 and 4 heads of 80 fp16 31 / 30 / 30.  (147 registers: the chip holds 768 at a time, so of
// two long sides' 1024 a quarter waits for a second round.)
constexpr int kHnGradBlocks = 512;
// Heads of a group up to which one workgroup takes a side of the gradient, and its dw needs no
// second launch.  One launch / two, 32 and 8 heads of 128 bf16: 1 token 6.7 / 8.9 us, 2 tokens 7.4 / 8.8, 4 (four
// heads a group) 9.1 / 8.8, 6 11.1 / 8.9; a launch costs the host 3.
constexpr int kHnAlone = 4;
// Heads that a lane adds to its fp32 share of dw before the workgroup's fp64 sums take it
constexpr int kHnRun = 256;

struct HnSide {
  ltx_headnorm_rows r;
  int per_block;      // tokens of a tile
  int tiles, blocks;  // (forward: a workgroup each)
};
struct HnArgs {
  HnSide side[2];
  int batch, tokens, all;
  int head_dim, rotary;
  const void* positions;
  int64_t pos_batch;
  int pos_type;
  const double* inv_freq;
  float factor, eps, offset;
  int lanes;       // of a head's group
  int table;       // table entries of a token: its pairs, up to a multiple of 4
  float* partial;  // gradient: dw of each workgroup, (blocks, head_dim)
  bool alone;      // gradient: a workgroup per side, whose dw is the result
};

__device__ __forceinline__ double hn_position(const HnArgs& p, int64_t i) {
  switch (p.pos_type) {
    case 0: return (double)((const int32_t*)p.positions)[i];
    case 1: return (double)((const int64_t*)p.positions)[i];
    case 2: return (double)((const float*)p.positions)[i];
    default: return ((const double*)p.positions)[i];
  }
}

// sum over the lanes of a group (of G consecutive ones, a power of two)
template <int CTRL>
__device__ __forceinline__ float hn_dpp(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ void hn_group_sum(float (&v)[N], int G) {
  auto all = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = f(v[e]);
  };
  if (G < 2) return;
  all([](float x) { return hn_dpp<0xB1>(x); });  // the neighbour
  if (G < 4) return;
  all([](float x) { return hn_dpp<0x4E>(x); });  // the other pair of four
  if (G < 8) return;
  all([](float x) { return hn_dpp<0x141>(x); });  // eight lanes mirrored
  if (G < 16) return;
  all([](float x) { return hn_dpp<0x140>(x); });  // sixteen mirrored
  if (G < 32) return;
  all([](float x) { return x + __shfl_xor(x, 16, kWave); });
  if (G < 64) return;
  all([](float x) { return x + __shfl_xor(x, 32, kWave); });
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

// the rotation of an item's values (fp32), cosines and sines of its token at cv, sv (16-byte aligned)
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ void hn_rotate(const HnItem& it, const float* cv, const float* sv, float (&a)[VEC],
                                          float (&b)[VEC]) {
  if (!it.rot) return;
  if constexpr (INTERLEAVED && VEC > 1) {
    using P = HnVec<float, VEC / 2>;
    const P c0 = *reinterpret_cast<const P*>(cv + it.at), s0 = *reinterpret_cast<const P*>(sv + it.at);
    const P c1 = *reinterpret_cast<const P*>(cv + it.at1), s1 = *reinterpret_cast<const P*>(sv + it.at1);
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) {
      const float u = a[2 * k], w = a[2 * k + 1], y = b[2 * k], z = b[2 * k + 1];
      a[2 * k] = u * c0.v[k] - w * s0.v[k];
      a[2 * k + 1] = w * c0.v[k] + u * s0.v[k];
      b[2 * k] = y * c1.v[k] - z * s1.v[k];
      b[2 * k + 1] = z * c1.v[k] + y * s1.v[k];
    }
  } else {
    constexpr int Q = VEC < 4 ? VEC : 4;
    using P = HnVec<float, Q>;
#pragma unroll
    for (int k = 0; k < VEC; k += Q) {
      const P c = *reinterpret_cast<const P*>(cv + it.at + k), s = *reinterpret_cast<const P*>(sv + it.at + k);
#pragma unroll
      for (int e = 0; e < Q; ++e) {
        const float u = a[k + e], w = b[k + e];
        a[k + e] = u * c.v[e] - w * s.v[e];
        b[k + e] = w * c.v[e] + u * s.v[e];
      }
    }
  }
}

// IPL items per lane (more than one only where a head has more than 64); BATCH heads of
// a group at work, as many on their way.
template <typename T, int VEC, bool INTERLEAVED, int IPL, bool GRAD>
__global__ __launch_bounds__(kHnThreads) void headnorm_kernel(HnArgs p) {
  using V = HnVec<T, VEC>;
  constexpr int BATCH = IPL > 1 || GRAD ? 1 : 2;
  __shared__ __attribute__((aligned(16))) float cs[kHnTable], sn[kHnTable];
  __shared__ double dws[GRAD ? kHnMaxDim : 1];  // gradient: the workgroup's dw
  const bool keys = (int)blockIdx.x >= p.side[0].blocks;
  const HnSide& side = p.side[keys];
  const ltx_headnorm_rows& r = side.r;
  const int block = (int)blockIdx.x - (keys ? p.side[0].blocks : 0);
  const int pairs = p.rotary / 2, heads = (int)r.heads;
  const int G = p.lanes, groups = kHnThreads / G;
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  HnItem it[IPL];
#pragma unroll
  for (int s = 0; s < IPL; ++s) it[s] = hn_item<VEC, INTERLEAVED>(lane + s * G, p.head_dim, p.rotary);

  // Heads of a group in flight.  Loads past the tile's tokens repeat its last one's, those of
  // a lane without an item the head's first vector: no branch waits for them.
  struct Heads {
    V xa[BATCH][IPL], xb[BATCH][IPL], ga[GRAD ? BATCH : 1][IPL], gb[GRAD ? BATCH : 1][IPL];
    int t[BATCH], h[BATCH];
  };
  const int dh = groups % heads, dt = groups / heads;
  int first = 0, count = 0, t = 0, h = 0;  // the tile; (token, head) of the group's next load
  // element (token t of the tile, head h) of a tensor
  auto offset = [&](int tt, int hh, int64_t batch, int64_t token, int64_t head) __attribute__((always_inline)) {
    uint32_t row = (uint32_t)(first + tt);
    int64_t at = 0;
    if (p.batch > 1) {
      const uint32_t b = row / (uint32_t)p.tokens;
      row -= b * (uint32_t)p.tokens;
      at = (int64_t)b * batch;
    }
    // (token and head strides below 2^32)
    return at + (int64_t)((uint64_t)row * (uint32_t)token) + (int64_t)((uint64_t)(uint32_t)hh * (uint32_t)head);
  };
  auto load = [&](Heads& n) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < BATCH; ++e) {
      n.t[e] = t;
      n.h[e] = h;
      const int tt = t < count ? t : count - 1;
      const T* src = (const T*)r.x + offset(tt, h, r.x_batch, r.x_token, r.x_head);
#pragma unroll
      for (int s = 0; s < IPL; ++s) {
        n.xa[e][s] = *reinterpret_cast<const V*>(src + it[s].c0);
        n.xb[e][s] = *reinterpret_cast<const V*>(src + it[s].c1);
      }
      if constexpr (GRAD) {
        const T* up = (const T*)r.g + offset(tt, h, r.g_batch, r.g_token, r.g_head);
#pragma unroll
        for (int s = 0; s < IPL; ++s) {
          n.ga[e][s] = *reinterpret_cast<const V*>(up + it[s].c0);
          n.gb[e][s] = *reinterpret_cast<const V*>(up + it[s].c1);
        }
      }
      h += dh;
      t += dt;
      if (h >= heads) {
        h -= heads;
        ++t;
      }
    }
  };

  float u0[IPL][VEC], u1[IPL][VEC], d0[GRAD ? IPL : 1][VEC], d1[GRAD ? IPL : 1][VEC];
  const float mean = 1.0f / (float)p.head_dim;
  auto work = [&](const Heads& c) __attribute__((always_inline)) {
    float sums[GRAD ? 2 * BATCH : BATCH];            // of x^2, of gz u x
    float za[BATCH][IPL][VEC], zb[BATCH][IPL][VEC];  // gz
#pragma unroll
    for (int e = 0; e < BATCH; ++e) {
      float ss = 0.0f, sg = 0.0f;
#pragma unroll
      for (int s = 0; s < IPL; ++s) {
        if constexpr (GRAD) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            za[e][s][k] = (float)c.ga[e][s].v[k];
            zb[e][s][k] = (float)c.gb[e][s].v[k];
          }
          const int at = (c.t[e] < count ? c.t[e] : 0) * p.table;
          hn_rotate<VEC, INTERLEAVED>(it[s], cs + at, sn + at, za[e][s], zb[e][s]);
        }
        float sa = 0.0f, sb = 0.0f, ta = 0.0f, tb = 0.0f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float va = (float)c.xa[e][s].v[k], vb = (float)c.xb[e][s].v[k];
          sa += va * va;
          sb += vb * vb;
          if constexpr (GRAD) {
            ta += va * (za[e][s][k] * u0[s][k]);
            tb += vb * (zb[e][s][k] * u1[s][k]);
          }
        }
        ss += it[s].have ? sa + (it[s].two ? sb : 0.0f) : 0.0f;
        if constexpr (GRAD) sg += it[s].have ? ta + (it[s].two ? tb : 0.0f) : 0.0f;
      }
      sums[e] = ss;
      if constexpr (GRAD) sums[BATCH + e] = sg;
    }
    hn_group_sum(sums, G);
#pragma unroll
    for (int e = 0; e < BATCH; ++e) {
      if (c.t[e] >= count) break;
      const float rn = rsqrt_rn(sums[e] * mean + p.eps);
      T* dst = (T*)r.out + offset(c.t[e], c.h[e], r.out_batch, r.out_token, r.out_head);
      const int at = c.t[e] * p.table;
#pragma unroll
      for (int s = 0; s < IPL; ++s) {
        if (!it[s].have) continue;
        float va[VEC], vb[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float na = (float)c.xa[e][s].v[k] * rn, nb = (float)c.xb[e][s].v[k] * rn;
          if constexpr (GRAD) {
            const float kk = sums[BATCH + e] * mean * rn;
            d0[s][k] += za[e][s][k] * na;
            d1[s][k] += zb[e][s][k] * nb;
            va[k] = rn * (za[e][s][k] * u0[s][k] - na * kk);
            vb[k] = rn * (zb[e][s][k] * u1[s][k] - nb * kk);
          } else {
            va[k] = na * u0[s][k];
            vb[k] = nb * u1[s][k];
          }
        }
        if constexpr (!GRAD) hn_rotate<VEC, INTERLEAVED>(it[s], cs + at, sn + at, va, vb);
        V oa, ob;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          oa.v[k] = (T)va[k];
          ob.v[k] = (T)vb[k];
        }
        *reinterpret_cast<V*>(dst + it[s].c0) = oa;
        *reinterpret_cast<V*>(dst + it[s].c1) = ob;
      }
    }
  };
  // The lanes' shares of dw to the workgroup's sums: the groups of a wave by lane exchanges, the
  // waves through LDS in wave order.  All threads, at the same turn.
  int run = 0;
  if (GRAD)
    for (int c = threadIdx.x; c < p.head_dim; c += kHnThreads) dws[c] = 0.0;  // (a thread adds to its own ones only)
  auto share = [&]() __attribute__((always_inline)) {
    if constexpr (GRAD) {
      __shared__ float waves[kHnThreads / kWave][kHnMaxDim];
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));  // (keeps what depends on it out of the registers of the turns)
      const int wave = tid / kWave, own = tid % kWave;
      run = 0;
      if (r.dweight == nullptr) return;
      auto from = [](float v, int from_lane) __attribute__((always_inline)) {
        return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(from_lane * 4, __builtin_bit_cast(int, v)));
      };
      __syncthreads();
#pragma unroll
      for (int s = 0; s < IPL; ++s)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float va = d0[s][k], vb = d1[s][k];
          d0[s][k] = d1[s][k] = 0.0f;
          for (int off = G; off < kWave; off <<= 1) {
            va += from(va, own ^ off);
            vb += from(vb, own ^ off);
          }
          if (own < G && it[s].have) {
            waves[wave][it[s].c0 + k] = va;
            if (it[s].two) waves[wave][it[s].c1 + k] = vb;
          }
        }
      __syncthreads();
      for (int c = tid; c < p.head_dim; c += kHnThreads) {
        const float part = (waves[0][c] + waves[1][c]) + (waves[2][c] + waves[3][c]);
        dws[c] += (double)part;
      }
    }
  };
  for (int tile = block; tile < side.tiles; tile += side.blocks) {
    first = tile * side.per_block;
    count = p.all - first < side.per_block ? p.all - first : side.per_block;
    t = group / heads;
    h = group % heads;
    Heads now;
    load(now);
    if (!GRAD || tile == block) {
#pragma unroll
      for (int s = 0; s < IPL; ++s)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          u0[s][k] = r.weight ? p.offset + r.weight[it[s].c0 + k] : 1.0f;
          u1[s][k] = r.weight ? p.offset + r.weight[it[s].c1 + k] : 1.0f;
          if constexpr (GRAD) d0[s][k] = d1[s][k] = 0.0f;
        }
    } else {
      __syncthreads();  // the last tile's table
    }
    for (int i = threadIdx.x; i < count * pairs; i += kHnThreads) {
      const int tt = i / pairs, j = i - tt * pairs;
      uint32_t row = (uint32_t)(first + tt);
      int64_t at = 0;
      if (p.batch > 1) {
        at = (int64_t)(row / (uint32_t)p.tokens) * p.pos_batch;
        row %= (uint32_t)p.tokens;
      }
      double turns = hn_position(p, at + row) * p.inv_freq[j] * 0.15915494309189533576888;  // 1 / (2 pi)
      turns -= rint(turns);
      float sine, cosine;
      sincospif((float)(2.0 * turns), &sine, &cosine);
      cs[tt * p.table + j] = cosine * p.factor;
      sn[tt * p.table + j] = (GRAD ? -sine : sine) * p.factor;
    }
    __syncthreads();
    const int turns = (int)(((int64_t)count * heads + groups * BATCH - 1) / (groups * BATCH));
    for (int i = 1; i < turns; ++i) {
      Heads next;
      load(next);
      work(now);
      now = next;
      if (GRAD && ++run == kHnRun) share();
    }
    work(now);
    if (GRAD && ++run == kHnRun) share();
  }
  if constexpr (GRAD) {
    if (r.dweight == nullptr) return;
    share();
    float* dw = p.alone ? r.dweight : p.partial + (int64_t)blockIdx.x * p.head_dim;
    for (int c = threadIdx.x; c < p.head_dim; c += kHnThreads) dw[c] = (float)dws[c];
  }
}

// dw from the workgroups' shares: eight channels per workgroup, 64 threads each
__global__ __launch_bounds__(512) void headnorm_dw_kernel(const float* __restrict__ partial, int blocks_q, int blocks_k,
                                                          int head_dim, float* dwq, float* dwk) {
  const bool keys = blockIdx.y != 0;
  const int c = blockIdx.x * 8 + threadIdx.x % 8, part = threadIdx.x / 8;
  const int from = keys ? blocks_q : 0, to = keys ? blocks_q + blocks_k : blocks_q;
  float* dw = keys ? dwk : dwq;
  if (dw == nullptr) return;
  __shared__ double sum[512];
  double a = 0.0;
  if (c < head_dim) {
#pragma unroll 8
    for (int b = from + part; b < to; b += 64) a += (double)partial[(int64_t)b * head_dim + c];
  }
  sum[threadIdx.x] = a;
  __syncthreads();
  for (int n = 256; n >= 8; n /= 2) {
    if ((int)threadIdx.x < n) sum[threadIdx.x] += sum[threadIdx.x + n];
    __syncthreads();
  }
  if (part == 0 && c < head_dim) dw[c] = (float)sum[threadIdx.x];
}

// Tokens of a tile: a power of two, of up to 96 KiB of heads (48 KiB in fp32, with half the
// arithmetic per byte, and in the gradient) where 300 tiles remain.  24 / 48 / 96 / 192 KiB: 3456 x 32 heads of 128
// bf16 of each side 40 / 31 / 29 / 29 us, 14640 x 32 and 8 heads 90 / 68 / 65 / 67, 14639 x 32
// and 8 heads of 64 fp32 71 / 59 / 62 / 66.
static int hn_tokens(int64_t all, int64_t token_bytes, bool small, int table) {
  const int64_t most = small ? 49152 : 98304;
  int n = 1;
  while (2 * n <= kHnTokens && 2 * n * table <= kHnTable &&
         ((2 * n * token_bytes <= most && 2 * n <= all / 300) || all / n > kHnBlocks))
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
static void hn_launch_type(const HnArgs& p, int dtype, int vec, bool interleaved, int items, int blocks,
                           hipStream_t s) {
  if (dtype == 0) hn_launch_vec<bf16, GRAD>(p, vec, interleaved, items, blocks, s);
  else if (dtype == 1) hn_launch_vec<_Float16, GRAD>(p, vec, interleaved, items, blocks, s);
  else hn_launch_vec<float, GRAD>(p, vec, interleaved, items, blocks, s);
}

// Checks and arguments of both entry points; *vec and *items: the kernel's form.
// LTX_OK with no tiles on either side: nothing to do.
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
  p->side[0].r = *q;
  if (k) p->side[1].r = *k;
  const bool interleaved = (flags & LTX_ROTARY_INTERLEAVED) != 0;
  // the widest vector that divides every extent, stride and address
  int64_t bits = interleaved ? rotary_dim : rotary_dim / 2;
  bits |= head_dim - rotary_dim;
  int64_t heads = 0;
  for (HnSide& side : p->side) {
    ltx_headnorm_rows& r = side.r;
    if (!grad) r.dweight = nullptr;
    if (r.heads < 0 || (r.dweight && !r.weight)) return LTX_ERR_INVALID_ARG;
    if (r.heads > kHnHeads) return LTX_ERR_UNSUPPORTED;
    if ((uintptr_t)r.weight % 4 || (uintptr_t)r.dweight % 4) return LTX_ERR_ALIGNMENT;
    if (r.heads == 0 || !some) continue;
    heads += r.heads;
    if (!r.x || !r.out || (grad && !r.g)) return LTX_ERR_INVALID_ARG;
    if ((uintptr_t)r.x % size || (uintptr_t)r.out % size || (grad && (uintptr_t)r.g % size)) return LTX_ERR_ALIGNMENT;
    bits |= (int64_t)((uintptr_t)r.x / size | (uintptr_t)r.out / size | (grad ? (uintptr_t)r.g / size : 0));
    // the stride of an axis of one entry is never used; offsets of tokens and heads are products of 32 bits
    auto narrow = [grad](int64_t x, int64_t out, int64_t g) {
      return (uint64_t)x >> 32 == 0 && (uint64_t)out >> 32 == 0 && (!grad || (uint64_t)g >> 32 == 0);
    };
    if ((tokens > 1 && !narrow(r.x_token, r.out_token, r.g_token)) ||
        (r.heads > 1 && !narrow(r.x_head, r.out_head, r.g_head)))
      return LTX_ERR_UNSUPPORTED;
    if (batch > 1) bits |= r.x_batch | r.out_batch | (grad ? r.g_batch : 0);
    if (tokens > 1) bits |= r.x_token | r.out_token | (grad ? r.g_token : 0);
    if (r.heads > 1) bits |= r.x_head | r.out_head | (grad ? r.g_head : 0);
  }
  if (heads == 0) return LTX_OK;
  if (tokens > 4 * kHnBlocks / batch) return LTX_ERR_UNSUPPORTED;  // (4 tokens of any width fit a tile)
  *vec = (int)(16 / size);
  while (*vec > 1 && (bits & (*vec - 1))) *vec >>= 1;
  *items = hn_items(*vec, interleaved, (int)head_dim, (int)rotary_dim);
  p->lanes = 1;
  while (p->lanes < *items && p->lanes < kWave) p->lanes *= 2;
  p->batch = (int)batch;
  p->tokens = (int)tokens;
  p->all = (int)(batch * tokens);
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
  const int64_t groups = kHnThreads / p->lanes;
  p->alone = grad;
  for (const HnSide& side : p->side)
    if (p->all * side.r.heads > kHnAlone * groups || (side.r.heads == 0 && side.r.dweight)) p->alone = false;
  for (HnSide& side : p->side) {
    if (side.r.heads == 0) continue;
    if (p->alone) {
      side.per_block = 1;
      while (side.per_block < p->all && 2 * side.per_block * p->table <= kHnTable) side.per_block *= 2;
    } else {
      side.per_block = hn_tokens(p->all, side.r.heads * head_dim * (int64_t)size, size == 4 || grad, p->table);
    }
    side.tiles = (p->all + side.per_block - 1) / side.per_block;
    side.blocks = p->alone ? 1 : (!grad || side.tiles < kHnGradBlocks ? side.tiles : kHnGradBlocks);
  }
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
  const int blocks = p.side[0].blocks + p.side[1].blocks;
  if (st != LTX_OK || blocks == 0) return st;
  hn_launch_type<false>(p, dtype, vec, (flags & LTX_ROTARY_INTERLEAVED) != 0, items, blocks, (hipStream_t)stream);
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
  float *dwq = p.side[0].r.dweight, *dwk = p.side[1].r.dweight;
  const int blocks = p.side[0].blocks + p.side[1].blocks;
  if (blocks > 0 && (dwq || dwk)) {
    if (!workspace || workspace_bytes < ltx_headnorm_rotary_grad_workspace_bytes(head_dim)) return LTX_ERR_INVALID_ARG;
    if ((uintptr_t)workspace % 4) return LTX_ERR_ALIGNMENT;
  }
  hipStream_t s = (hipStream_t)stream;
  if (blocks > 0) {
    p.partial = workspace;
    hn_launch_type<true>(p, dtype, vec, (flags & LTX_ROTARY_INTERLEAVED) != 0, items, blocks, s);
    const int e = ltx_launch_status();
    if (e != LTX_OK) return e;
  }
  if ((!dwq && !dwk) || p.alone) return LTX_OK;
  headnorm_dw_kernel<<<dim3((unsigned)(head_dim + 7) / 8, 2), 512, 0, s>>>(
      workspace, p.side[0].blocks, p.side[1].blocks, (int)head_dim, dwq, dwk);
  return ltx_launch_status();
}
