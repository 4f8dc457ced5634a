// RMS norm of every query and key head with the rotation by position in the same pass, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,  y = turn(n)      for every head x of every token, D = head dimension
//   turn: the first R dimensions in pairs (a, b) -> (a cos - b sin, b cos + a sin), the others unchanged; the pairs are
//   (i, i + R/2), or (2i, 2i + 1) when interleaved; cos / sin come from tables, row = the token's position
//   backward: g = turn by the negative angle of dy;  dw = sum g x r;  dx = r (g w - x r^2 mean(g w x))
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.  The norm is recomputed from x in
// the backward, which has to read x anyway, so nothing is kept between the two.
//
// A head is split into units of two vectors of VEC elements, chosen so that a rotation never leaves a unit: for split
// halves the vectors lie R/2 apart, for interleaved pairs they are neighbours.  A unit sits in one lane, so the rotation
// needs no exchange, and the norm is one reduction over the group of lanes (a power of two) that shares a head: at D = 64
// in 16 bits a head is four lanes with two 16-byte loads each, eight heads per warp.  A group walks over some heads
// of one token and keeps the token's cos / sin and the weight in registers, while its next heads are copied to shared memory.
//
// Measured on a B200 (bf16, queries of 32 and keys of 8 heads of 128 at 8 x 2048 tokens, slices of a packed projection): forward 68 us =
// 4.9 TB/s, 0.75 of the measured copy bandwidth (82 us with loads that waited for the head before), where issue slots run out (70 %
// busy); backward with the weights' gradients 126 us = 4.0 TB/s, 0.61 (178 us).  The backward is short of warps: 121 registers leave two
// blocks of 256 threads on an SM, 24 % of its warps, which keep 60 % of the issue slots busy.  fp32, 16 + 16 heads of 64: 50 and 74 us =
// 5.4 and 5.5 TB/s.  Head dimensions that leave lanes of a group idle or narrow the vectors run at 1.3 to 2.5 TB/s (80: five of eight
// lanes; 100: vectors of two).
#include "kernels_api.h"
#include "row_vec.cuh"

namespace {

using namespace rowvec;

constexpr int kThreads = 256;

// One side of the pass: the queries or the keys.
struct Side {
  const void* x;
  const void* dy;       // backward
  void* out;            // y or dx, contiguous [tokens, heads, D]
  const void* weight;   // [D] or null
  float* dw_partial;    // backward: [blocks of this side][D], or null
  long long xs_b, xs_l, xs_h, gs_b, gs_l, gs_h;  // strides of x and dy in elements
  int heads, weight_dtype;
  int heads_per_item, items_per_token;
  unsigned items;       // tokens * items_per_token
  int blocks;
};
struct Args {
  Side side[2];
  const float* cos;
  const float* sin;
  const void* positions;  // int64 / int32, or null: the token's place in its sequence
  long long pos_b, pos_l;
  int pos_is_64;
  long long table_rows;
  int* bad_flag;        // set when a position lies behind the tables; may be null
  unsigned L;
  int D, R, group;      // lanes per head
  float eps;
};

__device__ __forceinline__ float weight_at(const void* w, int dt, int i) {
  if (dt == B200_F32) return static_cast<const float*>(w)[i];
  if (dt == B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// Where the two vectors of a unit begin, and whether they rotate.
template <int VEC, bool INTER>
__device__ __forceinline__ void place(int unit, int R, int& lo, int& hi, bool& rot) {
  const int first = unit * 2 * VEC;
  if (INTER || first >= R) { lo = first; hi = first + VEC; rot = first < R; }
  else { lo = unit * VEC; hi = R / 2 + unit * VEC; rot = true; }
}

// The arithmetic takes elements in pairs, two to an instruction, wherever a vector has any.
template <int VEC>
__device__ __forceinline__ float2 pair(const float (&a)[VEC], int i) { return make_float2(a[2 * i], a[2 * i + 1]); }
template <int VEC>
__device__ __forceinline__ void put(float (&a)[VEC], int i, float2 v) {
  a[2 * i] = v.x;
  a[2 * i + 1] = v.y;
}
// a = a * b
template <int VEC>
__device__ __forceinline__ void times(float (&a)[VEC], const float (&b)[VEC]) {
  if constexpr (VEC == 1) a[0] *= b[0];
  else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) put(a, i, mul2(pair(a, i), pair(b, i)));
  }
}
// acc += a * b, element by element
template <int VEC>
__device__ __forceinline__ void add_products(float (&acc)[VEC], const float (&a)[VEC], const float (&b)[VEC]) {
  if constexpr (VEC == 1) acc[0] = fmaf(a[0], b[0], acc[0]);
  else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) put(acc, i, fma2(pair(a, i), pair(b, i), pair(acc, i)));
  }
}
template <int VEC>
__device__ __forceinline__ void scale(float (&a)[VEC], float f) {
  float v[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = f;
  times(a, v);
}
template <int VEC>
__device__ __forceinline__ float total(const float (&a)[VEC]) {
  float t = a[0];
#pragma unroll
  for (int k = 1; k < VEC; ++k) t += a[k];
  return t;
}

template <int VEC, bool INTER>
__device__ __forceinline__ void turn(float (&a)[VEC], float (&b)[VEC], const float (&c)[VEC], const float (&s)[VEC]) {
  if constexpr (VEC == 1) {
    const float x = a[0], y = b[0];
    a[0] = x * c[0] - y * s[0];
    b[0] = y * c[0] + x * s[0];
  } else if constexpr (!INTER) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 x = pair(a, i), y = pair(b, i), cc = pair(c, i), ss = pair(s, i);
      put(a, i, fma2(y, make_float2(-ss.x, -ss.y), mul2(x, cc)));
      put(b, i, fma2(x, ss, mul2(y, cc)));
    }
  } else {
    // the unit is one run of 2 VEC elements: pair i is (2i, 2i + 1)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float(&v)[VEC] = 2 * i < VEC ? a : b;
      const int k = i % (VEC / 2);
      const float2 x = pair(v, k);
      put(v, k, fma2(make_float2(x.y, x.x), make_float2(-s[i], s[i]), mul2(x, both(c[i]))));
    }
  }
}

// A group's way through its heads: item after item, the heads of an item in turn.
struct Cursor {
  unsigned item, token;
  int i, h0, hn;            // head within the item; the item's first head and number of heads (0: no item)
  long long x_at, g_at;     // the token's place
  unsigned b, l;
  __device__ __forceinline__ void enter(const Args& p, const Side& sd, unsigned at) {
    item = at;
    i = 0;
    hn = 0;
    token = b = l = 0;
    h0 = 0;
    if (at < sd.items) {
      token = at / (unsigned)sd.items_per_token;
      h0 = (int)(at % (unsigned)sd.items_per_token) * sd.heads_per_item;
      hn = min(sd.heads_per_item, sd.heads - h0);
      b = token / p.L;
      l = token % p.L;
    }
    x_at = b * sd.xs_b + l * sd.xs_l;
    g_at = b * sd.gs_b + l * sd.gs_l;
  }
  // returns whether a new item has begun
  __device__ __forceinline__ bool advance(const Args& p, const Side& sd, unsigned stride) {
    if (++i < sd.heads_per_item) return false;
    enter(p, sd, item < sd.items ? item + stride : item);
    return true;
  }
};

constexpr int ring_depth(bool bwd) { return bwd ? 3 : 4; }
constexpr int resident_blocks(int ch, bool bwd) { return ch > 1 ? 1 : (bwd ? 2 : 3); }

template <typename T, int VEC, int CH, bool INTER, bool BWD>
__global__ void __launch_bounds__(kThreads, resident_blocks(CH, BWD)) qk_norm_rotary_kernel(const __grid_constant__ Args p) {
  // heads on their way: each thread copies its vectors of the next heads to a place of its own.  Behind the last head: partial dw.
  extern __shared__ __align__(16) unsigned char shared[];
  using V = Pack<T, VEC>;
  constexpr bool kAsync = sizeof(V) >= 4;
  constexpr int kDepth = ring_depth(BWD), kPerHead = CH * 2 * (BWD ? 2 : 1);
  const bool keys = blockIdx.x >= (unsigned)p.side[0].blocks;
  const Side& sd = p.side[keys ? 1 : 0];
  const unsigned block = keys ? blockIdx.x - p.side[0].blocks : blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = p.group, gl = threadIdx.x & (G - 1);
  const unsigned groups_per_block = kThreads / G;
  const int units = p.D / (2 * VEC);
  const T* x = static_cast<const T*>(sd.x);
  const T* dy = static_cast<const T*>(sd.dy);
  T* out = static_cast<T*>(sd.out);
  const float inv_d = 1.f / (float)p.D;

  int lo[CH], hi[CH];
  bool rot[CH], on[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int u = gl + c * G;
    on[c] = u < units;
    place<VEC, INTER>(on[c] ? u : 0, p.R, lo[c], hi[c], rot[c]);
  }

  // All groups of a warp run the same number of rounds, since the reductions take the whole warp.
  const unsigned stride = (unsigned)sd.blocks * groups_per_block;
  const unsigned first = block * groups_per_block + threadIdx.x / G;
  const unsigned warp_first = block * groups_per_block + (threadIdx.x & ~31u) / G;
  V* ring = reinterpret_cast<V*>(shared) + threadIdx.x;
  Cursor ahead;
  ahead.enter(p, sd, first);
  auto fetch = [&](int stage) {
    if (kAsync) {
      const bool there = ahead.i < ahead.hn;
      const int h = ahead.h0 + (there ? ahead.i : 0);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        V* slot = ring + (stage * kPerHead + c * (BWD ? 4 : 2)) * kThreads;
        const T* xh = x + ahead.x_at + h * sd.xs_h;
        copy_async<kAsync ? sizeof(V) : 4>(slot, xh + lo[c], there && on[c]);
        copy_async<kAsync ? sizeof(V) : 4>(slot + kThreads, xh + hi[c], there && on[c]);
        if (BWD) {
          const T* gh = dy + ahead.g_at + h * sd.gs_h;
          copy_async<kAsync ? sizeof(V) : 4>(slot + 2 * kThreads, gh + lo[c], there && on[c]);
          copy_async<kAsync ? sizeof(V) : 4>(slot + 3 * kThreads, gh + hi[c], there && on[c]);
        }
      }
      ahead.advance(p, sd, stride);
    }
    copies_commit();
  };
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fetch(d);

  float wl[CH][VEC], wh[CH][VEC];
  float dl[CH][VEC], dh[CH][VEC];  // backward: this lane's part of dw
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      wl[c][k] = sd.weight ? weight_at(sd.weight, sd.weight_dtype, lo[c] + k) : 1.f;
      wh[c][k] = sd.weight ? weight_at(sd.weight, sd.weight_dtype, hi[c] + k) : 1.f;
      dl[c][k] = dh[c][k] = 0.f;
    }
  }

  Cursor now;
  int stage = 0;
  for (unsigned long long base = warp_first, item = first; base < sd.items; base += stride, item += stride) {
    now.enter(p, sd, item < sd.items ? (unsigned)item : sd.items);
    long long pos = now.l;
    if (p.positions) {
      const long long at = now.b * p.pos_b + now.l * p.pos_l;
      pos = p.pos_is_64 ? static_cast<const long long*>(p.positions)[at] : (long long)static_cast<const int*>(p.positions)[at];
    }
    const bool inside = now.hn > 0 && pos >= 0 && pos < p.table_rows;
    if (now.hn > 0 && pos >= p.table_rows && p.bad_flag && gl == 0) *p.bad_flag = 1;
    float cs[CH][VEC], sn[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) { cs[c][k] = 1.f; sn[c][k] = 0.f; }
      if (inside && on[c] && rot[c]) {
        const long long at = pos * (p.R / 2) + (INTER ? lo[c] / 2 : lo[c]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          cs[c][k] = __ldg(p.cos + at + k);
          sn[c][k] = BWD ? -__ldg(p.sin + at + k) : __ldg(p.sin + at + k);
        }
      }
    }
    T* ot = out + ((long long)now.token * sd.heads + now.h0) * p.D;
    for (int i = 0; i < sd.heads_per_item; ++i, ot += p.D) {
      const bool act = i < now.hn;
      fetch(stage == 0 ? kDepth - 1 : stage - 1);
      copies_wait<kDepth - 1>();
      V raw[CH][BWD ? 4 : 2];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int n = 0; n < (BWD ? 4 : 2); ++n) {
          if (kAsync) {
            raw[c][n] = ring[(stage * kPerHead + c * (BWD ? 4 : 2) + n) * kThreads];
          } else {
            const T* from = n < 2 ? x + now.x_at + (now.h0 + i) * sd.xs_h : dy + now.g_at + (now.h0 + i) * sd.gs_h;
            if (act && on[c]) raw[c][n] = *reinterpret_cast<const V*>(from + (n % 2 ? hi[c] : lo[c]));
          }
          if (!inside || (!kAsync && !(act && on[c]))) {  // what a token outside the tables holds counts for nothing
#pragma unroll
            for (int k = 0; k < VEC; ++k) raw[c][n].v[k] = from_f32<T>(0.f);
          }
        }
      }
      stage = stage == kDepth - 1 ? 0 : stage + 1;
      float a[CH][VEC], z[CH][VEC], sq[VEC], dt[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) sq[k] = dt[k] = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        unpack(raw[c][0], a[c]);
        unpack(raw[c][1], z[c]);
        add_products(sq, a[c], a[c]);
        add_products(sq, z[c], z[c]);
      }
      if (!BWD) {
        const float r = rsqrtf(group_sum(total(sq), G) * inv_d + p.eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          scale(a[c], inside ? r : 0.f);
          scale(z[c], inside ? r : 0.f);
          times(a[c], wl[c]);
          times(z[c], wh[c]);
          turn<VEC, INTER>(a[c], z[c], cs[c], sn[c]);
          if (act && on[c]) {
            store<T, VEC>(ot + lo[c], a[c]);
            store<T, VEC>(ot + hi[c], z[c]);
          }
        }
      } else {
        float ga[CH][VEC], gz[CH][VEC];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          unpack(raw[c][2], ga[c]);
          unpack(raw[c][3], gz[c]);
          turn<VEC, INTER>(ga[c], gz[c], cs[c], sn[c]);
        }
        float ss = total(sq);
        for (int o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = act && inside ? rsqrtf(ss * inv_d + p.eps) : 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          scale(a[c], r);  // the normalised head
          scale(z[c], r);
          add_products(dl[c], ga[c], a[c]);
          add_products(dh[c], gz[c], z[c]);
          times(ga[c], wl[c]);
          times(gz[c], wh[c]);
          add_products(dt, ga[c], a[c]);
          add_products(dt, gz[c], z[c]);
        }
        const float m = -group_sum(total(dt), G) * inv_d;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float v[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[k] = m;
          add_products(ga[c], a[c], v);
          add_products(gz[c], z[c], v);
          scale(ga[c], r);
          scale(gz[c], r);
          if (act && on[c]) {
            store<T, VEC>(ot + lo[c], ga[c]);
            store<T, VEC>(ot + hi[c], gz[c]);
          }
        }
      }
    }
  }

  if (BWD && sd.dw_partial) {
    // the groups of a warp, then the warps, in a fixed order: the same inputs give the same bits
    copies_wait<0>();
    __syncthreads();
    float* sh_dw = reinterpret_cast<float*>(shared);  // [warps][D]
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float u = dl[c][k], v = dh[c][k];
        for (int o = G; o < 32; o <<= 1) {
          u += __shfl_xor_sync(0xffffffffu, u, o);
          v += __shfl_xor_sync(0xffffffffu, v, o);
        }
        if (lane < G && on[c]) {
          sh_dw[warp * p.D + lo[c] + k] = u;
          sh_dw[warp * p.D + hi[c] + k] = v;
        }
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += kThreads) {
      float s = 0.f;
      for (int w = 0; w < kThreads / 32; ++w) s += sh_dw[w * p.D + d];
      sd.dw_partial[(long long)block * p.D + d] = s;
    }
  }
}

// dw[d] = sum over blocks of partial[block][d], in a fixed order; grid.y: queries, keys.  Some hundred rows of partial sums: 32 of
// them side by side with several loads under way, since this is latency and nothing else.
__global__ void __launch_bounds__(1024) qk_dweight_kernel(const float* pq, int nq, void* dq, int dtq, const float* pk, int nk, void* dk,
                                                          int dtk, int D) {
  __shared__ float sh[32][33];
  const float* part = blockIdx.y ? pk : pq;
  const int n = blockIdx.y ? nk : nq, dt = blockIdx.y ? dtk : dtq;
  void* out = blockIdx.y ? dk : dq;
  if (!out) return;
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int i = row; i < n; i += 32) s += part[(long long)i * D + d];
  }
  sh[row][lane] = s;
  __syncthreads();
  s = group_sum(sh[lane][row], 32);  // warp `row` adds column `row`
  const int e = blockIdx.x * 32 + row;
  if (lane == 0 && e < D) {
    if (dt == B200_F32) static_cast<float*>(out)[e] = s;
    else if (dt == B200_BF16) static_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16(s);
    else static_cast<__half*>(out)[e] = __float2half(s);
  }
}

// The widest vector (at most 16 bytes) that divides the halves, the heads and every stride and address.
int vector_width(const B200QkNormRotary& p, bool bwd) {
  const int es = p.dtype == B200_F32 ? 4 : 2;
  for (int v = 16 / es; v > 1; v >>= 1) {
    bool ok = p.D % (2 * v) == 0 && (p.interleaved ? p.R % (2 * v) == 0 : (p.R % (2 * v) == 0 && (p.D - p.R) % (2 * v) == 0));
    for (int s = 0; ok && s < 2; ++s) {
      const B200QkSide& q = p.side[s];
      for (int i = 0; i < 3; ++i) ok = ok && q.x_stride[i] % v == 0 && (!bwd || q.dy_stride[i] % v == 0);
      ok = ok && (uintptr_t)q.x % (v * es) == 0 && (uintptr_t)q.out % (v * es) == 0 && (!bwd || (uintptr_t)q.dy % (v * es) == 0);
    }
    if (ok) return v;
  }
  return 1;
}

int power_of_two_at_least(int n, int most) {
  int g = 1;
  while (g < n && g < most) g <<= 1;
  return g;
}

struct Plan {
  Args a;
  int vec, ch, grid;
};

// The same plan for the launch and for the workspace size.
Plan make_plan(const B200QkNormRotary& p, bool bwd) {
  Plan pl{};
  Args& a = pl.a;
  pl.vec = vector_width(p, bwd);
  const int units = p.D / (2 * pl.vec);
  a.group = power_of_two_at_least(units, 32);
  pl.ch = (units + a.group - 1) / a.group;
  a.cos = p.cos; a.sin = p.sin; a.positions = p.positions; a.pos_b = p.pos_stride[0]; a.pos_l = p.pos_stride[1];
  a.pos_is_64 = p.positions_dtype == B200_I64; a.table_rows = p.table_rows; a.bad_flag = p.bad_flag;
  a.L = (unsigned)p.L; a.D = p.D; a.R = p.R; a.eps = p.eps;
  const long long tokens = p.B * p.L, heads = (long long)p.side[0].heads + p.side[1].heads;
  // Heads per item, which share a token's cos / sin and place: as many as leave every SM 512 threads, at most eight.
  int hpi = 1;
  while (hpi < 8 && tokens * heads / (hpi * 2) * a.group >= 148LL * 512) hpi *= 2;
  const long long per_block = kThreads / a.group, resident = 148 * resident_blocks(pl.ch, bwd);
  for (int s = 0; s < 2; ++s) {
    const B200QkSide& q = p.side[s];
    Side& d = a.side[s];
    d.x = q.x; d.dy = q.dy; d.out = q.out; d.weight = q.weight; d.weight_dtype = q.weight_dtype; d.heads = q.heads;
    d.xs_b = q.x_stride[0]; d.xs_l = q.x_stride[1]; d.xs_h = q.x_stride[2];
    d.gs_b = q.dy_stride[0]; d.gs_l = q.dy_stride[1]; d.gs_h = q.dy_stride[2];
    if (q.heads == 0) continue;
    d.heads_per_item = hpi < q.heads ? hpi : q.heads;
    d.items_per_token = (q.heads + d.heads_per_item - 1) / d.heads_per_item;
    d.items = (unsigned)(tokens * d.items_per_token);
    // one wave of blocks, shared out by the number of heads
    const long long blocks = (d.items + per_block - 1) / per_block, share = (resident * q.heads + heads - 1) / heads;
    d.blocks = (int)(blocks < share ? blocks : share);
    pl.grid += d.blocks;
  }
  return pl;
}

template <typename T, int VEC, int CH, bool INTER, bool BWD>
int launch_one(const Plan& pl, cudaStream_t s) {
  size_t smem = (size_t)ring_depth(BWD) * CH * 2 * (BWD ? 2 : 1) * kThreads * sizeof(T) * VEC;
  const size_t dw = BWD ? (size_t)(kThreads / 32) * pl.a.D * sizeof(float) : 0;
  if (smem < dw) smem = dw;
  auto kernel = qk_norm_rotary_kernel<T, VEC, CH, INTER, BWD>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
  }
  kernel<<<pl.grid, kThreads, smem, s>>>(pl.a);
  return (int)cudaGetLastError();
}
template <typename T, int VEC, int CH, bool BWD>
int launch(const Plan& pl, bool interleaved, cudaStream_t s) {
  return interleaved ? launch_one<T, VEC, CH, true, BWD>(pl, s) : launch_one<T, VEC, CH, false, BWD>(pl, s);
}
template <typename T, int WIDEST, bool BWD>
int dispatch(const Plan& pl, bool interleaved, cudaStream_t s) {
  // units of one head: D / (2 VEC) over at most 32 lanes, D at most 512
  if (pl.vec == 8 && WIDEST == 8) return launch<T, WIDEST == 8 ? 8 : 4, 1, BWD>(pl, interleaved, s);
  if (pl.vec == 4 && pl.ch == 1) return launch<T, 4, 1, BWD>(pl, interleaved, s);
  if (pl.vec == 4) return launch<T, 4, 2, BWD>(pl, interleaved, s);
  if (pl.vec == 2 && pl.ch == 1) return launch<T, 2, 1, BWD>(pl, interleaved, s);
  if (pl.vec == 2) return launch<T, 2, 4, BWD>(pl, interleaved, s);
  if (pl.ch == 1) return launch<T, 1, 1, BWD>(pl, interleaved, s);
  return launch<T, 1, 8, BWD>(pl, interleaved, s);
}

bool valid(const B200QkNormRotary* p) {
  if (p->D <= 0 || p->D % 2 || p->D > B200_QK_MAX_HEAD_DIM || p->R < 0 || p->R % 2 || p->R > p->D) return false;
  for (int s = 0; s < 2; ++s)
    if (p->side[s].heads < 0 || p->B * p->L * (long long)p->side[s].heads >= (1LL << 31)) return false;
  return true;
}

}  // namespace

extern "C" long long b200_qk_norm_rotary_workspace(const B200QkNormRotary* p) {
  if (!valid(p) || p->B * p->L <= 0) return 0;
  return (long long)make_plan(*p, true).grid * p->D * sizeof(float);
}

extern "C" int b200_qk_norm_rotary_fwd(const B200QkNormRotary* p, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  if (p->B * p->L <= 0) return 0;
  const Plan pl = make_plan(*p, false);
  if (pl.grid == 0) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (p->dtype == B200_BF16) return dispatch<__nv_bfloat16, 8, false>(pl, p->interleaved, s);
  if (p->dtype == B200_F16) return dispatch<__half, 8, false>(pl, p->interleaved, s);
  if (p->dtype == B200_F32) return dispatch<float, 4, false>(pl, p->interleaved, s);
  return (int)cudaErrorInvalidValue;
}

extern "C" int b200_qk_norm_rotary_bwd(const B200QkNormRotary* p, void* workspace, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  cudaStream_t s = (cudaStream_t)stream;
  Plan pl = p->B * p->L > 0 ? make_plan(*p, true) : Plan{};
  float* ws = static_cast<float*>(workspace);
  for (int i = 0; i < 2; ++i) {
    if (p->side[i].dweight) pl.a.side[i].dw_partial = ws;
    ws += (long long)pl.a.side[i].blocks * p->D;
  }
  if (pl.grid > 0) {
    int rc;
    if (p->dtype == B200_BF16) rc = dispatch<__nv_bfloat16, 8, true>(pl, p->interleaved, s);
    else if (p->dtype == B200_F16) rc = dispatch<__half, 8, true>(pl, p->interleaved, s);
    else if (p->dtype == B200_F32) rc = dispatch<float, 4, true>(pl, p->interleaved, s);
    else rc = (int)cudaErrorInvalidValue;
    if (rc) return rc;
  }
  if (p->side[0].dweight || p->side[1].dweight) {
    qk_dweight_kernel<<<dim3((p->D + 31) / 32, 2), 1024, 0, s>>>(
        pl.a.side[0].dw_partial, pl.a.side[0].blocks, p->side[0].dweight, p->side[0].weight_dtype, pl.a.side[1].dw_partial,
        pl.a.side[1].blocks, p->side[1].dweight, p->side[1].weight_dtype, p->D);
  }
  return (int)cudaGetLastError();
}
