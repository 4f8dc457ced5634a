// Softmax over attention scores with a learned relative position bias, a scale and a mask, forward and backward.
//
//   a_ij = scale s_ij + table[bucket(j - i - offset)][h] + mask_ij        p = softmax over j
//   backward: d_ij = p_ij (g_ij - sum_j p_ij g_ij);  ds = scale d;  dtable[b][h] = sum of d over the pairs (i, j) of bucket b
//   a row whose a are all -inf (the mask leaves nothing) has p = 0 and d = 0
//
// Bound by memory: forward reads s and writes p; backward reads s and g and writes ds.  The bias is never written out as
// [heads, Lq, Lk]: it depends on the distance alone and is the same for all distances from `reach` (at most max_distance) on,
// so a block, which works on one head, keeps the 2 reach + 1 values it can take in shared memory.  The backward recomputes p from s
// and two numbers a row (maximum and 1 / sum, fp32): reading s costs what reading p would, and p is not rounded in between.
//
// Table gradient: d is summed over distances first.  Far distances go to two registers a thread; near ones to shared memory, in a copy
// for every group of lanes that walks over rows of its own.  In one row no two elements have the same distance, so no atomics
// are needed and the order of every sum is fixed: the same inputs give the same bits.
#include "kernels_api.h"
#include "row_vec.cuh"

namespace {

using namespace rowvec;

constexpr int kMaxThreads = 256;
constexpr float kNegInf = -__builtin_huge_valf();

struct Args {
  const void* s;
  const void* g;        // backward: gradient of p
  void* out;            // p or ds
  float2* stats;        // (maximum, 1 / sum) of each row; forward: may be null
  float* partial;       // backward: [H][blocks_per_head][2 reach + 1], or null
  const void* table;
  const void* mask;     // or null
  long long st_b, st_h, st_i;     // of s, g and out (their last dimension is dense)
  long long mk_b, mk_h, mk_i, mk_j;
  int table_dtype, mask_dtype;
  int H, Lq, Lk, reach, offset;
  unsigned rows;        // of one head: B * Lq
  unsigned rows_per_block;
  int blocks_per_head, group;
  float scale;
  B200RelativeBuckets rb;
};

__device__ __forceinline__ float scalar_at(const void* p, long long i, int dt) {
  if (dt == B200_F32) return static_cast<const float*>(p)[i];
  if (dt == B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dt == B200_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const unsigned char*>(p)[i] ? 0.f : kNegInf;  // bool: true keeps
}

__device__ __forceinline__ int bucket_of(int rel, const B200RelativeBuckets& rb) {
  int d = -rel, up = 0;
  if (rb.bidirectional) {
    up = rel > 0 ? rb.per_side : 0;
    d = abs(rel);
  }
  if (d < rb.exact) return up + max(d, 0);
  int b = rb.exact;
  for (int k = 1; k < rb.per_side - rb.exact; ++k) b += d >= rb.first[k] ? 1 : 0;
  return up + b;
}

// One pad word every 32: lanes that read eight neighbours each then meet in different banks.
__device__ __forceinline__ int padded(int x) { return x + (x >> 5); }

__device__ __forceinline__ void fill_lut(float* lut, const Args& p, int h) {
  for (int x = threadIdx.x; x <= 2 * p.reach; x += blockDim.x)
    lut[padded(x)] = scalar_at(p.table, (long long)bucket_of(x - p.reach, p.rb) * p.H + h, p.table_dtype);
}

// The elements [j0, j0 + VEC) of a row; those outside [0, n) are left alone.  A vector lies on a 16-byte boundary.
template <typename T, int VEC>
__device__ __forceinline__ void load_part(const T* row, int j0, int n, float (&v)[VEC]) {
  if (j0 >= 0 && j0 + VEC <= n) {
    load<T, VEC>(row + j0, v);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = j0 + k >= 0 && j0 + k < n ? to_f32<T>(row[j0 + k]) : 0.f;
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_part(T* row, int j0, int n, const float (&v)[VEC]) {
  if (j0 >= 0 && j0 + VEC <= n) {
    store<T, VEC>(row + j0, v);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (j0 + k >= 0 && j0 + k < n) row[j0 + k] = from_f32<T>(v[k]);
  }
}

template <typename M, int VEC>
__device__ __forceinline__ void add_mask_vector(const M* m, float (&a)[VEC]) {
  float v[VEC];
  constexpr int W = 16 / sizeof(M) < VEC ? 16 / sizeof(M) : VEC;
#pragma unroll
  for (int o = 0; o < VEC; o += W) {
    float part[W];
    load<M, W>(m + o, part);
#pragma unroll
    for (int k = 0; k < W; ++k) v[o + k] = part[k];
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) a[k] = v[k] == kNegInf ? kNegInf : a[k] + v[k];
}

// Adds the mask to the scores of [j0, j0 + VEC); excluded elements become -inf whatever they held, NaN too.
template <int VEC>
__device__ __forceinline__ void add_mask(const Args& p, long long row, int j0, float (&a)[VEC]) {
  const long long at = row + (long long)j0 * p.mk_j;
  if (p.mk_j == 1 && j0 >= 0 && j0 + VEC <= p.Lk) {
    const int es = p.mask_dtype == B200_F32 ? 4 : (p.mask_dtype == B200_BF16 || p.mask_dtype == B200_F16 ? 2 : 1);
    const char* m = static_cast<const char*>(p.mask) + at * es;
    const int bytes = VEC * es < 16 ? VEC * es : 16;
    if ((reinterpret_cast<uintptr_t>(m) & (bytes - 1)) == 0) {
      if (es == 4) { add_mask_vector<float, VEC>(reinterpret_cast<const float*>(m), a); return; }
      if (p.mask_dtype == B200_BF16) { add_mask_vector<__nv_bfloat16, VEC>(reinterpret_cast<const __nv_bfloat16*>(m), a); return; }
      if (p.mask_dtype == B200_F16) { add_mask_vector<__half, VEC>(reinterpret_cast<const __half*>(m), a); return; }
      const Pack<unsigned char, VEC> keep = *reinterpret_cast<const Pack<unsigned char, VEC>*>(m);
#pragma unroll
      for (int k = 0; k < VEC; ++k) a[k] = keep.v[k] ? a[k] : kNegInf;
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    if (j0 + k >= 0 && j0 + k < p.Lk) {
      const float v = scalar_at(p.mask, at + k * p.mk_j, p.mask_dtype);
      a[k] = v == kNegInf ? kNegInf : a[k] + v;
    }
  }
}

// Scores to logits: scale, bias by distance, mask; -inf outside the row.  x0 = distance of the first element + reach.
template <int VEC>
__device__ __forceinline__ void to_logits(const Args& p, const float* lut, long long mask_row, int j0, int x0, float (&a)[VEC]) {
  const int last = 2 * p.reach;
  if (x0 >= last || x0 + VEC - 1 <= 0) {  // all as far as the bias tells apart
    const float b = lut[padded(x0 > 0 ? last : 0)];
#pragma unroll
    for (int k = 0; k < VEC; ++k) a[k] = fmaf(a[k], p.scale, b);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) a[k] = fmaf(a[k], p.scale, lut[padded(min(max(x0 + k, 0), last))]);
  }
  if (p.mask) add_mask<VEC>(p, mask_row, j0, a);
  if (j0 < 0 || j0 + VEC > p.Lk) {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (j0 + k < 0 || j0 + k >= p.Lk) a[k] = kNegInf;
  }
}

__device__ __forceinline__ float weight_of(float a, float m) { return a == kNegInf ? 0.f : __expf(a - m); }

// d to the table gradient's sums over distances
template <int VEC>
__device__ __forceinline__ void add_distances(float* acc, int last, int x0, const float (&d)[VEC], float& below, float& above) {
  if (x0 >= last || x0 + VEC - 1 <= 0) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) t += d[k];
    if (x0 > 0) above += t; else below += t;
    return;
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int x = x0 + k;
    if (x <= 0) below += d[k];
    else if (x >= last) above += d[k];
    else acc[padded(x)] += d[k];
  }
}

struct RowAt {
  long long at, mask_row;
  long long stat;
  int first_x;  // distance of key 0 plus reach
};
__device__ __forceinline__ RowAt row_at(const Args& p, unsigned r, int h) {
  const unsigned b = r / (unsigned)p.Lq, i = r % (unsigned)p.Lq;
  RowAt w;
  w.at = b * p.st_b + h * p.st_h + i * p.st_i;
  w.mask_row = b * p.mk_b + h * p.mk_h + i * p.mk_i;
  w.stat = ((long long)b * p.H + h) * p.Lq + i;
  w.first_x = p.reach - p.offset - (int)i;
  return w;
}

// A row to a group of lanes, in registers: NV vectors of VEC elements for each lane.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kMaxThreads) bias_softmax_fwd_rows(const __grid_constant__ Args p) {
  extern __shared__ float lut[];
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  fill_lut(lut, p, h);
  __syncthreads();
  const int G = p.group, gl = threadIdx.x & (G - 1), groups = blockDim.x / G;
  const unsigned r0 = part * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
  for (unsigned base = r0; base < r1; base += groups) {
    const unsigned r = base + threadIdx.x / G;
    const bool live = r < r1;
    const RowAt w = row_at(p, live ? r : r0, h);
    const T* s = static_cast<const T*>(p.s) + w.at;
    const int phase = (int)((reinterpret_cast<uintptr_t>(s) / sizeof(T)) & (VEC - 1));
    float a[NV][VEC], m = kNegInf;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * G) * VEC - phase;
      if (j0 < p.Lk) load_part<T, VEC>(s, j0, p.Lk, a[n]);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * G) * VEC - phase;
      if (j0 < p.Lk) {
        to_logits<VEC>(p, lut, w.mask_row, j0, w.first_x + j0, a[n]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = fmaxf(m, a[n][k]);
      }
    }
    m = group_max(m, G);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if ((gl + n * G) * VEC - phase < p.Lk) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          a[n][k] = weight_of(a[n][k], m);
          sum += a[n][k];
        }
      }
    }
    sum = group_sum(sum, G);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (!live) continue;
    T* o = static_cast<T*>(p.out) + w.at;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * G) * VEC - phase;
      if (j0 < p.Lk) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) a[n][k] *= inv;
        store_part<T, VEC>(o, j0, p.Lk, a[n]);
      }
    }
    if (p.stats && gl == 0) p.stats[w.stat] = make_float2(m, inv);
  }
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kMaxThreads) bias_softmax_bwd_rows(const __grid_constant__ Args p) {
  extern __shared__ float lut[];
  const int last = 2 * p.reach, words = padded(last) + 1;
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  const int G = p.group, gl = threadIdx.x & (G - 1), groups = blockDim.x / G;
  float* all = lut + words;
  float* acc = all + (threadIdx.x / G) * words;
  fill_lut(lut, p, h);
  if (p.partial)
    for (int x = threadIdx.x; x < groups * words; x += blockDim.x) all[x] = 0.f;
  __syncthreads();
  float below = 0.f, above = 0.f;
  const unsigned r0 = part * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
  for (unsigned base = r0; base < r1; base += groups) {
    const unsigned r = base + threadIdx.x / G;
    const bool live = r < r1;
    const RowAt w = row_at(p, live ? r : r0, h);
    const T* s = static_cast<const T*>(p.s) + w.at;
    const T* g = static_cast<const T*>(p.g) + w.at;
    const int phase = (int)((reinterpret_cast<uintptr_t>(s) / sizeof(T)) & (VEC - 1));
    const float2 st = p.stats[w.stat];
    float a[NV][VEC], d[NV][VEC], dot = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * G) * VEC - phase;
      if (j0 < p.Lk) {
        load_part<T, VEC>(s, j0, p.Lk, a[n]);
        load_part<T, VEC>(g, j0, p.Lk, d[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * G) * VEC - phase;
      if (j0 < p.Lk) {
        to_logits<VEC>(p, lut, w.mask_row, j0, w.first_x + j0, a[n]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          a[n][k] = weight_of(a[n][k], st.x) * st.y;
          dot += a[n][k] == 0.f ? 0.f : a[n][k] * d[n][k];  // an excluded key counts nothing, whatever its gradient holds
        }
      }
    }
    dot = group_sum(dot, G);
    if (live) {
      T* o = static_cast<T*>(p.out) + w.at;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int j0 = (gl + n * G) * VEC - phase;
        if (j0 < p.Lk) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            d[n][k] = a[n][k] == 0.f ? 0.f : a[n][k] * (d[n][k] - dot);
            a[n][k] = d[n][k] * p.scale;
          }
          store_part<T, VEC>(o, j0, p.Lk, a[n]);
          if (p.partial) add_distances<VEC>(acc, last, w.first_x + j0, d[n], below, above);
        }
      }
    }
    __syncwarp();  // the next row of this group adds to the same sums from other lanes
  }
  if (!p.partial) return;
  below = group_sum(below, G);
  above = group_sum(above, G);
  if (gl == 0) {  // the slots of the two ends are used for nothing else
    acc[padded(0)] = below;
    acc[padded(last)] += above;  // reach 0: both ends are one slot
  }
  __syncthreads();
  float* out = p.partial + ((long long)h * p.blocks_per_head + part) * (last + 1);
  for (int x = threadIdx.x; x <= last; x += blockDim.x) {
    float t = 0.f;
    for (int q = 0; q < groups; ++q) t += all[q * words + padded(x)];
    out[x] = t;
  }
}

// A row to a whole block, any length: two passes over the row, of which the second finds it in the caches.
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = group_sum(v, 32);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = group_sum(threadIdx.x % 32 < blockDim.x / 32 ? sh[threadIdx.x % 32] : 0.f, 32);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_max(float v, float* sh) {
  v = group_max(v, 32);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = group_max(threadIdx.x % 32 < blockDim.x / 32 ? sh[threadIdx.x % 32] : kNegInf, 32);
  __syncthreads();
  return v;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kMaxThreads) bias_softmax_fwd_long(const __grid_constant__ Args p) {
  extern __shared__ float lut[];
  __shared__ float sh[32];
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  fill_lut(lut, p, h);
  __syncthreads();
  const unsigned r0 = part * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
  for (unsigned r = r0; r < r1; ++r) {
    const RowAt w = row_at(p, r, h);
    const T* s = static_cast<const T*>(p.s) + w.at;
    const int phase = (int)((reinterpret_cast<uintptr_t>(s) / sizeof(T)) & (VEC - 1));
    float m = kNegInf, sum = 0.f;
    for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.Lk; j0 += blockDim.x * VEC) {
      float a[VEC], top = kNegInf;
      load_part<T, VEC>(s, j0, p.Lk, a);
      to_logits<VEC>(p, lut, w.mask_row, j0, w.first_x + j0, a);
#pragma unroll
      for (int k = 0; k < VEC; ++k) top = fmaxf(top, a[k]);
      if (top > m) {
        sum *= __expf(m - top);  // m = -inf: 0
        m = top;
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum += weight_of(a[k], m);
    }
    const float all = block_max(m, sh);
    sum = block_sum(m == kNegInf ? sum : sum * __expf(m - all), sh);  // m = -inf: 0, or NaN from a NaN score
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* o = static_cast<T*>(p.out) + w.at;
    for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.Lk; j0 += blockDim.x * VEC) {
      float a[VEC];
      load_part<T, VEC>(s, j0, p.Lk, a);
      to_logits<VEC>(p, lut, w.mask_row, j0, w.first_x + j0, a);
#pragma unroll
      for (int k = 0; k < VEC; ++k) a[k] = weight_of(a[k], all) * inv;
      store_part<T, VEC>(o, j0, p.Lk, a);
    }
    if (p.stats && threadIdx.x == 0) p.stats[w.stat] = make_float2(all, inv);
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kMaxThreads) bias_softmax_bwd_long(const __grid_constant__ Args p) {
  extern __shared__ float lut[];
  __shared__ float sh[32];
  const int last = 2 * p.reach, words = padded(last) + 1;
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  float* acc = lut + words;
  fill_lut(lut, p, h);
  if (p.partial)
    for (int x = threadIdx.x; x < words; x += blockDim.x) acc[x] = 0.f;
  __syncthreads();
  float below = 0.f, above = 0.f;
  const unsigned r0 = part * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
  for (unsigned r = r0; r < r1; ++r) {
    const RowAt w = row_at(p, r, h);
    const T* s = static_cast<const T*>(p.s) + w.at;
    const T* g = static_cast<const T*>(p.g) + w.at;
    const int phase = (int)((reinterpret_cast<uintptr_t>(s) / sizeof(T)) & (VEC - 1));
    const float2 st = p.stats[w.stat];
    float dot = 0.f;
    for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.Lk; j0 += blockDim.x * VEC) {
      float a[VEC], d[VEC];
      load_part<T, VEC>(s, j0, p.Lk, a);
      load_part<T, VEC>(g, j0, p.Lk, d);
      to_logits<VEC>(p, lut, w.mask_row, j0, w.first_x + j0, a);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float q = weight_of(a[k], st.x) * st.y;
        dot += q == 0.f ? 0.f : q * d[k];
      }
    }
    dot = block_sum(dot, sh);  // its barriers also order this row's sums over distances behind the last row's
    T* o = static_cast<T*>(p.out) + w.at;
    for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.Lk; j0 += blockDim.x * VEC) {
      float a[VEC], d[VEC];
      load_part<T, VEC>(s, j0, p.Lk, a);
      load_part<T, VEC>(g, j0, p.Lk, d);
      to_logits<VEC>(p, lut, w.mask_row, j0, w.first_x + j0, a);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float q = weight_of(a[k], st.x) * st.y;
        d[k] = q == 0.f ? 0.f : q * (d[k] - dot);
        a[k] = d[k] * p.scale;
      }
      store_part<T, VEC>(o, j0, p.Lk, a);
      if (p.partial) add_distances<VEC>(acc, last, w.first_x + j0, d, below, above);
    }
  }
  if (!p.partial) return;
  below = block_sum(below, sh);
  above = block_sum(above, sh);
  if (threadIdx.x == 0) {
    acc[padded(0)] = below;
    acc[padded(last)] += above;
  }
  __syncthreads();
  float* out = p.partial + ((long long)h * p.blocks_per_head + part) * (last + 1);
  for (int x = threadIdx.x; x <= last; x += blockDim.x) out[x] = acc[padded(x)];
}

// One block per head and bucket: sums over the blocks' partial sums for the distances of the bucket, in a fixed order.  A
// bucket's distances are neighbours, so its slots are one run [x0, x1].
__global__ void __launch_bounds__(kMaxThreads) bias_table_grad(const float* partial, int blocks, int reach, const __grid_constant__ B200RelativeBuckets rb,
                                                               int H, void* out, int dtype) {
  __shared__ float sh[32];
  const int h = blockIdx.x, bucket = blockIdx.y, slots = 2 * reach + 1;
  const bool upper = rb.bidirectional && bucket >= rb.per_side;
  const int c = upper ? bucket - rb.per_side : bucket, far = c - rb.exact;
  int lo = far >= 0 ? rb.first[far] : c;
  int hi = c == rb.per_side - 1 ? reach : (far >= 0 ? rb.first[far + 1] : c + 1) - 1;
  if (upper && lo == 0) lo = 1;  // distance 0 belongs to the lower half
  hi = min(hi, reach);
  int x0 = upper ? reach + lo : reach - hi, x1 = upper ? reach + hi : reach - lo;
  if (!rb.bidirectional && c == 0) x1 = 2 * reach;  // keys after the query
  float t = 0.f;
  if (lo <= hi) {
    const float* mine = partial + (long long)h * blocks * slots + x0;
    const unsigned run = (unsigned)(x1 - x0 + 1), n = run * (unsigned)blocks;
    for (unsigned i = threadIdx.x; i < n; i += blockDim.x) t += mine[(long long)(i / run) * slots + i % run];
  }
  t = block_sum(t, sh);
  if (threadIdx.x == 0) {
    const long long at = (long long)bucket * H + h;
    if (dtype == B200_F32) static_cast<float*>(out)[at] = t;
    else if (dtype == B200_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16(t);
    else static_cast<__half*>(out)[at] = __float2half(t);
  }
}

struct Plan {
  Args a;
  int threads, nv;  // nv 0: a block per row
  size_t smem;
};

Plan make_plan(const B200BiasSoftmax& p, bool bwd) {
  Plan pl{};
  Args& a = pl.a;
  a.s = p.scores; a.g = p.grad; a.out = p.out; a.stats = reinterpret_cast<float2*>(p.stats);
  a.table = p.table; a.mask = p.mask; a.table_dtype = p.table_dtype; a.mask_dtype = p.mask_dtype;
  a.st_b = p.stride[0]; a.st_h = p.stride[1]; a.st_i = p.stride[2];
  a.mk_b = p.mask_stride[0]; a.mk_h = p.mask_stride[1]; a.mk_i = p.mask_stride[2]; a.mk_j = p.mask_stride[3];
  a.H = p.H; a.Lq = p.Lq; a.Lk = p.Lk; a.offset = p.query_offset; a.scale = p.scale; a.rb = p.buckets;
  a.rows = (unsigned)((long long)p.B * p.Lq);
  // beyond the farthest distance of this call nothing has to be told apart either
  const long long ahead = (long long)p.Lk - 1 - p.query_offset, behind = (long long)p.Lq - 1 + p.query_offset;
  long long far = ahead > behind ? ahead : behind;
  if (far < -ahead) far = -ahead;
  if (far < -behind) far = -behind;
  a.reach = (int)(far + 1 < p.buckets.max_distance ? far + 1 : p.buckets.max_distance);
  const int vec = p.dtype == B200_F32 ? 4 : 8;
  const bool aligned = p.Lk % vec == 0 && p.stride[0] % vec == 0 && p.stride[1] % vec == 0 && p.stride[2] % vec == 0;
  const int nvec = aligned ? p.Lk / vec : (p.Lk + 2 * vec - 2) / vec;  // an unaligned row may touch one vector more
  const int words = 2 * a.reach + (2 * a.reach >> 5) + 1;
  pl.threads = kMaxThreads;
  int groups;
  if (nvec <= 32 * 4) {
    int G = 1;
    while (G < nvec && G < 32) G <<= 1;
    if (bwd)  // sums over distances for each group: wider groups where there would be too many
      while (G < 32 && (kMaxThreads / G) * words * 4 > 64 * 1024) G <<= 1;
    a.group = G;
    const int nv = (nvec + G - 1) / G;
    pl.nv = nv <= 1 ? 1 : (nv <= 2 ? 2 : 4);
    if (bwd)
      while (pl.threads > 32 && (pl.threads / G + 1) * words * 4 > 96 * 1024) pl.threads >>= 1;
    groups = pl.threads / G;
    pl.smem = (size_t)(bwd ? groups + 1 : 1) * words * 4;
  } else {
    groups = 1;
    pl.smem = (size_t)(bwd ? 2 : 1) * words * 4;
  }
  long long blocks = 148LL * 8 * kMaxThreads / pl.threads / (p.H > 0 ? p.H : 1);
  const long long most = ((long long)a.rows + groups - 1) / groups;
  if (blocks > most) blocks = most;
  if (blocks < 1) blocks = 1;
  a.rows_per_block = (unsigned)((a.rows + blocks - 1) / blocks);
  a.rows_per_block = (a.rows_per_block + groups - 1) / groups * groups;
  if (a.rows_per_block < 1) a.rows_per_block = 1;
  a.blocks_per_head = (int)((a.rows + a.rows_per_block - 1) / a.rows_per_block);
  return pl;
}

template <typename K>
int launch(K kernel, const Plan& pl, cudaStream_t s) {
  if (pl.smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pl.smem);
    if (e != cudaSuccess) return (int)e;
  }
  kernel<<<(unsigned)(pl.a.blocks_per_head * pl.a.H), pl.threads, pl.smem, s>>>(pl.a);
  return (int)cudaGetLastError();
}

template <typename T, int VEC>
int dispatch(const Plan& pl, bool bwd, cudaStream_t s) {
  switch (pl.nv) {
    case 1: return bwd ? launch(bias_softmax_bwd_rows<T, VEC, 1>, pl, s) : launch(bias_softmax_fwd_rows<T, VEC, 1>, pl, s);
    case 2: return bwd ? launch(bias_softmax_bwd_rows<T, VEC, 2>, pl, s) : launch(bias_softmax_fwd_rows<T, VEC, 2>, pl, s);
    case 4: return bwd ? launch(bias_softmax_bwd_rows<T, VEC, 4>, pl, s) : launch(bias_softmax_fwd_rows<T, VEC, 4>, pl, s);
    default: return bwd ? launch(bias_softmax_bwd_long<T, VEC>, pl, s) : launch(bias_softmax_fwd_long<T, VEC>, pl, s);
  }
}
int dispatch_type(const Plan& pl, int dtype, bool bwd, cudaStream_t s) {
  if (dtype == B200_BF16) return dispatch<__nv_bfloat16, 8>(pl, bwd, s);
  if (dtype == B200_F16) return dispatch<__half, 8>(pl, bwd, s);
  if (dtype == B200_F32) return dispatch<float, 4>(pl, bwd, s);
  return (int)cudaErrorInvalidValue;
}

bool valid(const B200BiasSoftmax* p) {
  const B200RelativeBuckets& r = p->buckets;
  return p->B >= 0 && p->H >= 0 && p->Lq >= 0 && p->Lk >= 0 && (long long)p->B * p->Lq < (1LL << 31) &&
         p->Lk < (1 << 30) && r.exact >= 1 && r.per_side > r.exact && r.per_side - r.exact <= B200_MAX_FAR_BUCKETS &&
         r.max_distance > r.exact && r.max_distance <= B200_MAX_BIAS_DISTANCE;
}
bool empty(const B200BiasSoftmax* p) { return (long long)p->B * p->Lq == 0 || p->H == 0 || p->Lk == 0; }

}  // namespace

extern "C" int b200_bias_softmax_fwd(const B200BiasSoftmax* p, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  if (empty(p)) return 0;
  return dispatch_type(make_plan(*p, false), p->dtype, false, (cudaStream_t)stream);
}

extern "C" long long b200_bias_softmax_workspace(const B200BiasSoftmax* p) {
  if (!valid(p) || empty(p) || !p->dtable) return 0;
  const Plan pl = make_plan(*p, true);
  return (long long)p->H * pl.a.blocks_per_head * (2 * pl.a.reach + 1) * (long long)sizeof(float);
}

extern "C" int b200_bias_softmax_bwd(const B200BiasSoftmax* p, void* workspace, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  cudaStream_t s = (cudaStream_t)stream;
  if (empty(p)) {
    const int buckets = p->buckets.per_side * (p->buckets.bidirectional ? 2 : 1);
    if (!p->dtable || p->H == 0) return 0;
    return (int)cudaMemsetAsync(p->dtable, 0, (size_t)buckets * p->H * (p->table_dtype == B200_F32 ? 4 : 2), s);
  }
  Plan pl = make_plan(*p, true);
  pl.a.partial = p->dtable ? static_cast<float*>(workspace) : nullptr;
  const int rc = dispatch_type(pl, p->dtype, true, s);
  if (rc || !p->dtable) return rc;
  const int buckets = p->buckets.per_side * (p->buckets.bidirectional ? 2 : 1);
  bias_table_grad<<<dim3((unsigned)p->H, (unsigned)buckets), kMaxThreads, 0, s>>>(pl.a.partial, pl.a.blocks_per_head, pl.a.reach, p->buckets, p->H,
                                                                                p->dtable, p->table_dtype);
  return (int)cudaGetLastError();
}
