// Distillation against a teacher of which the K largest logits of every row are kept: loss and gradient.
//
//   p = softmax over the row's kept logits of t / T       q = softmax over the whole vocabulary of z / T
//   loss_row = T^2 sum_k p_k (log p_k - log q_{idx_k})    dz_j = g T (q_j - sum of p_k over the k with idx_k = j)
//   An entry with a negative index (or a teacher logit of -inf) is absent; a row without entries has loss and gradient 0 and does not
//   count in the mean.  The same index may occur more than once: its shares add up.
//
// Bound by memory: z has to be read and dz written once.  A block owns a row: it takes the running maximum and sum in one pass;
// when the caller wants gradients, it reads the row again while that is still in the caches and writes dz at once with the
// factor that backward() begins with, 1 (over the number of rows for a mean).  When another factor arrives, the backward writes dz anew
// from z and the two saved numbers of each row, so that every gradient is rounded once whatever the factor.
#include "kernels_api.h"
#include "row_vec.cuh"

namespace {

using namespace rowvec;

constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kThreads = 512;

struct Shared {
  float red[32];
  int idx[B200_DISTILL_MAX_K];
  float share[B200_DISTILL_MAX_K];
};

__device__ __forceinline__ float warp_red(float v, bool is_max) { return is_max ? group_max(v, 32) : group_sum(v, 32); }
__device__ __forceinline__ float block_red(float v, bool is_max, float* sh) {
  v = warp_red(v, is_max);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = warp_red((threadIdx.x & 31) < blockDim.x / 32 ? sh[threadIdx.x & 31] : (is_max ? kNegInf : 0.f), is_max);
  __syncthreads();
  return v;
}

__device__ __forceinline__ float teacher_at(const void* p, long long i, int dt) {
  if (dt == B200_F32) return static_cast<const float*>(p)[i];
  if (dt == B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ long long index_at(const B200Distill& p, long long row, int k) {
  const long long at = row * p.index_ld + k;
  return p.index_dtype == B200_I64 ? static_cast<const long long*>(p.index)[at] : (long long)static_cast<const int*>(p.index)[at];
}
// Whether entry k of a row is there.
__device__ __forceinline__ bool present(const B200Distill& p, long long row, int k) {
  const long long i = index_at(p, row, k);
  return i >= 0 && i < p.V && teacher_at(p.teacher, row * p.teacher_ld + k, p.teacher_dtype) != kNegInf;
}

// Loads the row's entries into shared memory: indices (-1: absent) and shares.  Returns whether there are any; *plogp: this
// thread's part of sum p log p.
__device__ __forceinline__ bool load_teacher(const B200Distill& p, long long row, Shared& sh, float* plogp) {
  float top = kNegInf;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const long long i = index_at(p, row, k);
    const float t = teacher_at(p.teacher, row * p.teacher_ld + k, p.teacher_dtype);
    const bool there = i >= 0 && i < p.V && t != kNegInf;
    if (i >= p.V && p.bad_flag) *p.bad_flag = 1;
    sh.idx[k] = there ? (int)i : -1;
    sh.share[k] = t;
    if (there) top = fmaxf(top, t);
  }
  int any = 0;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) any |= sh.idx[k] >= 0;
  any = __syncthreads_or(any);
  top = block_red(top, true, sh.red);
  float sum = 0.f;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x)
    if (sh.idx[k] >= 0) sum += __expf((sh.share[k] - top) * p.inv_temperature);
  sum = block_red(sum, false, sh.red);
  const float logsum = logf(sum);
  float part = 0.f;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    if (sh.idx[k] < 0) continue;
    const float lp = (sh.share[k] - top) * p.inv_temperature - logsum, share = expf(lp);
    sh.share[k] = share;
    part += share == 0.f ? 0.f : share * lp;
  }
  *plogp = part;
  __syncthreads();
  return any != 0;
}

template <typename T, int VEC, bool FWD, bool GRAD>
__global__ void __launch_bounds__(kThreads) distill_kernel(const __grid_constant__ B200Distill p) {
  __shared__ Shared sh;
  // the factor of the gradient: what backward() was given, over the number of rows for a mean
  float count_inv = 1.f;
  if (GRAD && p.count) count_inv = 1.f / fmaxf(*p.count, 1.f);
  if (GRAD && !FWD && p.skip_factor_one && *p.grad == 1.f) return;  // the forward has written this gradient
  const float c = p.inv_temperature * 1.4426950408889634f;
  for (long long row = blockIdx.x; row < p.N; row += gridDim.x) {
    const T* z = static_cast<const T*>(p.logits) + row * p.ld;
    const int phase = (int)((reinterpret_cast<uintptr_t>(z) / sizeof(T)) & (VEC - 1));
    float plogp;
    const bool any = load_teacher(p, row, sh, &plogp);
    float m, s;
    if (FWD) {
      m = kNegInf;
      s = 0.f;
      for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.V; j0 += kThreads * VEC) {
        float v[VEC];
        const bool whole = j0 >= 0 && j0 + VEC <= p.V;
        if (whole) {
          load<T, VEC>(z + j0, v);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[k] = j0 + k >= 0 && j0 + k < p.V ? to_f32<T>(z[j0 + k]) : kNegInf;
        }
        float top = v[0];
#pragma unroll
        for (int k = 1; k < VEC; ++k) top = fmaxf(top, v[k]);
        if (top > m) {
          s *= exp2f((m - top) * c);
          m = top;
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) s += v[k] == kNegInf ? 0.f : exp2f((v[k] - m) * c);
      }
      const float top = block_red(m, true, sh.red);
      s = block_red(m == kNegInf ? s : s * exp2f((m - top) * c), false, sh.red);
      m = top;
      if (p.stats && threadIdx.x == 0) reinterpret_cast<float2*>(p.stats)[row] = make_float2(m, s);
      const float logs = logf(s);
      float part = plogp;
      for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
        if (sh.idx[k] < 0 || sh.share[k] == 0.f) continue;
        part -= sh.share[k] * ((to_f32<T>(z[sh.idx[k]]) - m) * p.inv_temperature - logs);
      }
      part = block_red(part, false, sh.red);
      if (threadIdx.x == 0) p.row_loss[row] = any ? part * p.temperature * p.temperature : 0.f;
    } else {
      const float2 st = reinterpret_cast<const float2*>(p.stats)[row];
      m = st.x;
      s = st.y;
    }
    if (GRAD) {
      T* d = static_cast<T*>(p.dlogits) + row * p.ld;
      const float factor = any ? (FWD ? 1.f : p.grad[p.grad_per_row ? row * p.grad_ld : 0]) * count_inv * p.temperature : 0.f;
      const float scale = factor / s;
      for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.V; j0 += kThreads * VEC) {
        float v[VEC];
        if (j0 >= 0 && j0 + VEC <= p.V) {
          load<T, VEC>(z + j0, v);
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[k] = any ? scale * exp2f((v[k] - m) * c) : 0.f;
          store<T, VEC>(d + j0, v);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            if (j0 + k >= 0 && j0 + k < p.V) d[j0 + k] = from_f32<T>(any ? scale * exp2f((to_f32<T>(z[j0 + k]) - m) * c) : 0.f);
        }
      }
      __syncthreads();
      // the kept entries: the first occurrence of an index writes the value with the shares of all of them
      for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
        const int i = sh.idx[k];
        if (i < 0) continue;
        bool first = true;
        float share = 0.f;
        for (int o = 0; o < p.K; ++o) {
          if (sh.idx[o] != i) continue;
          first = first && o >= k;
          share += sh.share[o];
        }
        if (first) d[i] = from_f32<T>(scale * exp2f((to_f32<T>(z[i]) - m) * c) - factor * share);
      }
    }
    __syncthreads();  // the next row overwrites the entries
  }
}

// The number of rows with at least one entry.
__global__ void __launch_bounds__(1024) distill_count_kernel(const __grid_constant__ B200Distill p) {
  __shared__ float red[32];
  float n = 0.f;
  for (long long row = threadIdx.x; row < p.N; row += blockDim.x) {
    int k = 0;
    while (k < p.K && !present(p, row, k)) ++k;
    n += k < p.K ? 1.f : 0.f;
  }
  n = block_red(n, false, red);
  if (threadIdx.x == 0) *p.count = n;
}

// Sum of the rows' losses over `count` (null: 1), in a fixed order.
__global__ void __launch_bounds__(1024) distill_sum_kernel(const float* rows, long long n, const float* count, float* loss) {
  __shared__ float red[32];
  float s = 0.f;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) s += rows[i];
  s = block_red(s, false, red);
  if (threadIdx.x == 0) *loss = count ? s / fmaxf(*count, 1.f) : s;
}

bool valid(const B200Distill* p) {
  return p->N >= 0 && p->V >= 1 && p->V < (1LL << 31) - 8192 && p->K >= 0 && p->K <= B200_DISTILL_MAX_K && p->temperature > 0.f &&
         (p->index_dtype == B200_I64 || p->index_dtype == B200_I32);
}

template <bool FWD, bool GRAD>
int launch(const B200Distill& p, cudaStream_t s) {
  const unsigned grid = (unsigned)(p.N < 148 * 4 ? p.N : 148 * 4);
  if (p.dtype == B200_BF16) distill_kernel<__nv_bfloat16, 8, FWD, GRAD><<<grid, kThreads, 0, s>>>(p);
  else if (p.dtype == B200_F16) distill_kernel<__half, 8, FWD, GRAD><<<grid, kThreads, 0, s>>>(p);
  else if (p.dtype == B200_F32) distill_kernel<float, 4, FWD, GRAD><<<grid, kThreads, 0, s>>>(p);
  else return (int)cudaErrorInvalidValue;
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" int b200_distill_fwd(const B200Distill* p, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  cudaStream_t s = (cudaStream_t)stream;
  if (p->count) distill_count_kernel<<<1, 1024, 0, s>>>(*p);
  if (p->N > 0) {
    const int rc = p->dlogits ? launch<true, true>(*p, s) : launch<true, false>(*p, s);
    if (rc) return rc;
  }
  if (p->loss) distill_sum_kernel<<<1, 1024, 0, s>>>(p->row_loss, p->N, p->count, p->loss);
  return (int)cudaGetLastError();
}

extern "C" int b200_distill_bwd(const B200Distill* p, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  return p->N > 0 ? launch<false, true>(*p, (cudaStream_t)stream) : 0;
}
