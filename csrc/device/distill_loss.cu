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
//
// Measured on a B200, bf16, loss and gradient: 4096 x 30522, 64 kept: 128 us = 3.9 TB/s, 0.60 of the measured copy bandwidth; 4096 x 131072,
// 128 kept: 530 us = 4.1 TB/s, 0.62; the loss alone 64 us (3.9 TB/s) and 213 us (5.0 TB/s).  With a factor other than 1 the early gradient was
// written for nothing: 231 us with the backward at 4096 x 30522; a caller who knows leaves it out (163 us: the loss and a pass of its own).
// What bounds the pass: issue slots (72 % busy) at 30522 words; at 131072 also L2, where half of the second reading misses.  Many short
// rows are bound by their reductions and by the last block's sum over them: 8192 x 1000, 5 kept, 31 us for the loss, 40 with its gradient, 0.08
// and 0.13 of the copy.
#include "kernels_api.h"
#include "row_vec.cuh"

namespace {

using namespace rowvec;

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxThreads = 512;
// (4096 x 30522 bf16 with gradient: units of 2 and 4 under way 129 us, 2 and 6: 148, 4 and 3: 142.)
constexpr int kUnit = 2;   // vectors that a thread takes at a time: a unit of a row is kUnit vectors for each thread
constexpr int kDepth = 4;  // units under way

struct Shared {
  float2 student[kMaxThreads / 32], teacher[kMaxThreads / 32];  // each warp's (maximum, sum of exponentials)
  float loss[kMaxThreads / 32];
  __align__(16) int idx[B200_DISTILL_MAX_K];
  __align__(16) float share[B200_DISTILL_MAX_K];
  int last;
};

__device__ __forceinline__ float finite_max(float m) { return m == kNegInf ? 0.f : m; }
// (maximum, sum of the exponentials of c times the distance to it) of 32 lanes, for the student's logits and the teacher's at once: the
// two chains of exchanges hide one another.
__device__ __forceinline__ void join(float2& a, float2& b, float c) {
  float ta = a.x, tb = b.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ta = fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, o));
    tb = fmaxf(tb, __shfl_xor_sync(0xffffffffu, tb, o));
  }
  float sa = a.y * exp2_fast((a.x - finite_max(ta)) * c);  // maximum -inf: nothing, or a NaN
  float sb = b.y * exp2_fast((b.x - finite_max(tb)) * c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sa += __shfl_xor_sync(0xffffffffu, sa, o);
    sb += __shfl_xor_sync(0xffffffffu, sb, o);
  }
  a = make_float2(ta, sa);
  b = make_float2(tb, sb);
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

// A kept entry of the row in work: each thread has up to two.
struct Entry {
  int idx;      // -1: absent
  float value;  // the teacher's logit, then its share
};
// The same as it stands in memory, asked for a row ahead.
struct Asked {
  long long index;
  float value;
};
__device__ __forceinline__ void ask(const B200Distill& p, long long row, Asked (&a)[2]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int k = threadIdx.x + q * blockDim.x;
    if (k < p.K && row < p.N) {
      a[q].index = index_at(p, row, k);
      a[q].value = teacher_at(p.teacher, row * p.teacher_ld + k, p.teacher_dtype);
    }
  }
}

// A row: `head` elements up to the first 16-byte boundary, whole vectors, `tail` elements.
template <typename T, int VEC>
struct Row {
  const T* z;
  int head, tail;
  unsigned vectors;
  __device__ __forceinline__ Row(const T* p, int V) : z(p) {
    head = (int)((VEC - ((reinterpret_cast<uintptr_t>(p) / sizeof(T)) & (VEC - 1))) & (VEC - 1));
    if (head > V) head = V;
    vectors = (unsigned)(V - head) / VEC;
    tail = (V - head) % VEC;
  }
  __device__ __forceinline__ int ragged(int e, int V) const { return e < head ? e : V - tail + e - head; }  // place of ragged element e
};

// The units that a block will take, in order: a row's once for its sum, again for its gradient (then out of L2), then the next row's.
// Each thread copies its vectors of the units to come to a place of its own in shared memory, so that reading never stops: not at a
// row's reductions nor while its gradient is written.
template <typename T, int VEC, int PASSES>
struct Stream {
  const B200Distill& p;
  Pack<T, VEC>* ring;  // this thread's first vector; unit d begins at d * kUnit * blockDim
  long long row;
  int pass, put, got;
  unsigned at, vectors;
  const T* body;
  const uint64_t keep = l2_evict_last(), drop = l2_evict_first();
  __device__ __forceinline__ Stream(const B200Distill& args, void* shared)
      : p(args), ring(static_cast<Pack<T, VEC>*>(shared) + threadIdx.x), row(blockIdx.x), pass(0), put(0), got(0), at(0) {
    enter();
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d) next();
  }
  __device__ __forceinline__ void enter() {
    if (row >= p.N) return;
    const Row<T, VEC> r(static_cast<const T*>(p.logits) + row * p.ld, (int)p.V);
    body = r.z + r.head;
    vectors = r.vectors;
  }
  __device__ __forceinline__ void next() {
    if (row < p.N) {
#pragma unroll
      for (int u = 0; u < kUnit; ++u) {
        const unsigned v = at + u * blockDim.x + threadIdx.x;
        if (v < vectors) copy16_async(ring + (put * kUnit + u) * blockDim.x, body + (size_t)v * VEC, PASSES == 2 && pass == 0 ? keep : drop);
      }
      at += kUnit * blockDim.x;
      if (at >= vectors) {
        at = 0;
        if (++pass == PASSES) {
          pass = 0;
          row += gridDim.x;
          enter();
        }
      }
    }
    copies_commit();
    put = put == kDepth - 1 ? 0 : put + 1;
  }
  __device__ __forceinline__ void take(Pack<T, VEC> (&raw)[kUnit]) {
    next();
    copies_wait<kDepth - 1>();
#pragma unroll
    for (int u = 0; u < kUnit; ++u) raw[u] = ring[(got * kUnit + u) * blockDim.x];
    got = got == kDepth - 1 ? 0 : got + 1;
  }
};

// Rows are counted by up to 32 blocks, each of about 8192 entries.
constexpr int kCountThreads = 1024;
__host__ __device__ __forceinline__ int count_blocks(const B200Distill& p) {
  const long long blocks = p.N * p.K / 8192 + 1;
  return blocks < B200_DISTILL_SCRATCH - 1 ? (int)blocks : B200_DISTILL_SCRATCH - 1;
}
// Their sum; called by whole warps.
__device__ __forceinline__ float rows_counted(const B200Distill& p) {
  const int lane = threadIdx.x & 31;
  return (float)__reduce_add_sync(0xffffffffu, lane < count_blocks(p) ? __ldcg(p.scratch + 1 + lane) : 0u);
}

template <typename T, int VEC, bool FWD, bool GRAD>
__global__ void __launch_bounds__(kMaxThreads, 2) distill_kernel(const __grid_constant__ B200Distill p) {
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char ring[];
  if (GRAD && !FWD && p.skip_factor_one && *p.grad == 1.f) return;  // the forward has written this gradient
  const int V = (int)p.V, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float c = p.inv_temperature * kLog2e;
  Stream<T, VEC, FWD && GRAD ? 2 : 1> stream(p, ring);
  Pack<T, VEC> raw[kUnit];
  float count_inv = GRAD && !FWD && p.count ? 1.f / fmaxf(*p.count, 1.f) : 1.f;
  bool counted = false;
  Asked asked[2];
  ask(p, blockIdx.x, asked);
  for (long long row = blockIdx.x; row < p.N; row += gridDim.x) {
    const Row<T, VEC> r(static_cast<const T*>(p.logits) + row * p.ld, V);
    Entry e[2];
    T z[2];  // the student's logits there, on their way while the row is read
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      e[q].idx = -1;
      z[q] = from_f32<T>(0.f);
      if (threadIdx.x + q * blockDim.x < p.K) {
        const long long i = asked[q].index;
        e[q].value = asked[q].value;
        if (i >= 0 && i < p.V && e[q].value != kNegInf) {
          e[q].idx = (int)i;
          z[q] = r.z[i];
        }
        if (i >= p.V && p.bad_flag) *p.bad_flag = 1;
      }
    }
    const int place = (int)threadIdx.x < r.head + r.tail ? r.ragged(threadIdx.x, V) : -1;  // at most 14 elements outside whole vectors
    const T ragged = place >= 0 ? r.z[place] : from_f32<T>(0.f);
    float m, s;
    if (FWD) {
      m = kNegInf;
      s = 0.f;
      unsigned v0 = threadIdx.x;
      do {
        stream.take(raw);
        float top = m;
#pragma unroll
        for (int u = 0; u < kUnit; ++u)
          if (v0 + u * blockDim.x < r.vectors) top = fmaxf(top, max_of(raw[u]));
        if (top > m) {
          s *= exp2_fast((m - top) * c);
          m = top;
        }
        const float2 minus = both(-finite_max(m));
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
          if (v0 + u * blockDim.x < r.vectors) {
#pragma unroll
            for (int k = 0; k < VEC / 2; ++k) {
              const float2 x = mul2(add2(pair_of(raw[u], k), minus), both(c));
              sum = add2(sum, make_float2(exp2_fast(x.x), exp2_fast(x.y)));
            }
          }
        }
        s += sum.x + sum.y;
        v0 += kUnit * blockDim.x;
      } while (v0 - threadIdx.x < r.vectors);
      if (place >= 0) {
        const float x = to_f32<T>(ragged);
        if (x > m) {
          s *= exp2_fast((m - x) * c);
          m = x;
        }
        s += exp2_fast((x - finite_max(m)) * c);
      }
    } else {
      const float2 st = reinterpret_cast<const float2*>(p.stats)[row];
      m = st.x;
      s = st.y;
    }
    // both softmax sums over the block
    float2 t = make_float2(kNegInf, 0.f);
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (e[q].idx >= 0) t.x = fmaxf(t.x, e[q].value);
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (e[q].idx >= 0) t.y += exp2_fast((e[q].value - finite_max(t.x)) * c);
    float2 st = make_float2(m, s);
    join(st, t, c);
    if (lane == 0) {
      sh.student[warp] = st;
      sh.teacher[warp] = t;
    }
    const bool any = __syncthreads_or(e[0].idx >= 0 || e[1].idx >= 0);
    const bool mine = lane < blockDim.x / 32;
    st = mine ? sh.student[lane] : make_float2(kNegInf, 0.f);
    t = mine ? sh.teacher[lane] : make_float2(kNegInf, 0.f);
    join(st, t, c);
    if (FWD) {
      m = finite_max(st.x);
      s = st.y;
      if (p.stats && threadIdx.x == 0) reinterpret_cast<float2*>(p.stats)[row] = make_float2(m, s);
    }
    ask(p, row + gridDim.x, asked);
    const float t_log = logf(t.y), s_log = FWD ? logf(s) : 0.f;
    float part = 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = threadIdx.x + q * blockDim.x;
      if (k >= p.K) continue;
      if (e[q].idx >= 0) {
        const float lp = (e[q].value - t.x) * p.inv_temperature - t_log;
        e[q].value = expf(lp);
        if (FWD && e[q].value != 0.f) part += e[q].value * (lp - ((to_f32<T>(z[q]) - m) * p.inv_temperature - s_log));
      }
      if (GRAD) {
        sh.idx[k] = e[q].idx;
        sh.share[k] = e[q].value;
      }
    }
    if (GRAD && threadIdx.x < 3 && p.K + threadIdx.x < B200_DISTILL_MAX_K) sh.idx[p.K + threadIdx.x] = -1;
    if (FWD) {
      part = group_sum(part, 32);
      if (lane == 0) sh.loss[warp] = part;
    }
    __syncthreads();
    if (FWD && warp == 0) {
      part = group_sum(lane < blockDim.x / 32 ? sh.loss[lane] : 0.f, 32);
      if (lane == 0) p.row_loss[row] = any ? part * p.temperature * p.temperature : 0.f;
    }
    if (GRAD) {
      if (FWD && !counted) {  // the number of rows comes from the kernel in front, which may still run
        if (p.count) {
          cudaGridDependencySynchronize();
          count_inv = 1.f / fmaxf(rows_counted(p), 1.f);
        }
        counted = true;
      }
      T* d = static_cast<T*>(p.dlogits) + row * p.dlogits_ld;
      T* d_body = d + r.head;
      const float factor = any ? (FWD ? 1.f : p.grad[p.grad_per_row ? row * p.grad_ld : 0]) * count_inv * p.temperature : 0.f;
      const float scale = any ? factor / s : 0.f;
      const float2 minus = both(-m);
      unsigned v0 = threadIdx.x;
      do {
        stream.take(raw);
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
          if (v0 + u * blockDim.x < r.vectors) {
            if (any) {
#pragma unroll
              for (int k = 0; k < VEC / 2; ++k) {
                const float2 x = mul2(add2(pair_of(raw[u], k), minus), both(c));
                set_pair(raw[u], k, mul2(make_float2(exp2_fast(x.x), exp2_fast(x.y)), both(scale)));
              }
            } else {
#pragma unroll
              for (int k = 0; k < VEC / 2; ++k) set_pair(raw[u], k, make_float2(0.f, 0.f));
            }
            __stcs(reinterpret_cast<uint4*>(d_body + (size_t)(v0 + u * blockDim.x) * VEC), *reinterpret_cast<const uint4*>(&raw[u]));
          }
        }
        v0 += kUnit * blockDim.x;
      } while (v0 - threadIdx.x < r.vectors);
      if (place >= 0) d[place] = from_f32<T>(any ? scale * exp2_fast((to_f32<T>(ragged) - m) * c) : 0.f);
      __syncthreads();
      // the kept entries: the first occurrence of an index writes the value with the shares of all of them
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = threadIdx.x + q * blockDim.x, i = e[q].idx;
        if (i < 0) continue;
        bool first = true;
        float share = 0.f;
        for (int o = 0; o < p.K; o += 4) {  // (behind the last entry: -1)
          const int4 at = *reinterpret_cast<const int4*>(sh.idx + o);
          if (at.x != i && at.y != i && at.z != i && at.w != i) continue;
          const int four[4] = {at.x, at.y, at.z, at.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (four[u] != i) continue;
            first = first && o + u >= k;
            share += sh.share[o + u];
          }
        }
        if (first) d[i] = from_f32<T>(scale * exp2_fast((to_f32<T>(z[q]) - m) * c) - factor * share);
      }
    }
  }
  if (!FWD || !p.loss) return;
  // The block that ends last adds up the rows' losses, in an order that does not depend on which one it is.
  cudaGridDependencySynchronize();  // ticket and numbers were set by the kernel in front
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    sh.last = atomicAdd(p.scratch, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!sh.last) return;
  float sum = 0.f;
  for (long long i = threadIdx.x; i < p.N; i += blockDim.x) sum += __ldcg(p.row_loss + i);
  sum = group_sum(sum, 32);
  if (lane == 0) sh.loss[warp] = sum;
  __syncthreads();
  const float count = p.count ? rows_counted(p) : 1.f;
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < blockDim.x / 32; ++w) sum += sh.loss[w];
    *p.loss = sum / fmaxf(count, 1.f);
    if (p.count) *p.count = count;
  }
}

// The number of rows with at least one entry (for a mean), in a part for each block, and the ticket of the blocks that follow.  The kernel
// behind starts at once and needs the number only when its first gradients are written.  A lane looks at the first entry of a row of its
// own, which decides most rows; those that it leaves open are gone through by groups of lanes, four entries to a lane.  (A mean and its
// gradient, bf16, 85 % of the rows without entries: 16384 x 4000, 128 kept, 1060 us with a thread for each row in one block, 153 us so;
// 4096 x 30522, 64 kept: 228 and 122 us.)
__global__ void __launch_bounds__(kCountThreads) distill_count_kernel(const __grid_constant__ B200Distill p) {
  cudaTriggerProgrammaticLaunchCompletion();
  __shared__ int red[kCountThreads / 32];
  if (threadIdx.x == 0 && blockIdx.x == 0) p.scratch[0] = 0;
  if (!p.count) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int G = 1;
  while (G < 32 && 4 * G < p.K - 1) G *= 2;
  const long long warps = (long long)gridDim.x * (kCountThreads / 32), share = (p.N + warps - 1) / warps;
  const int rows = share < 32 ? (int)share : 32;  // of a warp at a time
  int n = 0;
  for (long long base = (blockIdx.x * (kCountThreads / 32) + warp) * (long long)rows; base < p.N; base += warps * rows) {
    const bool mine = lane < rows && base + lane < p.N;
    const bool first = mine && p.K > 0 && present(p, base + lane, 0);
    n += first;
    for (unsigned open = __ballot_sync(0xffffffffu, mine && !first); open;) {
      const unsigned pick = __fns(open, 0, lane / G + 1);  // this group's row; none left: beyond 31
      bool there = false;
      if (pick < 32) {
        const long long row = base + pick;
        for (int k = 1 + lane % G; k < p.K; k += 4 * G) {
          long long i[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) i[u] = k + u * G < p.K ? index_at(p, row, k + u * G) : -1;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            there |= i[u] >= 0 && i[u] < p.V && teacher_at(p.teacher, row * p.teacher_ld + k + u * G, p.teacher_dtype) != kNegInf;
        }
      }
      const unsigned hits = __ballot_sync(0xffffffffu, there) >> (lane / G * G) & (0xffffffffu >> (32 - G));
      n += lane % G == 0 && hits != 0;
      for (int q = 0; q < 32 / G; ++q) open &= open - 1;
    }
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) red[warp] = n;
  __syncthreads();
  if (warp == 0) {
    n = __reduce_add_sync(0xffffffffu, red[lane]);
    if (lane == 0) p.scratch[1 + blockIdx.x] = (unsigned)n;
  }
}

bool valid(const B200Distill* p) {
  return p->N >= 0 && p->V >= 1 && p->V < (1LL << 31) - 8192 && p->K >= 0 && p->K <= B200_DISTILL_MAX_K && p->temperature > 0.f &&
         (p->index_dtype == B200_I64 || p->index_dtype == B200_I32) && (!p->loss || p->scratch);
}

// Threads for a row: at most 30 vectors for each, and at least half as many as there are kept entries.  Small blocks because a row's
// reductions leave an SM idle unless others are at work; not smaller, because more rows in work do not stay in L2 until their second
// pass.  Loss and gradient, us, with 128 / 256 / 512 threads (4096 rows, bf16): 24000 words 112 / 118 / 140, 31000 words (3875 vectors) 128 / 132 /
// 151, 32000: 146 / 146 / 165, 40000: 191 / 175 / 192, 61000: 280 / 234 / 249, 65536 (8192 vectors): 329 / 276 / 278, 98304: 501 / 454 / 394; fp32, where 256
// wins from 2800 vectors on: 10000 words 85 / 85 / 106, 15300 (3825): 122 / 116 / 132, 30522: 290 / 237 / 237, 35000: 331 / 286 / 265.  Fewer than 128
// only where a row has no 64 vectors to give (65536 x 256 bf16, loss and loss with gradient, 32 / 64 / 128 threads: 202 / 177 / 183 and 230 / 237 /
// 249; 16384 x 2000: 77 / 67 / 65 and 122 / 108 / 108).
int row_threads(const B200Distill& p) {
  const long long vectors = p.V / (p.dtype == B200_F32 ? 4 : 8);
  int t = vectors > 64 ? 128 : 64;
  while (t < kMaxThreads && (vectors > 30LL * t || p.K > 2 * t)) t *= 2;
  return t;
}

// `after`: the counting kernel is in front and this one may begin before it ends.
template <bool FWD, bool GRAD>
int launch(const B200Distill& p, bool after, cudaStream_t s) {
  const int threads = row_threads(p);
  const long long most = 148LL * (2 * kMaxThreads / threads);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.N < most ? p.N : most));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &overlap;
  cfg.numAttrs = after ? 1 : 0;
  cfg.dynamicSmemBytes = (size_t)kDepth * kUnit * 16 * threads;
  auto start = [&](auto kernel) {
    cudaError_t e = cudaSuccess;
    if (cfg.dynamicSmemBytes > 32 * 1024)
      e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDepth * kUnit * 16 * kMaxThreads);
    return (int)(e == cudaSuccess ? cudaLaunchKernelEx(&cfg, kernel, p) : e);
  };
  if (p.dtype == B200_BF16) return start(distill_kernel<__nv_bfloat16, 8, FWD, GRAD>);
  if (p.dtype == B200_F16) return start(distill_kernel<__half, 8, FWD, GRAD>);
  if (p.dtype == B200_F32) return start(distill_kernel<float, 4, FWD, GRAD>);
  return (int)cudaErrorInvalidValue;
}

}  // namespace

extern "C" int b200_distill_fwd(const B200Distill* p, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  cudaStream_t s = (cudaStream_t)stream;
  if (p->N == 0) return p->loss ? (int)cudaMemsetAsync(p->loss, 0, sizeof(float), s) : 0;
  if (p->loss) {
    distill_count_kernel<<<p->count ? count_blocks(*p) : 1, kCountThreads, 0, s>>>(*p);
    const int rc = (int)cudaGetLastError();
    if (rc) return rc;
  }
  return p->dlogits ? launch<true, true>(*p, p->loss != nullptr, s) : launch<true, false>(*p, p->loss != nullptr, s);
}

extern "C" int b200_distill_bwd(const B200Distill* p, void* stream) {
  if (!valid(p)) return (int)cudaErrorInvalidValue;
  return p->N > 0 ? launch<false, true>(*p, false, (cudaStream_t)stream) : 0;
}
