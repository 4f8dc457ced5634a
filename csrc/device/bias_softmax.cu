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
// Table gradient: d is summed over distances first, far ones in two registers a thread, near ones in shared memory, in a copy for every
// group of lanes that walks over rows of its own.  In one row no two elements have the same distance, so no atomics are needed and the order
// of every sum is fixed: the same inputs give the same bits.  From one row to the next a lane's distances fall by one, so its sums
// stay in registers and move up a place, and one of eight reaches shared memory (16 x 12 x 512 x 512 bf16: 91 us when all did, 72 so).
//
// Measured on a B200, 2 x 12 x 2048 x 2048 bf16: without a mask forward 81 us = 5.0 TB/s, 0.76 of the measured copy bandwidth, backward 113 us for
// the scores alone and 118 us with the table = 5.1 TB/s, 0.78; with a causal mask of 16 bits 117 and 180 us.  128 x 12 x 128 x 128 bf16 with an
// fp32 padding mask: 38 and 70 us (2.6 and 2.1 TB/s), where every distance is a near one.  Issue slots are what it runs out of (68 % and 63 %
// busy at 2048 keys; 18 and 23 instructions an element), and unaligned fp32 rows of 517 keys with a random bool mask run at 1.2 to 1.5 TB/s
// for the same reason.  Rows beyond the registers read the scores twice in each direction: 12 x 1024 x 16384 bf16 270 us forward, 712 backward
// for the scores, 737 with the table (0.45 and 0.25 of the copy), 12 x 1024 x 8192 fp32 212, 430 and 445 us; 12 x 1024 x 8192 bf16, the
// longest in registers, 95, 119 and 148 us.
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
  long long elements;             // of s
  long long mk_b, mk_h, mk_i, mk_j;
  int table_dtype, mask_dtype;
  int H, Lq, Lk, offset;
  int reach, last;      // distances -reach .. last - reach have a slot each, farther ones the slot at their end
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
__host__ __device__ __forceinline__ int padded(int x) { return x + (x >> 5); }

// Words of shared memory: the table of biases, the sums over distances of every group; the rows on their way begin behind them on a
// 16-byte boundary.
__host__ __device__ __forceinline__ int lut_words(int last) { return (padded(last) + 1 + 3) & ~3; }
__host__ __device__ __forceinline__ int acc_words(int last, int groups) { return (groups * (padded(last) + 1) + 3) & ~3; }

// Called by the whole block; ends with a barrier.
__device__ __forceinline__ void fill_lut(float* lut, const Args& p, int h) {
  for (int x = threadIdx.x; x <= p.last; x += blockDim.x)
    lut[padded(x)] = scalar_at(p.table, (long long)bucket_of(x - p.reach, p.rb) * p.H + h, p.table_dtype);
  __syncthreads();
}

// Vectors of VEC elements (16 bytes) on 16-byte boundaries.  EDGE: rows may begin anywhere and have any length, so that the
// first and the last vector can reach over the row's ends; without it (rows begin on boundaries and have whole vectors) those tests are gone.
// FULL: besides, the row fills every vector of its lanes.
// The elements [j0, j0 + VEC) of a row; those outside [0, n) read as 0 and are not written.
template <typename T, int VEC, bool EDGE>
__device__ __forceinline__ Pack<T, VEC> load_part(const T* row, int j0, int n) {
  if (!EDGE || (j0 >= 0 && j0 + VEC <= n)) return *reinterpret_cast<const Pack<T, VEC>*>(row + j0);
  Pack<T, VEC> v;
#pragma unroll
  for (int k = 0; k < VEC; ++k) v.v[k] = j0 + k >= 0 && j0 + k < n ? row[j0 + k] : from_f32<T>(0.f);
  return v;
}
template <typename T, int VEC, bool EDGE>
__device__ __forceinline__ void store_part(T* row, int j0, int n, const Pack<T, VEC>& v) {
  if (!EDGE || (j0 >= 0 && j0 + VEC <= n)) {
    *reinterpret_cast<Pack<T, VEC>*>(row + j0) = v;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (j0 + k >= 0 && j0 + k < n) row[j0 + k] = v.v[k];
  }
}

// Adds a vector of the mask; excluded elements become -inf whatever they held, NaN too.  Returns whether there are any.  Most vectors
// of most masks (padding, causal) are all 0 or all -inf, which takes a few tests on their bits instead of four instructions an element.
__device__ __forceinline__ bool add_mask_pair(float2& a, float2 m) {
  const bool x = m.x == kNegInf, y = m.y == kNegInf;
  a = make_float2(x ? kNegInf : a.x + m.x, y ? kNegInf : a.y + m.y);
  return x || y;
}
template <int N>
__device__ __forceinline__ bool exclude_all(float2 (&a)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) a[k] = both(kNegInf);
  return true;
}
template <typename M> __device__ __forceinline__ unsigned neg_inf_word();
template <> __device__ __forceinline__ unsigned neg_inf_word<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ unsigned neg_inf_word<__nv_bfloat16>() { return 0xff80ff80u; }
template <> __device__ __forceinline__ unsigned neg_inf_word<__half>() { return 0xfc00fc00u; }
template <typename M, int VEC>
__device__ __forceinline__ bool add_mask_vector(const M* m, float2 (&a)[VEC / 2]) {
  constexpr int W = 16 / sizeof(M) < VEC ? 16 / sizeof(M) : VEC, P = VEC / W, WORDS = sizeof(Pack<M, W>) / 4;
  Pack<M, W> part[P];
  unsigned any = 0, other = 0;
#pragma unroll
  for (int o = 0; o < P; ++o) {
    part[o] = *reinterpret_cast<const Pack<M, W>*>(m + o * W);
    const unsigned* w = reinterpret_cast<const unsigned*>(&part[o]);
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      any |= w[k];
      other |= w[k] ^ neg_inf_word<M>();
    }
  }
  if (any == 0) return false;
  if (other == 0) return exclude_all(a);
  bool out = false;
#pragma unroll
  for (int o = 0; o < P; ++o) {
#pragma unroll
    for (int k = 0; k < W / 2; ++k) out |= add_mask_pair(a[o * W / 2 + k], pair_of(part[o], k));
  }
  return out;
}

// The mask of one row: where key 0 has its element, and whether the row's vectors lie on the boundaries of wide loads.
struct MaskRow {
  const char* key0;
  bool wide;
};
__device__ __forceinline__ int mask_bytes(int dtype) { return dtype == B200_F32 ? 4 : (dtype == B200_BF16 || dtype == B200_F16 ? 2 : 1); }
template <int VEC>
__device__ __forceinline__ MaskRow mask_row(const Args& p, long long at, int phase) {
  const int es = mask_bytes(p.mask_dtype);
  MaskRow m;
  m.key0 = static_cast<const char*>(p.mask) + at * es;
  m.wide = p.mk_j == 1 && ((reinterpret_cast<uintptr_t>(m.key0) - phase * es) & ((VEC * es < 16 ? VEC * es : 16) - 1)) == 0;
  return m;
}

// Adds the mask to the scores of [j0, j0 + VEC).  Returns whether it excludes any.
template <int VEC, bool EDGE>
__device__ __forceinline__ bool add_mask(const Args& p, const MaskRow& row, int j0, float2 (&a)[VEC / 2]) {
  if (row.wide && (!EDGE || (j0 >= 0 && j0 + VEC <= p.Lk))) {
    const char* m = row.key0 + (long long)j0 * mask_bytes(p.mask_dtype);  // (bytes pass 32 bits before keys do)
    if (p.mask_dtype == B200_F32) return add_mask_vector<float, VEC>(reinterpret_cast<const float*>(m), a);
    if (p.mask_dtype == B200_BF16) return add_mask_vector<__nv_bfloat16, VEC>(reinterpret_cast<const __nv_bfloat16*>(m), a);
    if (p.mask_dtype == B200_F16) return add_mask_vector<__half, VEC>(reinterpret_cast<const __half*>(m), a);
    const Pack<unsigned char, VEC> keep = *reinterpret_cast<const Pack<unsigned char, VEC>*>(m);
    const unsigned* w = reinterpret_cast<const unsigned*>(&keep);
    unsigned kept = w[0], any = w[0];
    if (VEC == 8) {
      kept &= w[VEC / 4 - 1];
      any |= w[VEC / 4 - 1];
    }
    if (kept == 0x01010101u) return false;
    if (any == 0) return exclude_all(a);
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) a[k] = make_float2(keep.v[2 * k] ? a[k].x : kNegInf, keep.v[2 * k + 1] ? a[k].y : kNegInf);
    return true;
  }
  bool out = false;
#pragma unroll
  for (int k = 0; k < VEC / 2; ++k) {
    const int j = j0 + 2 * k;
    float2 m = make_float2(0.f, 0.f);
    if (j >= 0 && j < p.Lk) m.x = scalar_at(row.key0, j * p.mk_j, p.mask_dtype);
    if (j + 1 >= 0 && j + 1 < p.Lk) m.y = scalar_at(row.key0, (j + 1) * p.mk_j, p.mask_dtype);
    out |= add_mask_pair(a[k], m);
  }
  return out;
}

// Scores to logits: scale, bias by distance, mask; -inf outside the row.  x0 = slot of the first element's distance.  Returns
// whether any element is excluded.
template <typename T, int VEC, bool MASKED, bool EDGE>
__device__ __forceinline__ bool to_logits(const Args& p, const float* lut, const MaskRow& mask, int j0, int x0, const Pack<T, VEC>& s, float2 (&a)[VEC / 2]) {
  const int last = p.last;
  const float2 scale = both(p.scale);
  if (x0 >= last || x0 + VEC - 1 <= 0) {  // all as far as the bias tells apart
    const float2 b = both(lut[x0 > 0 ? padded(last) : 0]);
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) a[k] = fma2(pair_of(s, k), scale, b);
  } else {
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) {
      const int x = x0 + 2 * k;
      a[k] = fma2(pair_of(s, k), scale, make_float2(lut[padded(min(max(x, 0), last))], lut[padded(min(max(x + 1, 0), last))]));
    }
  }
  bool out = false;
  if (MASKED) out = add_mask<VEC, EDGE>(p, mask, j0, a);
  if (EDGE && (j0 < 0 || j0 + VEC > p.Lk)) {
    out = true;
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) {
      const int j = j0 + 2 * k;
      if (j < 0 || j >= p.Lk) a[k].x = kNegInf;
      if (j + 1 < 0 || j + 1 >= p.Lk) a[k].y = kNegInf;
    }
  }
  return out;
}

// e^(a - m).  The difference comes first: a and m may be as large as the type allows (a mask of its lowest value on a whole row).
// a = -inf gives 0 as long as m is finite, see finite_max.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float weight_of(float a, float m) { return exp2_fast((a - m) * kLog2e); }
__device__ __forceinline__ float2 weights_of(float2 a, float2 minus_m) {
  const float2 t = mul2(add2(a, minus_m), both(kLog2e));
  return make_float2(exp2_fast(t.x), exp2_fast(t.y));
}
__device__ __forceinline__ float finite_max(float m) { return m == kNegInf ? 0.f : m; }
// 1 / sum, 0 for a row with nothing left (a NaN stays one)
__device__ __forceinline__ float inverse_sum(float sum) { return sum == 0.f ? 0.f : __fdividef(1.f, sum); }
template <int N>
__device__ __forceinline__ float max_of(float m, const float2 (&a)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) m = fmaxf(m, fmaxf(a[k].x, a[k].y));
  return m;
}

// d to the table gradient's sums over distances
template <int VEC>
__device__ __forceinline__ void add_distances(float* acc, int last, int x0, const float2 (&d)[VEC / 2], float& below, float& above) {
  if (x0 >= last || x0 + VEC - 1 <= 0) {
    float2 t = d[0];
#pragma unroll
    for (int k = 1; k < VEC / 2; ++k) t = add2(t, d[k]);
    if (x0 > 0) above += t.x + t.y; else below += t.x + t.y;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int x = x0 + k;
      const float v = k % 2 ? d[k / 2].y : d[k / 2].x;
      if (x <= 0) below += v;
      else if (x >= last) above += v;
      else acc[padded(x)] += v;
    }
  }
}

// One sum of a distance to where it belongs.
__device__ __forceinline__ void add_distance(float* acc, int last, int x, float v, float& below, float& above) {
  if (x <= 0) below += v;
  else if (x >= last) above += v;
  else acc[padded(x)] += v;
}

// Walks over the rows (b, i) of a head.
struct RowWalk {
  unsigned i;
  int h;
  long long at, mask, stat;  // where the row's scores, mask and statistics begin
  __device__ __forceinline__ RowWalk(const Args& p, unsigned r, int head) : i(r % (unsigned)p.Lq), h(head) {
    const unsigned b = r / (unsigned)p.Lq;
    at = b * p.st_b + h * p.st_h + i * p.st_i;
    mask = b * p.mk_b + h * p.mk_h + i * p.mk_i;
    stat = ((long long)b * p.H + h) * p.Lq + i;
  }
  __device__ __forceinline__ void advance(const Args& p, unsigned step) {
    i += step;
    at += step * p.st_i;
    mask += step * p.mk_i;
    stat += step;
    while (i >= (unsigned)p.Lq) {
      i -= (unsigned)p.Lq;
      at += p.st_b - p.Lq * p.st_i;
      mask += p.mk_b - p.Lq * p.mk_i;
      stat += (long long)(p.H - 1) * p.Lq;
    }
  }
  __device__ __forceinline__ int first_x(const Args& p) const { return p.reach - p.offset - (int)i; }  // slot of key 0's distance
};

// (maximum, sum) of the lanes of one row.  WARPS = 1: the row belongs to a group of G lanes.  WARPS > 1: to the block, whose warps
// meet once in shared memory, in one of two places in turn, so that one barrier a row is enough.
template <int WARPS>
__device__ __forceinline__ float2 join_rows(float m, float sum, int G, float2 (*sh)[WARPS], int turn) {
  if (WARPS == 1) return make_float2(m, sum);  // m is the group's already
  if ((threadIdx.x & 31) == 0) sh[turn][threadIdx.x >> 5] = make_float2(m, sum);
  __syncthreads();
  float top = kNegInf, all = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sh[turn][w].x);
  const float t = finite_max(top);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const float2 o = sh[turn][w];
    all += o.y * weight_of(o.x, t);  // a warp without keys: 0 times 0; one with a NaN score: NaN
  }
  return make_float2(top, all);
}

// Rows on their way: each thread copies its vectors of the next rows to a place of its own in shared memory, so that several
// kilobytes for every block are under way while a row is worked on, at no registers.  An EDGE vector is copied whole, neighbours' elements
// and all, as long as it lies in the tensor; the very last one of the tensor may not and is read element by element when its turn comes.
// (2 x 12 x 2048 x 2048 bf16: forward 94 us with the next row in registers, 82 us so; three rows ahead forward, two backward.)
constexpr int ring_depth(int nv, bool bwd) { return nv == 1 ? 4 : (nv == 2 ? (bwd ? 3 : 4) : 2); }
template <typename T, int VEC, int NV, bool EDGE, bool FULL>
struct RowVectors {
  static __device__ __forceinline__ int phase_of(const T* row) { return EDGE ? (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (VEC - 1)) : 0; }
  // this thread's vectors of a row to slots `blockDim.x` apart
  static __device__ __forceinline__ void fetch(const T* base, long long elements, long long at, int Lk, int gl, int lanes, Pack<T, VEC>* slot) {
    const int phase = phase_of(base + at);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * lanes) * VEC - phase;
      if ((FULL || j0 < Lk) && (!EDGE || at + j0 + VEC <= elements)) copy16_async(slot + n * blockDim.x, base + at + j0);
    }
  }
  static __device__ __forceinline__ void take(const T* base, long long elements, long long at, int Lk, int gl, int lanes, const Pack<T, VEC>* slot,
                                              Pack<T, VEC> (&v)[NV]) {
    const int phase = phase_of(base + at);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * lanes) * VEC - phase;
      if (FULL || j0 < Lk) {
        if (!EDGE || at + j0 + VEC <= elements) v[n] = slot[n * blockDim.x];
        else v[n] = load_part<T, VEC, true>(base + at, j0, Lk);
      }
    }
  }
};

// Registers: 64 a thread forward hold 16 elements of a lane and leave 1024 threads for an SM, 80 backward 768; where a row belongs to a
// part of a warp 96 and 640, in smaller blocks.  Left alone, the compiler takes 120 for the loads of a mask whose keys are not side by
// side, which is the rare case.
constexpr int row_threads(int warps, bool bwd) { return warps == 1 ? (bwd ? 128 : kMaxThreads) : 32 * warps; }
constexpr int resident_threads(int warps, bool bwd) { return bwd ? (warps == 1 ? 640 : 768) : 1024; }
constexpr int row_blocks(int elements, int warps, bool bwd) {
  return elements <= 16 ? resident_threads(warps, bwd) / row_threads(warps, bwd) : 1;
}

// A row in registers: NV vectors of VEC elements for each of its lanes (a group of G of one warp, or the block's WARPS warps).
template <typename T, int VEC, int NV, int WARPS, bool MASKED, bool EDGE, bool FULL>
__global__ void __launch_bounds__(row_threads(WARPS, false), row_blocks(NV * VEC, WARPS, false)) bias_softmax_fwd_rows(const __grid_constant__ Args p) {
  extern __shared__ __align__(16) float lut[];
  __shared__ float2 meet[2][WARPS];
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  const int G = WARPS == 1 ? p.group : 32, lanes = G * WARPS;
  const int gl = WARPS == 1 ? threadIdx.x & (G - 1) : threadIdx.x, groups = WARPS == 1 ? blockDim.x / G : 1;
  const unsigned r0 = part * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
  const unsigned r = WARPS == 1 ? r0 + threadIdx.x / G : r0;
  using Vectors = RowVectors<T, VEC, NV, EDGE, FULL>;
  constexpr int kDepth = ring_depth(NV, false);
  const T* base = static_cast<const T*>(p.s);
  Pack<T, VEC>* ring = reinterpret_cast<Pack<T, VEC>*>(lut + lut_words(p.last)) + threadIdx.x;
  RowWalk row(p, min(r, p.rows - 1), h), ahead = row;  // a group behind the last row follows on rows that are there
  unsigned fetched = 0;
  auto fetch_next = [&](int stage) {
    if (r + fetched < r1) {
      Vectors::fetch(base, p.elements, ahead.at, p.Lk, gl, lanes, ring + stage * NV * blockDim.x);
      fetched += groups;
      if (r + fetched < r1) ahead.advance(p, groups);
    }
    copies_commit();
  };
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fetch_next(d);
  fill_lut(lut, p, h);
  int turn = 0, stage = 0;
  for (unsigned done = 0; r0 + done < r1; done += groups, turn ^= 1) {
    const bool live = r + done < r1;
    fetch_next(stage == 0 ? kDepth - 1 : stage - 1);
    copies_wait<kDepth - 1>();
    Pack<T, VEC> raw[NV];
    Vectors::take(base, p.elements, row.at, p.Lk, gl, lanes, ring + stage * NV * blockDim.x, raw);
    stage = stage == kDepth - 1 ? 0 : stage + 1;
    const int phase = Vectors::phase_of(base + row.at);
    const MaskRow mask = MASKED ? mask_row<VEC>(p, row.mask, phase) : MaskRow{};
    const int first_x = row.first_x(p);
    float2 a[NV][VEC / 2];
    float m = kNegInf;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * lanes) * VEC - phase;
      if (FULL || j0 < p.Lk) {
        to_logits<T, VEC, MASKED, EDGE>(p, lut, mask, j0, first_x + j0, raw[n], a[n]);
        m = max_of(m, a[n]);
      }
    }
    m = group_max(m, G);
    const float2 minus = both(-finite_max(m));
    float2 sum2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if (FULL || (gl + n * lanes) * VEC - phase < p.Lk) {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          a[n][k] = weights_of(a[n][k], minus);
          sum2 = add2(sum2, a[n][k]);
        }
      }
    }
    const float2 all = join_rows<WARPS>(m, group_sum(sum2.x + sum2.y, G), G, meet, turn);
    const float inv = inverse_sum(all.y), f = WARPS == 1 ? inv : inv * weight_of(m, finite_max(all.x));
    if (live) {
      T* o = static_cast<T*>(p.out) + row.at;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int j0 = (gl + n * lanes) * VEC - phase;
        if (FULL || j0 < p.Lk) {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) set_pair(raw[n], k, mul2(a[n][k], both(f)));
          store_part<T, VEC, EDGE>(o, j0, p.Lk, raw[n]);
        }
      }
      if (p.stats && gl == 0) p.stats[row.stat] = make_float2(finite_max(all.x), inv);
      if (r + done + groups < r1) row.advance(p, groups);
    }
  }
}

template <int WARPS>
__device__ __forceinline__ float join_sums(float v, float (*sh)[WARPS], int turn) {
  if (WARPS == 1) return v;
  if ((threadIdx.x & 31) == 0) sh[turn][threadIdx.x >> 5] = v;
  __syncthreads();
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) all += sh[turn][w];
  return all;
}

// The sums over distances of a block, to its place among the partial sums.
__device__ __forceinline__ void write_partial(const Args& p, float* all, int groups, int words, float* acc, int h, int part, float below, float above,
                                              bool first_lane) {
  if (first_lane) {  // the slots of the two ends are used for nothing else
    acc[padded(0)] = below;
    acc[padded(p.last)] = above;
  }
  __syncthreads();
  float* out = p.partial + ((long long)h * p.blocks_per_head + part) * (p.last + 1);
  for (int x = threadIdx.x; x <= p.last; x += blockDim.x) {
    float t = 0.f;
    for (int q = 0; q < groups; ++q) t += all[q * words + padded(x)];
    out[x] = t;
  }
}

// Sum over a block for a last step, with two barriers.
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = group_sum(v, 32);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = group_sum(threadIdx.x % 32 < blockDim.x / 32 ? sh[threadIdx.x % 32] : 0.f, 32);
  __syncthreads();
  return v;
}

template <typename T, int VEC, int NV, int WARPS, bool MASKED, bool EDGE, bool FULL>
__global__ void __launch_bounds__(row_threads(WARPS, true), row_blocks(NV * VEC, WARPS, true)) bias_softmax_bwd_rows(const __grid_constant__ Args p) {
  extern __shared__ __align__(16) float lut[];
  __shared__ float meet[2][WARPS];
  __shared__ float red[32];
  const int words = padded(p.last) + 1;
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  const int G = WARPS == 1 ? p.group : 32, lanes = G * WARPS;
  const int gl = WARPS == 1 ? threadIdx.x & (G - 1) : threadIdx.x, groups = WARPS == 1 ? blockDim.x / G : 1;
  float* all = lut + lut_words(p.last);
  float* acc = all + (WARPS == 1 ? (threadIdx.x / G) * words : 0);
  float below = 0.f, above = 0.f;
  // Every group takes rows that follow one another, so that an element's distance falls by one from row to row: between whole rows the
  // sums of a vector's distances stay in registers and move up by one place, and only the one that leaves at the end goes to shared memory.
  const unsigned each = p.rows_per_block / groups, begin = part * p.rows_per_block;
  const unsigned r0 = WARPS == 1 ? begin + threadIdx.x / G * each : begin;
  const unsigned r1 = min(r0 + each, p.rows), r = r0;
  float held[NV][VEC];
  int held_x = 0;  // slot of key 0's distance in the row that the sums stand for
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int k = 0; k < VEC; ++k) held[n][k] = 0.f;
  auto put_away = [&] {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * lanes) * VEC;
      if (FULL || j0 < p.Lk) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          add_distance(acc, p.last, held_x + j0 + k, held[n][k], below, above);
          held[n][k] = 0.f;
        }
      }
    }
  };
  using Vectors = RowVectors<T, VEC, NV, EDGE, FULL>;
  constexpr int kDepth = ring_depth(NV, true);
  const T* base = static_cast<const T*>(p.s);
  const T* gbase = static_cast<const T*>(p.g);
  Pack<T, VEC>* ring = reinterpret_cast<Pack<T, VEC>*>(lut + lut_words(p.last) + acc_words(p.last, groups)) + threadIdx.x;
  RowWalk row(p, min(r, p.rows - 1), h), ahead = row;
  unsigned fetched = 0;
  auto fetch_next = [&](int stage) {
    if (r + fetched < r1) {
      Vectors::fetch(base, p.elements, ahead.at, p.Lk, gl, lanes, ring + stage * 2 * NV * blockDim.x);
      Vectors::fetch(gbase, p.elements, ahead.at, p.Lk, gl, lanes, ring + (stage * 2 + 1) * NV * blockDim.x);
      ++fetched;
      if (r + fetched < r1) ahead.advance(p, 1);
    }
    copies_commit();
  };
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fetch_next(d);
  float2 st_next = p.stats[row.stat];
  if (p.partial)
    for (int x = threadIdx.x; x < groups * words; x += blockDim.x) all[x] = 0.f;
  fill_lut(lut, p, h);
  int turn = 0, stage = 0;
  for (unsigned done = 0; done < each && begin + done < p.rows; ++done, turn ^= 1) {
    const bool live = r + done < r1;
    const RowWalk now = row;
    const float2 st = st_next;
    if (r + done + 1 < r1) {
      row.advance(p, 1);
      st_next = p.stats[row.stat];
    }
    fetch_next(stage == 0 ? kDepth - 1 : stage - 1);
    copies_wait<kDepth - 1>();
    Pack<T, VEC> raw[NV], graw[NV];  // the gradient waits in its own type: half the registers for 16 bits
    Vectors::take(base, p.elements, now.at, p.Lk, gl, lanes, ring + stage * 2 * NV * blockDim.x, raw);
    Vectors::take(gbase, p.elements, now.at, p.Lk, gl, lanes, ring + (stage * 2 + 1) * NV * blockDim.x, graw);
    stage = stage == kDepth - 1 ? 0 : stage + 1;
    const int phase = Vectors::phase_of(base + now.at);
    const MaskRow mask = MASKED ? mask_row<VEC>(p, now.mask, phase) : MaskRow{};
    const int first_x = now.first_x(p);
    float2 a[NV][VEC / 2], dot2 = make_float2(0.f, 0.f);
    int excluded = 0;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int j0 = (gl + n * lanes) * VEC - phase;
      if (FULL || j0 < p.Lk) {
        const bool out = to_logits<T, VEC, MASKED, EDGE>(p, lut, mask, j0, first_x + j0, raw[n], a[n]);
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) a[n][k] = mul2(weights_of(a[n][k], both(-st.x)), both(st.y));
        if ((MASKED || EDGE) && out) {  // an excluded key counts nothing, whatever its gradient holds
          excluded |= 1 << n;
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            if ((k % 2 ? a[n][k / 2].y : a[n][k / 2].x) == 0.f) graw[n].v[k] = from_f32<T>(0.f);
        }
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) dot2 = fma2(a[n][k], pair_of(graw[n], k), dot2);
      }
    }
    // (with its barrier this row's sums over distances come behind the last row's)
    const float2 dot = both(-join_sums<WARPS>(group_sum(dot2.x + dot2.y, G), meet, turn));
    if (live) {
      T* o = static_cast<T*>(p.out) + now.at;
      const bool sums = p.partial != nullptr;
      if (!EDGE && sums && now.i == 0) put_away();  // another sequence: distances begin anew
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int j0 = (gl + n * lanes) * VEC - phase;
        if (FULL || j0 < p.Lk) {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) {
            const float2 d = mul2(a[n][k], add2(pair_of(graw[n], k), dot));
            if ((MASKED || EDGE) && (excluded >> n & 1)) a[n][k] = make_float2(a[n][k].x == 0.f ? 0.f : d.x, a[n][k].y == 0.f ? 0.f : d.y);
            else a[n][k] = d;
            set_pair(raw[n], k, mul2(a[n][k], both(p.scale)));
          }
          store_part<T, VEC, EDGE>(o, j0, p.Lk, raw[n]);
          if (EDGE && sums) add_distances<VEC>(acc, p.last, first_x + j0, a[n], below, above);
          if (!EDGE && sums) {
            add_distance(acc, p.last, held_x + j0 + VEC - 1, held[n][VEC - 1], below, above);
#pragma unroll
            for (int k = VEC - 1; k > 0; --k) held[n][k] = held[n][k - 1] + (k % 2 ? a[n][k / 2].y : a[n][k / 2].x);
            held[n][0] = a[n][0].x;
          }
        }
      }
      held_x = first_x;
    }
    if (WARPS == 1) __syncwarp();  // the next row of this group adds to the same sums from other lanes
  }
  if (!p.partial) return;
  if (!EDGE) {
    if (WARPS > 1) __syncthreads();  // behind the last row's
    put_away();
  }
  below = WARPS == 1 ? group_sum(below, G) : block_sum(below, red);
  above = WARPS == 1 ? group_sum(above, G) : block_sum(above, red);
  write_partial(p, all, groups, words, acc, h, part, below, above, gl == 0);
}

// A row to a whole block, any length: two passes over the row, of which the second finds it in the caches.
__device__ __forceinline__ float block_max(float v, float* sh) {
  v = group_max(v, 32);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = group_max(threadIdx.x % 32 < blockDim.x / 32 ? sh[threadIdx.x % 32] : kNegInf, 32);
  __syncthreads();
  return v;
}

template <typename T, int VEC, bool MASKED>
__global__ void __launch_bounds__(kMaxThreads) bias_softmax_fwd_long(const __grid_constant__ Args p) {
  extern __shared__ __align__(16) float lut[];
  __shared__ float sh[32];
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  fill_lut(lut, p, h);
  const unsigned r0 = part * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
  RowWalk walk(p, r0, h);
  for (unsigned r = r0; r < r1; ++r, walk.advance(p, 1)) {
    const T* s = static_cast<const T*>(p.s) + walk.at;
    const int phase = (int)((reinterpret_cast<uintptr_t>(s) / sizeof(T)) & (VEC - 1));
    const MaskRow mask = MASKED ? mask_row<VEC>(p, walk.mask, phase) : MaskRow{};
    const int first_x = walk.first_x(p);
    float m = kNegInf, sum = 0.f;
    for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.Lk; j0 += blockDim.x * VEC) {
      float2 a[VEC / 2], sum2 = make_float2(0.f, 0.f);
      to_logits<T, VEC, MASKED, true>(p, lut, mask, j0, first_x + j0, load_part<T, VEC, true>(s, j0, p.Lk), a);
      const float top = max_of(kNegInf, a);
      if (top > m) {
        sum *= weight_of(m, top);  // m = -inf: 0
        m = top;
      }
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) sum2 = add2(sum2, weights_of(a[k], both(-finite_max(m))));
      sum += sum2.x + sum2.y;
    }
    const float all = finite_max(block_max(m, sh));
    sum = block_sum(sum * weight_of(m, all), sh);
    const float inv = inverse_sum(sum);
    T* o = static_cast<T*>(p.out) + walk.at;
    for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.Lk; j0 += blockDim.x * VEC) {
      float2 a[VEC / 2];
      Pack<T, VEC> raw = load_part<T, VEC, true>(s, j0, p.Lk);
      to_logits<T, VEC, MASKED, true>(p, lut, mask, j0, first_x + j0, raw, a);
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) set_pair(raw, k, mul2(weights_of(a[k], both(-all)), both(inv)));
      store_part<T, VEC, true>(o, j0, p.Lk, raw);
    }
    if (p.stats && threadIdx.x == 0) p.stats[walk.stat] = make_float2(all, inv);
  }
}

template <typename T, int VEC, bool MASKED>
__global__ void __launch_bounds__(kMaxThreads) bias_softmax_bwd_long(const __grid_constant__ Args p) {
  extern __shared__ __align__(16) float lut[];
  __shared__ float sh[32];
  const int words = padded(p.last) + 1;
  const int h = blockIdx.x / p.blocks_per_head, part = blockIdx.x % p.blocks_per_head;
  float* acc = lut + lut_words(p.last);
  if (p.partial)
    for (int x = threadIdx.x; x < words; x += blockDim.x) acc[x] = 0.f;
  fill_lut(lut, p, h);
  float below = 0.f, above = 0.f;
  const unsigned r0 = part * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.rows);
  RowWalk walk(p, r0, h);
  for (unsigned r = r0; r < r1; ++r, walk.advance(p, 1)) {
    const T* s = static_cast<const T*>(p.s) + walk.at;
    const T* g = static_cast<const T*>(p.g) + walk.at;
    const int phase = (int)((reinterpret_cast<uintptr_t>(s) / sizeof(T)) & (VEC - 1));
    const MaskRow mask = MASKED ? mask_row<VEC>(p, walk.mask, phase) : MaskRow{};
    const int first_x = walk.first_x(p);
    const float2 st = p.stats[walk.stat];
    float dot = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      T* o = static_cast<T*>(p.out) + walk.at;
      float2 dot2 = make_float2(0.f, 0.f);
      for (int j0 = (int)threadIdx.x * VEC - phase; j0 < p.Lk; j0 += blockDim.x * VEC) {
        float2 a[VEC / 2];
        Pack<T, VEC> raw = load_part<T, VEC, true>(s, j0, p.Lk);
        const Pack<T, VEC> graw = load_part<T, VEC, true>(g, j0, p.Lk);
        to_logits<T, VEC, MASKED, true>(p, lut, mask, j0, first_x + j0, raw, a);
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          const float2 q = mul2(weights_of(a[k], both(-st.x)), both(st.y));
          float2 d = mul2(q, add2(pair_of(graw, k), both(-dot)));  // first pass: dot = 0
          if (MASKED) d = make_float2(q.x == 0.f ? 0.f : d.x, q.y == 0.f ? 0.f : d.y);
          dot2 = add2(dot2, d);
          a[k] = d;
          set_pair(raw, k, mul2(d, both(p.scale)));
        }
        if (pass) {
          store_part<T, VEC, true>(o, j0, p.Lk, raw);
          if (p.partial) add_distances<VEC>(acc, p.last, first_x + j0, a, below, above);
        }
      }
      if (!pass) dot = block_sum(dot2.x + dot2.y, sh);  // its barriers also order this row's sums over distances behind the last row's
    }
  }
  if (!p.partial) return;
  below = block_sum(below, sh);
  above = block_sum(above, sh);
  write_partial(p, acc, 1, words, acc, h, part, below, above, threadIdx.x == 0);
}

// One block per head and bucket: sums over the blocks' partial sums for the distances of the bucket, in a fixed order.  A
// bucket's distances are neighbours, so its slots are one run [x0, x1].
__global__ void __launch_bounds__(kMaxThreads) bias_table_grad(const float* partial, int blocks, int reach, int last, const __grid_constant__ B200RelativeBuckets rb,
                                                               int H, void* out, int dtype) {
  __shared__ float sh[32];
  const int h = blockIdx.x, bucket = blockIdx.y, slots = last + 1;
  const bool upper = rb.bidirectional && bucket >= rb.per_side;
  const int c = upper ? bucket - rb.per_side : bucket, far = c - rb.exact;
  int lo = far >= 0 ? rb.first[far] : c;
  int hi = c == rb.per_side - 1 ? reach : (far >= 0 ? rb.first[far + 1] : c + 1) - 1;
  if (upper && lo == 0) lo = 1;  // distance 0 belongs to the lower half
  hi = min(hi, reach);
  const int x0 = upper ? reach + lo : reach - hi, x1 = upper ? reach + hi : reach - lo;
  float t = 0.f;
  if (lo <= hi) {
    const float* mine = partial + (long long)h * blocks * slots + x0;
    const int run = x1 - x0 + 1, wide = run < (int)blockDim.x ? run : (int)blockDim.x, rows = blockDim.x / wide;
    const int x = threadIdx.x % wide, row = threadIdx.x / wide;
    if (row < rows) {
      for (int i = x; i < run; i += wide) {
#pragma unroll 8
        for (int b = row; b < blocks; b += rows) t += mine[(long long)b * slots + i];
      }
    }
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
  int threads, nv, warps;  // nv 0: any length
  bool edge, full;
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
  a.elements = (long long)p.B * p.H * p.Lq * p.Lk;
  // beyond the farthest distance of this call nothing has to be told apart either, nor after the query if those keys
  // share a bucket
  const long long ahead = (long long)p.Lk - 1 - p.query_offset, behind = (long long)p.Lq - 1 + p.query_offset;
  long long far = ahead > behind ? ahead : behind;
  if (far < -ahead) far = -ahead;
  if (far < -behind) far = -behind;
  a.reach = (int)(far + 1 < p.buckets.max_distance ? far + 1 : p.buckets.max_distance);
  a.last = p.buckets.bidirectional ? 2 * a.reach : a.reach;
  const int vec = p.dtype == B200_F32 ? 4 : 8;
  const bool aligned = p.Lk % vec == 0 && p.stride[0] % vec == 0 && p.stride[1] % vec == 0 && p.stride[2] % vec == 0;
  const int nvec = aligned ? p.Lk / vec : (p.Lk + 2 * vec - 2) / vec;  // an unaligned row may touch one vector more
  const int words = padded(a.last) + 1;
  pl.edge = !aligned;
  pl.threads = kMaxThreads;
  pl.warps = 1;
  if (nvec <= 32 * (16 / vec)) pl.threads = row_threads(1, bwd);
  int groups = 1;
  // 16 elements in a lane: fewer and the reductions and addresses of a row are too much for them, more and there are too few rows at once
  // (2048 keys in one / two / four / eight warps, before rows were copied ahead: forward 184 / 112 / 107 / 138 us, backward 530 / 271 / 172 /
  // 184 us).  Rows beyond eight warps of these take 32 elements a lane, and beyond 8192 keys of 16 bits (4096 of 32) two passes.
  const int wide = 16 / vec;  // vectors for 16 elements
  if (nvec <= 32 * wide) {
    int G = 1;
    while (G * wide < nvec) G <<= 1;
    if (bwd)  // sums over distances for each group: wider groups where there would be too many
      while (G < 32 && (pl.threads / G) * words * 4 > 32 * 1024) G <<= 1;
    a.group = G;
    const int nv = (nvec + G - 1) / G;
    pl.nv = nv <= 1 ? 1 : (nv <= 2 ? 2 : 4);
    if (bwd)
      while (pl.threads > 32 && (pl.threads / G + 1) * words * 4 > 96 * 1024) pl.threads >>= 1;
    groups = pl.threads / G;
  } else if (nvec <= kMaxThreads * 4) {
    pl.nv = nvec <= kMaxThreads * wide ? wide : 4;
    pl.warps = 2;
    while (pl.warps * 32 * pl.nv < nvec) pl.warps *= 2;
    pl.threads = 32 * pl.warps;
  }
  pl.full = aligned && nvec == pl.nv * (pl.warps == 1 ? a.group : pl.threads);
  pl.smem = (size_t)lut_words(a.last) * 4 + (bwd ? acc_words(a.last, groups) * 4 : 0) +
            (size_t)(pl.nv ? ring_depth(pl.nv, bwd) * pl.nv * pl.threads * 16 * (bwd ? 2 : 1) : 0);
  // One wave of blocks: each has to build its table of biases first, and what it leaves for the table gradient has to be added up.
  int resident = resident_threads(pl.warps, bwd) / pl.threads;
  const int by_smem = (int)(220 * 1024 / (pl.smem + 1536));
  if (resident > by_smem) resident = by_smem > 0 ? by_smem : 1;
  long long blocks = 148LL * resident / (p.H > 0 ? p.H : 1);
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
  if (pl.smem > 48 * 1024 - 512) {  // beside the static part
    // the same limit in every call: another thread may be between this and its launch
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    if (e != cudaSuccess) return (int)e;
  }
  kernel<<<(unsigned)(pl.a.blocks_per_head * pl.a.H), pl.threads, pl.smem, s>>>(pl.a);
  return (int)cudaGetLastError();
}

template <typename T, int VEC, int NV, int WARPS, bool MASKED, bool EDGE, bool FULL, bool BWD>
int launch_row(const Plan& pl, cudaStream_t s) {
  return BWD ? launch(bias_softmax_bwd_rows<T, VEC, NV, WARPS, MASKED, EDGE, FULL>, pl, s)
             : launch(bias_softmax_fwd_rows<T, VEC, NV, WARPS, MASKED, EDGE, FULL>, pl, s);
}
template <typename T, int VEC, int NV, int WARPS, bool BWD, bool MASKED>
int launch_rows(const Plan& pl, cudaStream_t s) {
  if (pl.full) return launch_row<T, VEC, NV, WARPS, MASKED, false, true, BWD>(pl, s);
  if (pl.edge) return launch_row<T, VEC, NV, WARPS, MASKED, true, false, BWD>(pl, s);
  return launch_row<T, VEC, NV, WARPS, MASKED, false, false, BWD>(pl, s);
}
template <typename T, int VEC, bool BWD, bool MASKED>
int dispatch(const Plan& pl, cudaStream_t s) {
  constexpr int kWide = 16 / VEC;
  if (pl.nv == 0) return BWD ? launch(bias_softmax_bwd_long<T, VEC, MASKED>, pl, s) : launch(bias_softmax_fwd_long<T, VEC, MASKED>, pl, s);
  if (pl.warps == 1) {
    if (pl.nv == 1) return launch_rows<T, VEC, 1, 1, BWD, MASKED>(pl, s);
    if (pl.nv == 2) return launch_rows<T, VEC, 2, 1, BWD, MASKED>(pl, s);
    return launch_rows<T, VEC, kWide, 1, BWD, MASKED>(pl, s);  // kWide = 2: not reached
  }
  if (pl.nv != kWide) return launch_rows<T, VEC, 4, 8, BWD, MASKED>(pl, s);
  if (pl.warps == 2) return launch_rows<T, VEC, kWide, 2, BWD, MASKED>(pl, s);
  if (pl.warps == 4) return launch_rows<T, VEC, kWide, 4, BWD, MASKED>(pl, s);
  return launch_rows<T, VEC, kWide, 8, BWD, MASKED>(pl, s);
}
template <bool BWD>
int dispatch_type(const Plan& pl, int dtype, cudaStream_t s) {
  const bool masked = pl.a.mask != nullptr;
  if (dtype == B200_BF16) return masked ? dispatch<__nv_bfloat16, 8, BWD, true>(pl, s) : dispatch<__nv_bfloat16, 8, BWD, false>(pl, s);
  if (dtype == B200_F16) return masked ? dispatch<__half, 8, BWD, true>(pl, s) : dispatch<__half, 8, BWD, false>(pl, s);
  if (dtype == B200_F32) return masked ? dispatch<float, 4, BWD, true>(pl, s) : dispatch<float, 4, BWD, false>(pl, s);
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
  return dispatch_type<false>(make_plan(*p, false), p->dtype, (cudaStream_t)stream);
}

extern "C" long long b200_bias_softmax_workspace(const B200BiasSoftmax* p) {
  if (!valid(p) || empty(p) || !p->dtable) return 0;
  const Plan pl = make_plan(*p, true);
  return (long long)p->H * pl.a.blocks_per_head * (pl.a.last + 1) * (long long)sizeof(float);
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
  const int rc = dispatch_type<true>(pl, p->dtype, s);
  if (rc || !p->dtable) return rc;
  const int buckets = p->buckets.per_side * (p->buckets.bidirectional ? 2 : 1);
  bias_table_grad<<<dim3((unsigned)p->H, (unsigned)buckets), kMaxThreads, 0, s>>>(pl.a.partial, pl.a.blocks_per_head, pl.a.reach, pl.a.last, p->buckets, p->H,
                                                                                p->dtable, p->table_dtype);
  return (int)cudaGetLastError();
}
