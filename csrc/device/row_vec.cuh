// Wide loads and stores of short vectors of fp32 / bf16 / fp16 elements, converted to fp32 in registers: shared by the
// per-row transformer kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace rowvec {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half(v); }

// N elements that start on a boundary of their own size (at most 16 bytes): one load or store instruction.
template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// Asynchronous copies of 16 bytes to shared memory; a thread waits for its own.
__device__ __forceinline__ void copy16_async(void* shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(shared)), "l"(global) : "memory");
}
// 4, 8 or 16 bytes, or zeros in their place.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* shared, const void* global, bool there) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(shared)), "l"(global), "r"(there ? 16 : 0)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"((unsigned)__cvta_generic_to_shared(shared)), "l"(global), "n"(BYTES),
                 "r"(there ? BYTES : 0)
                 : "memory");
}
// The same with a policy for L2.
__device__ __forceinline__ void copy16_async(void* shared, const void* global, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(shared)), "l"(global), "l"(policy)
               : "memory");
}
__device__ __forceinline__ uint64_t l2_evict_first() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t l2_evict_last() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

template <typename T, int N>
__device__ __forceinline__ void store(T* __restrict__ p, const float (&in)[N]) {
  Pack<T, N> raw;
#pragma unroll
  for (int k = 0; k < N; ++k) raw.v[k] = from_f32<T>(in[k]);
  *reinterpret_cast<Pack<T, N>*>(p) = raw;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Neighbouring elements of a pack as fp32, and back.
template <typename T, int N>
__device__ __forceinline__ float2 pair_of(const Pack<T, N>& p, int i) { return make_float2(to_f32<T>(p.v[2 * i]), to_f32<T>(p.v[2 * i + 1])); }
template <int N>
__device__ __forceinline__ float2 pair_of(const Pack<__nv_bfloat16, N>& p, int i) {  // the upper half of an fp32 number each
  const unsigned w = reinterpret_cast<const unsigned*>(&p)[i];
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <int N>
__device__ __forceinline__ float2 pair_of(const Pack<__half, N>& p, int i) { return __half22float2(reinterpret_cast<const __half2*>(&p)[i]); }
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float (&out)[N]) {
  if constexpr (N == 1) out[0] = to_f32<T>(p.v[0]);
  else {
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      const float2 v = pair_of(p, k);
      out[2 * k] = v.x;
      out[2 * k + 1] = v.y;
    }
  }
}
// The largest element (one that is no number counts only if all are).
template <int N>
__device__ __forceinline__ float max_of(const Pack<float, N>& p) {
  float m = p.v[0];
#pragma unroll
  for (int k = 1; k < N; ++k) m = fmaxf(m, p.v[k]);
  return m;
}
template <typename T2, typename T, int N>
__device__ __forceinline__ T2 max_pair(const Pack<T, N>& p) {
  const T2* w = reinterpret_cast<const T2*>(&p);
  T2 m = w[0];
#pragma unroll
  for (int k = 1; k < N / 2; ++k) m = __hmax2(m, w[k]);
  return m;
}
template <int N>
__device__ __forceinline__ float max_of(const Pack<__nv_bfloat16, N>& p) {
  const __nv_bfloat162 m = max_pair<__nv_bfloat162>(p);
  return fmaxf(__low2float(m), __high2float(m));
}
template <int N>
__device__ __forceinline__ float max_of(const Pack<__half, N>& p) {
  const __half2 m = max_pair<__half2>(p);
  return fmaxf(__low2float(m), __high2float(m));
}
template <int N>
__device__ __forceinline__ void set_pair(Pack<float, N>& p, int i, float2 v) { p.v[2 * i] = v.x; p.v[2 * i + 1] = v.y; }
template <int N>
__device__ __forceinline__ void set_pair(Pack<__nv_bfloat16, N>& p, int i, float2 v) {
  *reinterpret_cast<__nv_bfloat162*>(&p.v[2 * i]) = __float22bfloat162_rn(v);
}
template <int N>
__device__ __forceinline__ void set_pair(Pack<__half, N>& p, int i, float2 v) { *reinterpret_cast<__half2*>(&p.v[2 * i]) = __float22half2_rn(v); }

// 2^x; results below the smallest normal number become 0
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums over aligned groups of `width` lanes (a power of two up to 32); every lane of the warp takes part.
__device__ __forceinline__ float group_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float group_max(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

}  // namespace rowvec
