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

template <typename T, int N>
__device__ __forceinline__ void load(const T* __restrict__ p, float (&out)[N]) {
  const Pack<T, N> raw = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int k = 0; k < N; ++k) out[k] = to_f32<T>(raw.v[k]);
}
template <typename T, int N>
__device__ __forceinline__ void store(T* __restrict__ p, const float (&in)[N]) {
  Pack<T, N> raw;
#pragma unroll
  for (int k = 0; k < N; ++k) raw.v[k] = from_f32<T>(in[k]);
  *reinterpret_cast<Pack<T, N>*>(p) = raw;
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
