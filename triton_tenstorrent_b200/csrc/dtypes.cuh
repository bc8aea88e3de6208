// Element types of the norm and optimiser kernels: fp32, bf16 and fp16 in memory, fp32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200k {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// One rounding to nearest even.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements moved as one access (N * sizeof(T) is 2, 4, 8, 16 or 32 bytes; 32 bytes are two 16-byte accesses).
template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = to_f32<T>(p.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float (&f)[N]) {
  Pack<T, N> p;
#pragma unroll
  for (int i = 0; i < N; ++i) p.v[i] = from_f32<T>(f[i]);
  return p;
}

}  // namespace b200k
