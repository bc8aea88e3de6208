// Element types of the norm and optimiser kernels: fp32, bf16 and fp16 in memory, fp32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "ptx.cuh"

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

// Two 16-bit elements of one word (the low one first) and back.
template <typename T>
__device__ __forceinline__ void unpack_word(uint32_t w, float& lo, float& hi);
template <>
__device__ __forceinline__ void unpack_word<__nv_bfloat16>(uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void unpack_word<__half>(uint32_t w, float& lo, float& hi) {
  __half2 h;
  memcpy(&h, &w, 4);
  const float2 f = __half22float2(h);
  lo = f.x;
  hi = f.y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack_word(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_word<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack_word<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }

// N consecutive elements at p, moved in accesses of up to 16 bytes (p is aligned to min(16, N * sizeof(T)) bytes).  The accesses are spelled out as
// words: a struct of 16-bit elements would be copied element by element.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[N]) {
  constexpr int BYTES = N * static_cast<int>(sizeof(T));
  if constexpr (N == 1) {
    f[0] = to_f32<T>(*p);
  } else {
    constexpr int WORDS = BYTES / 4;
    uint32_t w[WORDS];
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else if constexpr (BYTES == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else {
      static_assert(BYTES == 4, "access size");
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) unpack_word<T>(w[i], f[2 * i], f[2 * i + 1]);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[N]) {
  constexpr int BYTES = N * static_cast<int>(sizeof(T));
  if constexpr (N == 1) {
    *p = from_f32<T>(f[0]);
  } else {
    constexpr int WORDS = BYTES / 4;
    uint32_t w[WORDS];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = pack_word<T>(f[2 * i], f[2 * i + 1]);
    }
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
      static_assert(BYTES == 4, "access size");
      *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  }
}

// VEC consecutive elements as N numbers of type V: pairs of fp32 (two of them go through one packed instruction, which halves the issue slots of
// kernels with a dozen operations per 16-bit element), or one fp32 when VEC is 1.
template <int VEC>
struct Lanes {
  using V = uint64_t;
  static constexpr int N = VEC / 2;
};
template <>
struct Lanes<1> {
  using V = float;
  static constexpr int N = 1;
};
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ uint64_t vadd(uint64_t a, uint64_t b) { return add_f32x2(a, b); }
__device__ __forceinline__ uint64_t vmul(uint64_t a, uint64_t b) { return mul_f32x2(a, b); }
__device__ __forceinline__ uint64_t vfma(uint64_t a, uint64_t b, uint64_t c) { return fma_f32x2(a, b, c); }
__device__ __forceinline__ float vsum(float a) { return a; }
__device__ __forceinline__ float vsum(uint64_t a) {
  float lo, hi;
  unpack_f32x2(a, lo, hi);
  return lo + hi;
}
template <typename V>
__device__ __forceinline__ V vsplat(float a);
template <>
__device__ __forceinline__ float vsplat<float>(float a) { return a; }
template <>
__device__ __forceinline__ uint64_t vsplat<uint64_t>(float a) { return pack_f32x2(a, a); }

template <typename T, int VEC>
__device__ __forceinline__ void load_lanes(const T* p, typename Lanes<VEC>::V (&v)[Lanes<VEC>::N]) {
  float f[VEC];
  load_vec<T, VEC>(p, f);
  if constexpr (VEC == 1) {
    v[0] = f[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) v[i] = pack_f32x2(f[2 * i], f[2 * i + 1]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_lanes(T* p, const typename Lanes<VEC>::V (&v)[Lanes<VEC>::N]) {
  float f[VEC];
  if constexpr (VEC == 1) {
    f[0] = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) unpack_f32x2(v[i], f[2 * i], f[2 * i + 1]);
  }
  store_vec<T, VEC>(p, f);
}

}  // namespace b200k
