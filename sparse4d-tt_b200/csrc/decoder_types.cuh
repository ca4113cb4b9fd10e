// Element types of the decoder operators: f32, bf16 and f16 loads and stores of one 16-byte vector
// or one element, widened to fp32 registers.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "s4d_decoder.h"

namespace s4d {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements as fp32: VEC = 1, or the elements of one aligned 16-byte vector.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = to_f32<T>(*p);
  } else {
    static_assert(VEC * sizeof(T) == 16, "one 16-byte vector");
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f32<T>(e[i]);
  }
}

// The same in two steps, for loads that are to be under way while something else is computed.
template <typename T, int VEC>
struct RawVec {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void widen(float (&f)[VEC]) const {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f32<T>(e[i]);
  }
};
template <typename T>
struct RawVec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void clear() { v = from_f32<T>(0.0f); }
  __device__ __forceinline__ void widen(float (&f)[1]) const { f[0] = to_f32<T>(v); }
};

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(f[0]);
  } else {
    uint4 v;
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = v;
  }
}

// SMs of the current device (148 on B200 if the query fails), cached per device.
inline int device_sms() {
  static int cache[64] = {};
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  if (dev >= 0 && dev < 64 && cache[dev] > 0) return cache[dev];
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
    cudaGetLastError();
    return 148;
  }
  if (dev >= 0 && dev < 64) cache[dev] = sms;
  return sms;
}

}  // namespace s4d
