#pragma once

// Element access shared by the expert-layer kernels: 16-byte vectors of bf16 / f16 / f32 as fp32
// values, and one rounding back.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>

namespace kl::capi {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

template <class T>
constexpr int kPerVec = 16 / int(sizeof(T));  // elements of a 16-byte vector

template <class T>
__device__ __forceinline__ void unpack(uint4 u, float* v) {
  T t[kPerVec<T>];
  memcpy(t, &u, 16);
#pragma unroll
  for (int i = 0; i < kPerVec<T>; ++i) v[i] = to_f32(t[i]);
}

template <class T>
__device__ __forceinline__ uint4 pack(const float* v) {
  T t[kPerVec<T>];
#pragma unroll
  for (int i = 0; i < kPerVec<T>; ++i) t[i] = from_f32<T>(v[i]);
  uint4 u;
  memcpy(&u, t, 16);
  return u;
}

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// The 32-bit arrays of a call; NULL = not given.
inline bool words_aligned(std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (!aligned(p, 4)) return false;
  return true;
}
inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace kl::capi
