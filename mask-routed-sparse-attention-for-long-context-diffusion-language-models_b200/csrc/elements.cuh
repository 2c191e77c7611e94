// Elements of bf16, fp16 and fp32 tensors, alone and in 16-byte vectors.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace mrsa {

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_float(float v) { return v; }

// V elements of T, read and written in one access.
template <typename T, int V> struct alignas(V * sizeof(T)) Elements { T e[V]; };

// Elements 2p and 2p + 1 as a pair of fp32 numbers (of a single element, it and 0).
template <typename T, int V> __device__ __forceinline__ float2 pair_of(const Elements<T, V>& x, int p) {
  if constexpr (V == 1) return make_float2(to_float(x.e[0]), 0.f);
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(x.e)[p]);
  else if constexpr (std::is_same_v<T, __half>) return __half22float2(reinterpret_cast<const __half2*>(x.e)[p]);
  else return make_float2(x.e[2 * p], x.e[2 * p + 1]);
}
template <typename T, int V> __device__ __forceinline__ void set_pair(Elements<T, V>& x, int p, float2 v) {
  if constexpr (V == 1) {
    x.e[0] = from_float<T>(v.x);
  } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    reinterpret_cast<__nv_bfloat162*>(x.e)[p] = __float22bfloat162_rn(v);
  } else if constexpr (std::is_same_v<T, __half>) {
    reinterpret_cast<__half2*>(x.e)[p] = __float22half2_rn(v);
  } else {
    x.e[2 * p] = v.x;
    x.e[2 * p + 1] = v.y;
  }
}

}  // namespace mrsa
