// Vectors of float32, float16 and bfloat16 values: one load or store of up to 32 bytes, arithmetic
// in float32, one rounding (to nearest even) on the way out.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace dr {

template <int Bytes>
struct Bits;
template <>
struct Bits<2> {
  using type = unsigned short;
};
template <>
struct Bits<4> {
  using type = unsigned int;
};
template <>
struct Bits<8> {
  using type = uint2;
};
template <>
struct Bits<16> {
  using type = uint4;
};

// V values of type T as they lie in memory (V * sizeof(T) is 2, 4, 8 or 16 bytes).
template <typename T, int V>
using Packed = typename Bits<V * static_cast<int>(sizeof(T))>::type;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Packed<T, V>& p, float (&v)[V]) {
  T t[V];
  memcpy(t, &p, sizeof(p));
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = to_float(t[j]);
}

template <typename T, int V>
__device__ __forceinline__ Packed<T, V> pack(const float (&v)[V]) {
  T t[V];
  if constexpr (V % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(v[j], v[j + 1]);
        t[j] = h.x, t[j + 1] = h.y;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[j], v[j + 1]);
        t[j] = h.x, t[j + 1] = h.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = from_float<T>(v[j]);
  }
  Packed<T, V> p;
  memcpy(&p, t, sizeof(p));
  return p;
}

// Element types of the C ABI (DR_FLOAT32, DR_FLOAT16, DR_BFLOAT16).
inline bool known_dtype(int dtype) { return dtype >= DR_FLOAT32 && dtype <= DR_BFLOAT16; }
inline int dtype_bytes(int dtype) { return dtype == DR_FLOAT32 ? 4 : 2; }

inline bool aligned_to(const void* p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace dr
