// Vectors of float32, float16 and bfloat16 values: one load or store of up to 16 bytes, arithmetic
// in float32, one rounding (to nearest even) on the way out.
#pragma once

#include <cstdint>
#include <cstring>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

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
  Packed<T, V> p;
  if constexpr (V > 1 && sizeof(T) == 2) {
    unsigned int words[V / 2];
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(v[j], v[j + 1]);
        memcpy(&words[j / 2], &h, sizeof(h));
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[j], v[j + 1]);
        memcpy(&words[j / 2], &h, sizeof(h));
      }
    }
    memcpy(&p, words, sizeof(p));
  } else {
    T t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = from_float<T>(v[j]);
    memcpy(&p, t, sizeof(p));
  }
  return p;
}

// Two float32 lanes of one instruction: sums, products and fused multiply-adds of pairs, each lane
// rounded to nearest as the scalar instruction rounds it.
__device__ __forceinline__ unsigned long long pair_bits(float2 v) {
  unsigned long long b;
  asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(v.x), "f"(v.y));
  return b;
}
__device__ __forceinline__ float2 bits_pair(unsigned long long b) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(b));
  return v;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return bits_pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return bits_pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
  return bits_pair(r);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// V values as pairs; a single value has a zero beside it.
template <int V>
struct Pairs {
  static constexpr int kCount = (V + 1) / 2;
  float2 p[kCount];

  __device__ __forceinline__ float get(int j) const { return j & 1 ? p[j / 2].y : p[j / 2].x; }
  __device__ __forceinline__ void set(int j, float v) { (j & 1 ? p[j / 2].y : p[j / 2].x) = v; }
};

// Two neighbouring 16-bit values as float32. A bfloat16 is the upper half of its float32.
template <typename T>
__device__ __forceinline__ float2 widen(unsigned int bits) {
  if constexpr (std::is_same_v<T, __half>) {
    __half2 h;
    memcpy(&h, &bits, sizeof(h));
    return __half22float2(h);
  } else {
    return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xFFFF0000u));
  }
}

template <typename T, int V>
__device__ __forceinline__ Pairs<V> load_pairs(const Packed<T, V>& bits) {
  Pairs<V> r;
  if constexpr (V > 1 && sizeof(T) == 2) {
    unsigned int words[V / 2];
    memcpy(words, &bits, sizeof(bits));
#pragma unroll
    for (int j = 0; j < V / 2; ++j) r.p[j] = widen<T>(words[j]);
  } else {
    float v[V];
    unpack<T, V>(bits, v);
    if (V == 1) r.p[0].y = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) r.set(j, v[j]);
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ Packed<T, V> pack_pairs(const Pairs<V>& r) {
  float v[V];
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = r.get(j);
  return pack<T, V>(v);
}

// Element types of the C ABI (DR_FLOAT32, DR_FLOAT16, DR_BFLOAT16).
inline bool known_dtype(int dtype) { return dtype >= DR_FLOAT32 && dtype <= DR_BFLOAT16; }
inline int dtype_bytes(int dtype) { return dtype == DR_FLOAT32 ? 4 : 2; }

inline bool aligned_to(const void* p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace dr
