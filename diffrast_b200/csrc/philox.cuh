// Random bits of the dropout masks: Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011), a function of a counter and a key, so
// that a mask is drawn again wherever it is needed and never stored.
//
//   key      the 64-bit seed
//   counter  (element / 8, low and high word; the layer; 0)
//   element  takes 16 of the 128 bits: bits 16 (e % 2) .. of word (e % 8) / 2
//
// An element is dropped when its 16 bits, as a number, are below the threshold, and a kept one is
// scaled by 65536 / (65536 - threshold), the reciprocal of the exact probability to be kept. Eight
// elements share one counter because the ten rounds cost about 50 instructions: at 32 bits an
// element they would cost more than the memory traffic of a 16-bit image; 16 bits leave the
// probability on a grid of 2^-16.
#pragma once

#include <cstdint>

#include "vector.cuh"

namespace dr {

struct DropKey {
  const long long* seed;     // one device word, or NULL
  unsigned long long value;  // the seed when `seed` is NULL
  unsigned int layer;
  unsigned int threshold;    // 0: nothing is dropped
  float scale;
};

inline bool bad_drop(int32_t threshold, int64_t layer) {
  return threshold < 0 || threshold > 65535 || layer < 0 || layer > 0xFFFFFFFFLL;
}

inline DropKey drop_key(const int64_t* seed, int64_t seed_value, int64_t layer,
                        int32_t threshold) {
  return {reinterpret_cast<const long long*>(seed), static_cast<unsigned long long>(seed_value),
          static_cast<unsigned int>(layer), static_cast<unsigned int>(threshold),
          static_cast<float>(65536.0 / (65536 - threshold))};
}

// The load carries its test with it as one instruction's predicate: written as a load under an if,
// it could be moved before the test, and `seed` is NULL with every seed that is a number.
__device__ __forceinline__ unsigned long long load_seed(const DropKey& key) {
  unsigned long long seed = key.value;
  asm volatile(
      "{\n\t"
      ".reg .pred given;\n\t"
      "setp.ne.u64 given, %1, 0;\n\t"
      "@given ld.global.u64 %0, [%1];\n\t"
      "}"
      : "+l"(seed)
      : "l"(key.seed)
      : "memory");
  return seed;
}

__device__ __forceinline__ uint4 philox(unsigned long long block, unsigned int layer,
                                        unsigned long long seed) {
  uint4 c = make_uint4(static_cast<unsigned int>(block), static_cast<unsigned int>(block >> 32),
                       layer, 0u);
  unsigned int k0 = static_cast<unsigned int>(seed), k1 = static_cast<unsigned int>(seed >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const unsigned long long p0 = static_cast<unsigned long long>(0xD2511F53u) * c.x;
    const unsigned long long p1 = static_cast<unsigned long long>(0xCD9E8D57u) * c.z;
    c = make_uint4(static_cast<unsigned int>(p1 >> 32) ^ c.y ^ k0, static_cast<unsigned int>(p1),
                   static_cast<unsigned int>(p0 >> 32) ^ c.w ^ k1, static_cast<unsigned int>(p0));
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

// v = kept ? v * scale : 0 for the V elements from `element` on (a multiple of V; V is 1, 2,
// 4 or 8, so they share a counter). A dropped NaN or infinity gives 0 too.
template <int V>
__device__ __forceinline__ void apply_dropout(Pairs<V>& v, long long element, const DropKey& key,
                                              unsigned long long seed) {
  const uint4 r = philox(static_cast<unsigned long long>(element) >> 3, key.layer, seed);
  unsigned int w[(V + 1) / 2];
  if constexpr (V == 8) {
    w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
  } else if constexpr (V == 4) {
    const bool high = element & 4;
    w[0] = high ? r.z : r.x;
    w[1] = high ? r.w : r.y;
  } else {
    const unsigned int low = element & 2 ? r.y : r.x, high = element & 2 ? r.w : r.z;
    w[0] = element & 4 ? high : low;
    if constexpr (V == 1) w[0] >>= (element & 1) * 16;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const unsigned int bits = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
    v.set(j, bits >= key.threshold ? v.get(j) * key.scale : 0.0f);
  }
}

}  // namespace dr
