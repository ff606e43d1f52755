// Dropout of a contiguous tensor, with an optional residual:
//
//   y = residual + (kept ? x * 65536 / (65536 - threshold) : 0)
//
// and its gradient, which is the same pass over the output's gradient without the residual: the
// mask comes from philox.cuh again and is never stored.
#include <cstdint>

#include "philox.cuh"
#include "vector.cuh"

namespace dr {
namespace {

constexpr int kThreads = 256;

// A thread has Counters counters of eight elements each: all their loads are issued first, and the
// rounds of the generator run while they are under way. Bound by memory: with a residual eight 512 x
// 512 x 64 bfloat16 images take 122 us, 6.6 TB/s. `Wide` tensors are read and written in 16-byte
// words; the others, whose address is not a multiple of 16, and the last elements one by one.
//
// With two counters bytes enough are under way but for large tensors of 2 bytes an element and no
// residual, which take four: the images' gradient takes 111, 98 and 93 us with one, two and four.
// At 32 MB two and four are even (14.6 us), at 8 MB four are slower (6.4 us instead of 5.6), and
// float32 is slower with four at every size (48 MB: 20.2 us instead of 17.9).
constexpr long long kManyBytes = 64LL << 20;

template <typename T, bool Wide, bool Residual, int Counters>
__global__ void __launch_bounds__(kThreads) dropout_kernel(
    const T* __restrict__ x, const T* __restrict__ residual, long long count, DropKey key,
    T* __restrict__ y) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte word
  constexpr int kWords = 8 / kPer;
  const long long base =
      (blockIdx.x * static_cast<long long>(kThreads * Counters) + threadIdx.x) * 8;
  const unsigned long long seed = load_seed(key);
  uint4 a[Counters][kWords], b[Counters][kWords];
#pragma unroll
  for (int n = 0; n < Counters; ++n) {
    const long long first = base + n * kThreads * 8;
    if constexpr (Wide) {
      if (first + 8 <= count) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          a[n][k] = __ldcs(reinterpret_cast<const uint4*>(x + first) + k);
          if (Residual) b[n][k] = __ldcs(reinterpret_cast<const uint4*>(residual + first) + k);
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < Counters; ++n) {
    const long long first = base + n * kThreads * 8;
    if (first >= count) return;
    const bool whole = Wide && first + 8 <= count;
    Pairs<8> v, r;
    if (whole) {
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
        const Pairs<kPer> part = load_pairs<T, kPer>(a[n][k]);
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) v.p[k * (kPer / 2) + j] = part.p[j];
        if (Residual) {
          const Pairs<kPer> skip = load_pairs<T, kPer>(b[n][k]);
#pragma unroll
          for (int j = 0; j < kPer / 2; ++j) r.p[k * (kPer / 2) + j] = skip.p[j];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v.set(j, first + j < count ? to_float(x[first + j]) : 0.0f);
        if (Residual) r.set(j, first + j < count ? to_float(residual[first + j]) : 0.0f);
      }
    }
    apply_dropout<8>(v, first, key, seed);
    if (Residual) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v.p[j] = add2(v.p[j], r.p[j]);
    }
    if (whole) {
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
        Pairs<kPer> part;
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) part.p[j] = v.p[k * (kPer / 2) + j];
        __stcs(reinterpret_cast<uint4*>(y + first) + k, pack_pairs<T, kPer>(part));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (first + j < count) y[first + j] = from_float<T>(v.get(j));
    }
  }
}

template <typename T>
int run(const void* x, const void* residual, long long count, const DropKey& key, void* y,
        cudaStream_t stream) {
  const bool wide = aligned_to(x, 16) && aligned_to(y, 16) &&
                    (residual == nullptr || aligned_to(residual, 16));
  auto launch = [&](auto kernel, int counters) {
    kernel<<<blocks_for((count + 7) / 8, kThreads * counters), kThreads, 0, stream>>>(
        static_cast<const T*>(x), static_cast<const T*>(residual), count, key, static_cast<T*>(y));
  };
  if (residual != nullptr) {
    wide ? launch(dropout_kernel<T, true, true, 2>, 2) : launch(dropout_kernel<T, false, true, 2>, 2);
    return launch_status();
  }
  if constexpr (sizeof(T) == 2) {
    if (wide && count * 2 >= kManyBytes) {
      launch(dropout_kernel<T, true, false, 4>, 4);
      return launch_status();
    }
  }
  wide ? launch(dropout_kernel<T, true, false, 2>, 2) : launch(dropout_kernel<T, false, false, 2>, 2);
  return launch_status();
}

}  // namespace
}  // namespace dr

using namespace dr;

extern "C" int dr_dropout(const void* x, const void* residual, int64_t count, int32_t dtype,
                          int32_t threshold, const int64_t* seed, int64_t seed_value,
                          int64_t layer, void* y, void* stream) {
  if (count < 0 || !known_dtype(dtype) || bad_drop(threshold, layer))
    return DR_ERR_INVALID_ARGUMENT;
  if (count == 0) return DR_OK;
  const size_t size = dtype_bytes(dtype);
  if (x == nullptr || y == nullptr || !aligned_to(x, size) || !aligned_to(y, size) ||
      !aligned_to(residual, size) || !aligned_to(seed, sizeof(int64_t)))
    return DR_ERR_INVALID_ARGUMENT;
  // At most 2^31 - 1 blocks.
  if (count > 8LL * kThreads * 2 * 0x7FFFFFFF) return DR_ERR_TOO_LARGE;
  const DropKey key = drop_key(seed, seed_value, layer, threshold);
  switch (dtype) {
    case DR_FLOAT32:
      return run<float>(x, residual, count, key, y, as_stream(stream));
    case DR_FLOAT16:
      return run<__half>(x, residual, count, key, y, as_stream(stream));
    default:
      return run<__nv_bfloat16>(x, residual, count, key, y, as_stream(stream));
  }
}
