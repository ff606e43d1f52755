// Group normalisation of channels-last images, shared by the forward and the backward pass: how an
// image is cut up, and the arithmetic of one thread's vectors.
//
// Per view n and group g, over the group's D channels of all pixels (M values):
//   m = mean x,  r = 1 / sqrt(mean (x - m)^2 + eps),  h = (x - m) r,  z = h w_c + b_c
//   y = act(z), then dropout
// and with q = dy (dropout applied) act'(z):
//   grad b_c = sum q,  grad w_c = sum q h          (over pixels, and over views if shared)
//   A = sum q w / M,  B = sum q w h / M            (over the group)
//   grad x = r (q w - A - h B)
//
// A view is a matrix of pixels by channels whose rows are read in vectors of V values. Where the
// channels do not fill whole 16-byte vectors but the rows follow one another without gaps, `fold`
// pixels are taken as one row of fold * channels (7 channels of float32: 4 pixels are 7 vectors).
// A block's threads are R rows by the vectors of a tile of columns, so that a thread keeps its
// channels, and their constants in registers, for all its rows.
#pragma once

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "philox.cuh"
#include "vector.cuh"

namespace dr {

constexpr int kNormThreads = 256;

// How the views are cut up (made by plan_norm).
struct NormShape {
  long long batch;
  long long rows;       // rows of a view: pixels / fold
  long long pixels;
  int channels, groups, group_channels;
  int fold;
  int cols;             // vectors in a row
  int tile_cols;        // vectors in a tile of columns (the last tile may have fewer)
  int tiles;            // tiles in a row
  int group_tiles;      // tiles a group is cut into (1: tiles hold whole groups)
  int group_cols;       // vectors of a group that is cut into tiles
  long long chunk_rows; // rows of one block's work
  int chunks;           // of a view
  // Elements between the rows of x and of the output's gradient.
  long long x_row, grad_row;
};

struct NormParam {
  const void* data;  // NULL: ones (weight) or zeros (bias)
  int dtype;
  long long view;    // elements between the views' rows (0: one row for all)
};

struct NormTile {
  int col, cols;       // first vector and vectors
  int group, groups;   // first group and groups (partly covered when groups are cut)
};

__host__ __device__ inline NormTile norm_tile(const NormShape& s, int vec, int tile) {
  NormTile t;
  if (s.group_tiles > 1) {
    const int g = tile / s.group_tiles, part = tile - g * s.group_tiles;
    t.col = g * s.group_cols + part * s.tile_cols;
    t.cols = min(s.tile_cols, s.group_cols - part * s.tile_cols);
    t.group = g, t.groups = 1;
  } else {
    t.col = tile * s.tile_cols;
    t.cols = min(s.tile_cols, s.cols - t.col);
    if (s.fold > 1) {
      t.group = 0, t.groups = s.groups;
    } else {
      t.group = t.col * vec / s.group_channels;
      t.groups = t.cols * vec / s.group_channels;
    }
  }
  return t;
}

__device__ __forceinline__ float load_param(const void* data, int dtype, long long i) {
  if (dtype == DR_FLOAT32) return __ldg(static_cast<const float*>(data) + i);
  if (dtype == DR_FLOAT16) return __half2float(__ldg(static_cast<const __half*>(data) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(data) + i));
}

__device__ __forceinline__ void store_param(void* data, int dtype, long long i, float v) {
  if (dtype == DR_FLOAT32)
    static_cast<float*>(data)[i] = v;
  else if (dtype == DR_FLOAT16)
    static_cast<__half*>(data)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(data)[i] = __float2bfloat16_rn(v);
}

// 1 / (1 + exp(-z)), from the hardware's exponential and reciprocal (each within two units in the
// last place of float32). For z below -88 the exponential is infinite and the result 0.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// The activations: SiLU, or a clamp from below that is the identity with bound -infinity and ReLU
// with bound 0. The comparisons are written so that NaN passes, as it does through both.
template <bool Silu>
__device__ __forceinline__ float activate(float z, float bound) {
  if (Silu) return z * sigmoid(z);
  return z <= bound ? bound : z;
}

// The derivative at z: s (1 + z (1 - s)) for SiLU. ReLU's is 0 at 0.
template <bool Silu>
__device__ __forceinline__ float activate_grad(float z, float bound) {
  if (Silu) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  return z <= bound ? 0.0f : 1.0f;
}

// Running moments of V channels. Values are summed as differences from the thread's first value
// k: with n values, sum (x - k)^2 is at most n times their sum of squared deviations from their
// mean (k is one of them), so rounding grows by no more than n, whatever the offset of the data.
// Blocks give a thread at most kMomentRows rows.
constexpr int kMomentRows = 256;

template <int V>
struct Moments {
  float pivot[V], sum[V], square[V];
  int count = 0;

  __device__ __forceinline__ void add(const float (&v)[V]) {
    if (count == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) pivot[j] = v[j], sum[j] = 0.0f, square[j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = v[j] - pivot[j];
      sum[j] += d;
      square[j] = fmaf(d, d, square[j]);
    }
    ++count;
  }

  // (mean, sum of squared deviations) of channel j.
  __device__ __forceinline__ float2 get(int j) const {
    if (count == 0) return make_float2(0.0f, 0.0f);
    const float n = static_cast<float>(count);
    const float offset = sum[j] / n;
    // An overflown or NaN sum of squares stays what it is.
    const float squares = square[j] < __int_as_float(0x7f800000)
                              ? fmaxf(0.0f, fmaf(-sum[j], offset, square[j]))
                              : square[j];
    return make_float2(pivot[j] + offset, squares);
  }
};

// NaN or infinite data give NaN statistics (their mean is NaN or infinite).
__device__ __forceinline__ float variance_of(float mean, float squares, float count) {
  return isfinite(mean) ? squares / count : __int_as_float(0x7fc00000);
}

// Lanes (a power of two, at most 32) that share one of `items` reductions of a block.
__device__ __forceinline__ int lanes_per(int items, int threads) {
  int lanes = 1;
  while (lanes < 32 && items * lanes * 2 <= threads) lanes *= 2;
  return lanes;
}

__device__ __forceinline__ float lane_sum(float v, int lanes) {
  for (int d = lanes / 2; d > 0; d /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

// Joins (mean, squared deviations) of parts with the given counts into those of their union:
//   mean = m_0 + sum n_i (m_i - m_0) / N,  squares = sum (s_i + n_i (m_i - mean)^2).
// `part(item, i, value)` returns the count of part i and its value; a part of count 0 has a finite
// one, and part 0 is never empty. All threads of the block call this with the same `items` of
// `parts` entries each; `done(item, mean, squares)` runs on one lane per item.
template <typename Part, typename Done>
__device__ __forceinline__ void join_moments(int items, int parts, int threads, Part part,
                                             Done done) {
  const int lanes = lanes_per(items, threads);
  const int lane = threadIdx.x % lanes;
  const int step = threads / lanes;
  for (int base = 0; base < items; base += step) {
    const int item = base + threadIdx.x / lanes;
    const bool live = item < items;
    float n = 0.0f, total = 0.0f;
    float2 first = make_float2(0.0f, 0.0f);
    if (live) {
      part(item, 0, first);
      for (int i = lane; i < parts; i += lanes) {
        float2 v;
        const float c = part(item, i, v);
        n += c;
        total = fmaf(c, v.x - first.x, total);
      }
    }
    n = lane_sum(n, lanes);
    total = lane_sum(total, lanes);
    const float mean = first.x + total / n;
    float squares = 0.0f;
    if (live) {
      for (int i = lane; i < parts; i += lanes) {
        float2 v;
        const float c = part(item, i, v);
        const float d = v.x - mean;
        squares += c > 0.0f ? fmaf(c * d, d, v.y) : 0.0f;
      }
    }
    squares = lane_sum(squares, lanes);
    if (live && lane == 0) done(item, mean, squares);
  }
}

// Sums pairs: `part(item, i)` is entry i of the item's `parts`.
template <typename Part, typename Done>
__device__ __forceinline__ void join_sums(int items, int parts, int threads, Part part,
                                          Done done) {
  const int lanes = lanes_per(items, threads);
  const int lane = threadIdx.x % lanes;
  const int step = threads / lanes;
  for (int base = 0; base < items; base += step) {
    const int item = base + threadIdx.x / lanes;
    const bool live = item < items;
    float2 total = make_float2(0.0f, 0.0f);
    if (live) {
      for (int i = lane; i < parts; i += lanes) {
        const float2 v = part(item, i);
        total.x += v.x;
        total.y += v.y;
      }
    }
    total.x = lane_sum(total.x, lanes);
    total.y = lane_sum(total.y, lanes);
    if (live && lane == 0) done(item, total);
  }
}

// ---- host --------------------------------------------------------------------------------------

constexpr int kNoPlan = 0;
constexpr int kMaxNormChannels = 1 << 16;

inline int greatest_divisor(long long a, long long b) {
  while (b != 0) {
    const long long t = a % b;
    a = b;
    b = t;
  }
  return static_cast<int>(a);
}

inline bool bad_norm_sizes(int64_t batch, int64_t pixels, int32_t channels, int32_t groups,
                           int32_t dtype) {
  return batch < 0 || pixels < 0 || channels < 1 || channels > kMaxNormChannels || groups < 1 ||
         channels % groups != 0 || !known_dtype(dtype);
}

inline bool bad_norm_param(const void* data, int32_t dtype, int64_t rows, int64_t batch) {
  return data != nullptr && (!known_dtype(dtype) || (rows != 1 && rows != batch));
}

inline float norm_bound(int activation) {
  return activation == DR_ACTIVATION_RELU ? 0.0f : -__builtin_huge_valf();
}

// A vector width and a number of folded pixels.
struct NormVector {
  int vec, fold;
};

// The widest vectors that the addresses, the strides and the channels allow. Strides are elements
// between the pixels of x and of the output's gradient (`channels` where there is none).
inline NormVector choose_vector(long long pixels, int channels, int dtype, long long x_stride,
                                long long grad_stride,
                                std::initializer_list<const void*> pointers) {
  const int size = dtype_bytes(dtype), widest = 16 / size;
  auto fits = [&](int v) {
    for (const void* p : pointers)
      if (!aligned_to(p, static_cast<size_t>(v) * size)) return false;
    return true;
  };
  auto divides = [&](int v) {
    return channels % v == 0 && x_stride % v == 0 && grad_stride % v == 0;
  };
  if (fits(widest)) {
    if (divides(widest)) return {widest, 1};
    const int fold = widest / greatest_divisor(channels, widest);
    if (x_stride == channels && grad_stride == channels && pixels % fold == 0 &&
        static_cast<long long>(channels) * fold / widest <= kNormThreads)
      return {widest, fold};
  }
  if (widest == 8 && fits(2) && divides(2)) return {2, 1};
  return {1, 1};
}

// Cuts views into tiles of columns and chunks of rows of about `chunk_bytes`. Lowers v.vec where a
// group is wider than a block's threads and not whole vectors (its tiles must not reach into the
// next group). False when there would be too many blocks.
inline bool cut_norm(NormShape& s, NormVector& v, long long batch, long long pixels, int channels,
                     int groups, int dtype, long long x_stride, long long grad_stride,
                     long long chunk_bytes) {
  s.batch = batch;
  s.pixels = pixels;
  s.channels = channels;
  s.groups = groups;
  s.group_channels = channels / groups;
  // Columns of the fewest whole groups that are whole vectors.
  const int d = s.group_channels;
  long long unit = d / greatest_divisor(d, v.vec);
  if (v.fold == 1 && unit > kNormThreads && d % v.vec != 0) {
    v.vec = 1;
    unit = d;
  }
  s.fold = v.fold;
  s.rows = pixels / s.fold;
  s.cols = static_cast<int>(static_cast<long long>(channels) * s.fold / v.vec);
  s.x_row = x_stride * s.fold;
  s.grad_row = grad_stride * s.fold;
  s.group_tiles = 1;
  s.group_cols = 0;
  if (s.cols <= kNormThreads) {
    s.tile_cols = s.cols;
    s.tiles = 1;
  } else if (unit <= kNormThreads) {
    s.tile_cols = static_cast<int>(kNormThreads / unit * unit);
    s.tiles = (s.cols + s.tile_cols - 1) / s.tile_cols;
  } else {
    s.group_cols = static_cast<int>(unit);
    s.group_tiles = static_cast<int>((unit + kNormThreads - 1) / kNormThreads);
    s.tile_cols = kNormThreads;
    s.tiles = groups * s.group_tiles;
  }
  const long long lanes = kNormThreads / s.tile_cols;  // rows that a block reads at once
  const long long tile_bytes = static_cast<long long>(s.tile_cols) * v.vec * dtype_bytes(dtype);
  const long long deep = chunk_bytes / tile_bytes / lanes;
  s.chunk_rows = std::max(1LL, std::min<long long>(deep, kMomentRows)) * lanes;
  const long long chunks = (s.rows + s.chunk_rows - 1) / s.chunk_rows;
  if (chunks > 0x7FFFFFFF || batch * s.tiles > 0x7FFFFFFF / std::max(1LL, chunks)) return false;
  s.chunks = static_cast<int>(chunks);
  return true;
}

// Bytes of a chunk: 64 KB, less where that would leave processors idle.
inline long long norm_chunk_bytes(long long batch, long long pixels, int channels, int dtype) {
  const long long total = batch * pixels * channels * dtype_bytes(dtype);
  return std::max(4096LL, std::min(65536LL, total / 592));
}

// Workspace of the forward pass: (mean, squares) of each group, chunk and tile.
inline size_t norm_forward_bytes(const NormShape& s) {
  return static_cast<size_t>(s.batch) * s.groups * s.chunks * s.group_tiles * sizeof(float2);
}

// Workspace of the backward pass: sums of each channel and chunk, of each view and channel, and
// the two means of each view and group.
inline size_t norm_backward_bytes(const NormShape& s) {
  const size_t views = static_cast<size_t>(s.batch) * s.channels * sizeof(float2);
  return align256(views * s.chunks) + align256(views) +
         static_cast<size_t>(s.batch) * s.groups * sizeof(float2);
}

// The larger workspace of all the vector widths that a call may turn out to take.
inline size_t norm_workspace_bytes(long long batch, long long pixels, int channels, int groups,
                                   int dtype, bool backward) {
  const int widest = 16 / dtype_bytes(dtype);
  const int fold = widest / greatest_divisor(channels, widest);
  size_t most = 0;
  for (NormVector v : {NormVector{widest, fold}, NormVector{2, 1}, NormVector{1, 1}}) {
    if (v.fold > 1 && (pixels % v.fold != 0 ||
                       static_cast<long long>(channels) * v.fold / widest > kNormThreads))
      continue;
    if (v.fold == 1 && channels % v.vec != 0) continue;
    NormShape s;
    if (cut_norm(s, v, batch, pixels, channels, groups, dtype, channels, channels,
                 norm_chunk_bytes(batch, pixels, channels, dtype)))
      most = std::max(most, backward ? norm_backward_bytes(s) : norm_forward_bytes(s));
  }
  return most;
}

template <typename T>
struct TypeTag {
  using type = T;
};

// Calls fn(TypeTag<T>, integral_constant<int, V>) for a type and one of its vector widths.
template <typename Fn>
int with_vector(int dtype, int vec, Fn fn) {
  auto half = [&](auto tag) {
    if (vec == 8) return fn(tag, std::integral_constant<int, 8>());
    if (vec == 2) return fn(tag, std::integral_constant<int, 2>());
    return fn(tag, std::integral_constant<int, 1>());
  };
  if (dtype == DR_FLOAT16) return half(TypeTag<__half>());
  if (dtype == DR_BFLOAT16) return half(TypeTag<__nv_bfloat16>());
  if (vec == 4) return fn(TypeTag<float>(), std::integral_constant<int, 4>());
  return fn(TypeTag<float>(), std::integral_constant<int, 1>());
}

}  // namespace dr
