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

// How the views are cut up (made by cut_norm).
struct NormShape {
  long long batch;
  long long rows;       // rows of a view: pixels / fold
  long long pixels;
  int channels, groups, group_channels;
  int fold;
  int cols;             // vectors in a row
  int tile_cols;        // vectors in a tile of columns (the last tile may have fewer)
  int tiles;            // of a row; whole groups each, unless groups are cut
  int pieces;           // tiles that a group is cut into, or 1
  int group_cols;       // vectors of a group that is cut
  int chunk_rows;       // rows of one block's work
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
  int col, cols;      // first vector and vectors
  int group, groups;  // first group and groups (the one group when it is cut)
};

// Work of one block: a chunk of rows in a tile of columns.
struct NormBlock {
  int view, chunk, piece;
  NormTile tile;
  int rows;
  long long first;  // first row, counted over the views
};

__device__ __forceinline__ NormBlock norm_block(const NormShape& s, int vec, int view0,
                                                unsigned int index) {
  NormBlock b;
  const unsigned int rest = index / s.chunks;
  b.chunk = static_cast<int>(index - rest * s.chunks);
  const unsigned int view = rest / s.tiles;
  const int tile = static_cast<int>(rest - view * s.tiles);
  b.view = view0 + static_cast<int>(view);
  b.piece = 0;
  if (s.pieces > 1) {
    b.tile.group = tile / s.pieces;
    b.piece = tile - b.tile.group * s.pieces;
    b.tile.col = b.tile.group * s.group_cols + b.piece * s.tile_cols;
    b.tile.cols = min(s.tile_cols, s.group_cols - b.piece * s.tile_cols);
    b.tile.groups = 1;
  } else {
    b.tile.col = tile * s.tile_cols;
    b.tile.cols = min(s.tile_cols, s.cols - b.tile.col);
    b.tile.group = s.fold > 1 ? 0 : b.tile.col * vec / s.group_channels;
    b.tile.groups = s.fold > 1 ? s.groups : b.tile.cols * vec / s.group_channels;
  }
  const long long row0 = static_cast<long long>(b.chunk) * s.chunk_rows;
  b.rows = static_cast<int>(min(static_cast<long long>(s.chunk_rows), s.rows - row0));
  b.first = b.view * s.rows + row0;
  return b;
}

// The channels of a thread's vector one after the other, with their groups: one division for all.
struct ChannelWalk {
  int channel, group, rest, channels, size;

  __device__ __forceinline__ ChannelWalk(const NormShape& s, int first)
      : channels(s.channels), size(s.group_channels) {
    channel = s.fold > 1 ? first % channels : first;
    group = channel / size;
    rest = channel - group * size;
  }
  __device__ __forceinline__ void next() {
    ++channel;
    if (++rest == size) rest = 0, ++group;
    if (channel == channels) channel = 0, group = 0;
  }
};

__device__ __forceinline__ float load_param(const void* data, int dtype, long long i) {
  if (dtype == DR_FLOAT32) return __ldg(static_cast<const float*>(data) + i);
  if (dtype == DR_FLOAT16) return __half2float(__ldg(static_cast<const __half*>(data) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(data) + i));
}

__device__ __forceinline__ float load_scale(const NormParam& w, long long view, int channel) {
  return w.data ? load_param(w.data, w.dtype, view * w.view + channel) : 1.0f;
}
__device__ __forceinline__ float load_shift(const NormParam& b, long long view, int channel) {
  return b.data ? load_param(b.data, b.dtype, view * b.view + channel) : 0.0f;
}

__device__ __forceinline__ void store_param(void* data, int dtype, long long i, float v) {
  if (dtype == DR_FLOAT32)
    static_cast<float*>(data)[i] = v;
  else if (dtype == DR_FLOAT16)
    static_cast<__half*>(data)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(data)[i] = __float2bfloat16_rn(v);
}

// 1 / (1 + exp(-z)), from the hardware's exponential (of 2) and reciprocal, each within two units
// in the last place of float32. For z below -88 the exponential is infinite and the result 0.
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  const float2 t = mul2(z, both(-1.4426950408889634f));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  e = add2(e, both(1.0f));
  float2 s;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(e.y));
  return s;
}

// The activations: SiLU, or a clamp from below that is the identity with bound -infinity and ReLU
// with bound 0. The comparisons are written so that NaN passes, as it does through both.
template <bool Silu>
__device__ __forceinline__ float2 activate(float2 z, float bound) {
  if (Silu) return mul2(z, sigmoid2(z));
  return make_float2(z.x <= bound ? bound : z.x, z.y <= bound ? bound : z.y);
}

// q times the derivative at z: s (1 + z (1 - s)) for SiLU. ReLU's is 0 at 0.
template <bool Silu>
__device__ __forceinline__ float2 activate_grad(float2 q, float2 z, float bound) {
  if (Silu) {
    const float2 s = sigmoid2(z);
    const float2 t = fma2(make_float2(-s.x, -s.y), z, z);
    return mul2(q, fma2(s, t, s));
  }
  return make_float2(z.x <= bound ? 0.0f : q.x, z.y <= bound ? 0.0f : q.y);
}

// Running moments of V channels. Values are summed as differences from the thread's first value
// k: with n values, sum (x - k)^2 is at most n times their sum of squared deviations from their
// mean (k is one of them), so rounding grows by no more than n, whatever the offset of the data.
// Blocks give a thread at most kMomentRows rows; a warp's threads that share a column are joined
// about the first one's pivot, which multiplies that number by the rows that a warp holds.
constexpr int kMomentRows = 64;

template <int V>
struct Moments {
  Pairs<V> pivot, sum, square;  // the pivot is kept negated

  __device__ __forceinline__ void start(const Pairs<V>& v) {
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j) {
      pivot.p[j] = make_float2(-v.p[j].x, -v.p[j].y);
      sum.p[j] = square.p[j] = both(0.0f);
    }
  }

  __device__ __forceinline__ void add(const Pairs<V>& v) {
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j) {
      const float2 d = add2(v.p[j], pivot.p[j]);
      sum.p[j] = add2(sum.p[j], d);
      square.p[j] = fma2(d, d, square.p[j]);
    }
  }

  // Moves to the pivots of a lane of the warp: sum (x - l) = sum (x - k) + n (k - l) and
  // sum (x - l)^2 = sum (x - k)^2 + (k - l) (2 sum (x - k) + n (k - l)). Without values (n = 0)
  // the sums stay zero.
  __device__ __forceinline__ void move_pivot(int from_lane, float n) {
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j) {
      float2 l;
      l.x = __shfl_sync(0xFFFFFFFFu, pivot.p[j].x, from_lane);
      l.y = V > 1 ? __shfl_sync(0xFFFFFFFFu, pivot.p[j].y, from_lane) : 0.0f;
      const float2 d = n > 0.0f ? make_float2(l.x - pivot.p[j].x, l.y - pivot.p[j].y) : both(0.0f);
      const float2 nd = mul2(both(n), d);
      square.p[j] = fma2(d, fma2(both(2.0f), sum.p[j], nd), square.p[j]);
      sum.p[j] = add2(sum.p[j], nd);
      pivot.p[j] = l;
    }
  }

  // Adds the sums of the lane at this distance, about the same pivots.
  __device__ __forceinline__ void add_lane(int distance) {
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j) {
      float2 a, b = both(0.0f);
      a.x = __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].x, distance);
      b.x = __shfl_xor_sync(0xFFFFFFFFu, square.p[j].x, distance);
      a.y = V > 1 ? __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].y, distance) : 0.0f;
      b.y = V > 1 ? __shfl_xor_sync(0xFFFFFFFFu, square.p[j].y, distance) : 0.0f;
      sum.p[j] = add2(sum.p[j], a);
      square.p[j] = add2(square.p[j], b);
    }
  }

  // (mean, sum of squared deviations) of channel j over n values.
  __device__ __forceinline__ float2 get(int j, float n, float inverse) const {
    const float offset = sum.get(j) * inverse;
    // An overflown or NaN sum of squares stays what it is.
    const float total = square.get(j);
    const float squares = total < __int_as_float(0x7f800000)
                              ? fmaxf(0.0f, fmaf(-n * offset, offset, total))
                              : total;
    return make_float2(offset - pivot.get(j), squares);
  }
};

// Moments of Q neighbouring channels of a thread, n values each, as one part of n Q values.
template <int Q, int V>
__device__ __forceinline__ float2 fold_channels(const Moments<V>& m, int first, float n,
                                                float inverse) {
  float2 part[Q];
  float mean = 0.0f;
#pragma unroll
  for (int j = 0; j < Q; ++j) part[j] = m.get(first + j, n, inverse);
#pragma unroll
  for (int j = 0; j < Q; ++j) mean += part[j].x - part[0].x;
  mean = fmaf(mean, 1.0f / Q, part[0].x);
  float squares = 0.0f;
#pragma unroll
  for (int j = 0; j < Q; ++j) {
    const float d = part[j].x - mean;
    squares += fmaf(n * d, d, part[j].y);
  }
  return make_float2(mean, squares);
}

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
__device__ __forceinline__ void join_moments(int items, int parts, Part part, Done done) {
  const int lanes = lanes_per(items, kNormThreads);
  const int lane = threadIdx.x & (lanes - 1);
  const int step = kNormThreads / lanes;
  for (int base = 0; base < items; base += step) {
    const int item = base + threadIdx.x / lanes;
    const bool live = item < items;
    float n = 0.0f, total = 0.0f;
    float2 first = make_float2(0.0f, 0.0f);
    if (live) {
      part(item, 0, first);
#pragma unroll 4
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
#pragma unroll 4
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
__device__ __forceinline__ void join_sums(int items, int parts, Part part, Done done) {
  const int lanes = lanes_per(items, kNormThreads);
  const int lane = threadIdx.x & (lanes - 1);
  const int step = kNormThreads / lanes;
  for (int base = 0; base < items; base += step) {
    const int item = base + threadIdx.x / lanes;
    const bool live = item < items;
    float2 total = make_float2(0.0f, 0.0f);
    if (live) {
#pragma unroll 8
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

// A thread's place in a tile of columns: `lanes` rows of the tile's vectors at a time.
struct TileThread {
  int lanes, lane, col;
  bool active;

  __device__ __forceinline__ explicit TileThread(int cols) {
    lanes = kNormThreads / cols;
    lane = threadIdx.x / cols;
    col = threadIdx.x - lane * cols;
    active = lane < lanes;
  }
};

// Copies to shared memory (a 32-bit address) that run beside the thread. A copy of 2 bytes, which
// the hardware does not have, is a load and a store.
template <int Bytes>
__device__ __forceinline__ void copy_async(unsigned int to, const void* from) {
  if constexpr (Bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else if constexpr (Bytes >= 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(Bytes)
                 : "memory");
  else
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(to),
                 "h"(*static_cast<const unsigned short*>(from))
                 : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int Pending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(Pending) : "memory");
}

template <typename P>
__device__ __forceinline__ P load_slot(unsigned int at) {
  P p;
  if constexpr (sizeof(P) == 16)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(p.x), "=r"(p.y), "=r"(p.z), "=r"(p.w)
                 : "r"(at)
                 : "memory");
  else if constexpr (sizeof(P) == 4)
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(p) : "r"(at) : "memory");
  else
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(p) : "r"(at) : "memory");
  return p;
}

// A thread's rows on their way to it: it copies its own vectors (of Images images) into its own
// slots of shared memory, Stages rows ahead of the one it works on. No slot is shared, so the
// copies need no barriers, and they hold no registers: with batches of loads in registers instead,
// the sums of the backward pass read memory at 1.9 TB/s, for want of bytes under way.
template <typename T, int V, int Images, int Stages>
struct RowRing {
  using P = Packed<T, V>;
  static constexpr unsigned int kSlot = sizeof(P) * kNormThreads;
  static constexpr size_t kBytes = static_cast<size_t>(kSlot) * Images * Stages;

  const T* at[Images];
  long long stride[Images];
  unsigned int slots;
  int count;

  // Rows lane, lane + lanes, ... below `rows` of columns that start at at[].
  __device__ __forceinline__ void start(void* shared, const TileThread& t, int rows) {
    slots = static_cast<unsigned int>(__cvta_generic_to_shared(shared)) +
            threadIdx.x * static_cast<unsigned int>(sizeof(P));
    count = t.active && t.lane < rows ? (rows - t.lane + t.lanes - 1) / t.lanes : 0;
#pragma unroll
    for (int k = 0; k < Images; ++k) {
      at[k] += t.lane * stride[k];
      stride[k] *= t.lanes;
    }
#pragma unroll
    for (int u = 0; u < Stages; ++u) {
      if (u < count) fetch(u);
      copy_commit();
    }
  }

  __device__ __forceinline__ void fetch(int u) {
#pragma unroll
    for (int k = 0; k < Images; ++k) {
      copy_async<sizeof(P)>(slots + (u * Images + k) * kSlot, at[k]);
      at[k] += stride[k];
    }
  }

  // Calls use(vectors) for the rows in order.
  template <typename Use>
  __device__ __forceinline__ void for_rows(Use use) {
    for (int left = count; left > 0; left -= Stages) {
#pragma unroll
      for (int u = 0; u < Stages; ++u) {
        if (u > 0 && u >= left) break;
        copy_wait<Stages - 1>();
        Pairs<V> v[Images];
#pragma unroll
        for (int k = 0; k < Images; ++k)
          v[k] = load_pairs<T, V>(load_slot<P>(slots + (u * Images + k) * kSlot));
        use(v);
        if (u + Stages < left) fetch(u);
        copy_commit();
      }
    }
  }
};

// The kernels of a pass depend on one another and are launched with programmatic dependence: a
// kernel's blocks may start while the last ones of the kernel before it run, and wait here before
// they read its results (through pointers that are not __restrict__: a load that the compiler knows
// to be constant could be moved before the wait). Every block of every kernel waits, so that a
// kernel's completion implies that of all before it.
__device__ __forceinline__ void wait_for_kernel_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_kernel_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- host --------------------------------------------------------------------------------------

constexpr int kMaxNormChannels = 1 << 16;
constexpr long long kMaxNormBlocks = 0x7FFFFFFF;  // of one launch

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

// Bytes that both passes over a part of the views may read for the second one to find them in L2
// (126 MB; 80 MB read and as much written in turn is what was seen to stay).
constexpr long long kPartBytes = 72LL << 20;

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

// Cuts views into tiles of at most `most_cols` columns (at least the fewest whole groups that are
// whole vectors) and chunks of rows of about `chunk_bytes`. Lowers v.vec where a group is wider than a block's
// threads and not whole vectors (its tiles must not reach into the next group). False when there
// would be too many blocks.
inline bool cut_norm(NormShape& s, NormVector& v, long long batch, long long pixels, int channels,
                     int groups, int dtype, long long x_stride, long long grad_stride,
                     int most_cols, long long chunk_bytes) {
  s.batch = batch;
  s.pixels = pixels;
  s.channels = channels;
  s.groups = groups;
  s.group_channels = channels / groups;
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
  s.pieces = 1;
  s.group_cols = 0;
  most_cols = std::min(most_cols, kNormThreads);
  if (s.fold > 1) {
    s.tile_cols = s.cols;
    s.tiles = 1;
  } else if (unit <= kNormThreads) {
    s.tile_cols =
        static_cast<int>(std::min<long long>(s.cols, std::max(1LL, most_cols / unit) * unit));
    s.tiles = (s.cols + s.tile_cols - 1) / s.tile_cols;
  } else {
    s.group_cols = static_cast<int>(unit);
    s.pieces = static_cast<int>((unit + kNormThreads - 1) / kNormThreads);
    s.tile_cols = kNormThreads;
    s.tiles = groups * s.pieces;
  }
  const long long lanes = kNormThreads / s.tile_cols;  // rows that a block reads at once
  const long long tile_bytes = static_cast<long long>(s.tile_cols) * v.vec * dtype_bytes(dtype);
  const long long deep = chunk_bytes / tile_bytes / lanes;
  s.chunk_rows = static_cast<int>(std::max(1LL, std::min<long long>(deep, kMomentRows)) * lanes);
  const long long chunks = (s.rows + s.chunk_rows - 1) / s.chunk_rows;
  if (chunks > kMaxNormBlocks || batch > kMaxNormBlocks / s.tiles ||
      chunks > kMaxNormBlocks / std::max(1LL, batch * s.tiles))
    return false;
  s.chunks = static_cast<int>(chunks);
  return true;
}

// The plan of a call in passes over memory. Chunks are 64 KB, less where that would leave
// processors idle, more where a view would have over a thousand.
inline bool plan_passes(NormShape& s, NormVector& v, long long batch, long long pixels,
                        int channels, int groups, int dtype, long long x_stride,
                        long long grad_stride) {
  const long long view = pixels * channels * dtype_bytes(dtype);
  const long long chunk = std::max(
      view / 1024, std::max(4096LL, std::min(65536LL, batch * view / (4 * 148))));
  return cut_norm(s, v, batch, pixels, channels, groups, dtype, x_stride, grad_stride, kNormThreads,
                  chunk);
}

// Views that are taken together, first pass and second: as many as stay in L2 in between.
inline int views_at_once(const NormShape& s, int dtype, int images) {
  const long long view = s.pixels * s.channels * dtype_bytes(dtype) * images;
  return static_cast<int>(std::max(1LL, std::min(s.batch, kPartBytes / std::max(1LL, view))));
}

// Workspace. Forward: (mean, squares) of each group (or piece of one) for each chunk. Backward: sums
// of each channel for each chunk and of each view, and the two means of each group.
struct NormSpace {
  size_t parts, sums, means, total;  // offsets, and the end
};

inline NormSpace norm_space(const NormShape& s, bool backward) {
  const size_t groups = static_cast<size_t>(s.batch) * s.groups * sizeof(float2);
  const size_t channels = static_cast<size_t>(s.batch) * s.channels * sizeof(float2);
  NormSpace w;
  w.parts = 0;
  w.sums = align256((backward ? channels : groups * s.pieces) * s.chunks);
  w.means = w.sums + (backward ? align256(channels) : 0);
  w.total = w.means + (backward ? groups : 0);
  return w;
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
    if (plan_passes(s, v, batch, pixels, channels, groups, dtype, channels, channels))
      most = std::max(most, norm_space(s, backward).total);
  }
  return most;
}

// Launches a kernel on a stream, with programmatic dependence on the one before it if `after`.
template <typename... Params, typename... Args>
cudaError_t launch_kernel(void (*kernel)(Params...), unsigned int blocks, unsigned int threads,
                          size_t shared, cudaStream_t stream, bool after, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

template <typename T, int V, bool Silu, bool Drop>
struct Variant {
  using Type = T;
  static constexpr int kVec = V;
  static constexpr bool kSilu = Silu, kDrop = Drop;
};

// Calls fn(Variant) for a type, one of its vector widths, an activation and with or without
// dropout.
template <typename Fn>
int with_variant(int dtype, int vec, int activation, int threshold, Fn fn) {
  const bool silu = activation == DR_ACTIVATION_SILU, drop = threshold != 0;
  auto flags = [&](auto type, auto width) {
    using T = typename decltype(type)::Type;
    constexpr int V = decltype(width)::value;
    if (silu)
      return drop ? fn(Variant<T, V, true, true>()) : fn(Variant<T, V, true, false>());
    return drop ? fn(Variant<T, V, false, true>()) : fn(Variant<T, V, false, false>());
  };
  auto half = [&](auto type) {
    if (vec == 8) return flags(type, std::integral_constant<int, 8>());
    if (vec == 2) return flags(type, std::integral_constant<int, 2>());
    return flags(type, std::integral_constant<int, 1>());
  };
  if (dtype == DR_FLOAT16) return half(Variant<__half, 0, false, false>());
  if (dtype == DR_BFLOAT16) return half(Variant<__nv_bfloat16, 0, false, false>());
  if (vec == 4) return flags(Variant<float, 0, false, false>(), std::integral_constant<int, 4>());
  return flags(Variant<float, 0, false, false>(), std::integral_constant<int, 1>());
}

}  // namespace dr
