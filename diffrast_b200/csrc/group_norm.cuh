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
// A block's threads are `lanes` rows by the vectors of a tile of columns (threadIdx.y and .x), so
// that a thread keeps its channels, and their constants in registers, for all its rows. Blocks sum
// over channels, whatever their groups, so tiles may cut groups; a small kernel between the two
// passes joins the blocks' sums of each channel and the channels of each group, and leaves the
// constants of each view's channels for the second pass as it reads them.
//
// What a block does once costs as much as many of its rows: with the statistics joined per group in
// every block, divisions for the threads' places and the channels' constants formed by every
// thread, 1000 instructions of a warp were spent beside 35 for each row of vectors, and a view of
// 8 MB took 17 us with all its data in L2. Hence the block's shape, the sums by channel and the
// tables of constants.
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
  long long rows;    // rows of a view: pixels / fold
  long long pixels;
  int channels, groups, group_channels;
  int fold;
  int cols;          // vectors in a row
  int tile_cols;     // vectors in a tile of columns (the last tile may have fewer)
  int tiles;         // of a row
  int lanes;         // rows of a block's threads
  int chunk_rows;    // rows of one block's work
  int lane_rows;     // of those, rows of each lane
  int chunks;        // of a view
  // Elements between the rows of x and of the output's gradient.
  long long x_row, grad_row;
};

// Weight or bias. `data` is an address that may be read even where the parameter is absent (the
// constant's table then): a kernel given NULL instead faulted although it read the parameter only
// under a test, as a load that the compiler moves before the test does.
struct NormParam {
  const void* data;
  bool present;      // otherwise ones (weight) or zeros (bias)
  int dtype;
  long long view;    // elements between the views' rows (0: one row for all)
};

__device__ __forceinline__ float load_param(const NormParam& p, long long view, int channel) {
  const long long i = view * p.view + channel;
  if (p.dtype == DR_FLOAT32) return static_cast<const float*>(p.data)[i];
  if (p.dtype == DR_FLOAT16) return __half2float(static_cast<const __half*>(p.data)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p.data)[i]);
}

__device__ __forceinline__ float load_scale(const NormParam& w, long long view, int channel) {
  return w.present ? load_param(w, view, channel) : 1.0f;
}
__device__ __forceinline__ float load_shift(const NormParam& b, long long view, int channel) {
  return b.present ? load_param(b, view, channel) : 0.0f;
}

__device__ __forceinline__ void store_param(void* data, int dtype, long long i, float v) {
  if (dtype == DR_FLOAT32)
    static_cast<float*>(data)[i] = v;
  else if (dtype == DR_FLOAT16)
    static_cast<__half*>(data)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(data)[i] = __float2bfloat16_rn(v);
}

// 1 / (1 + exp(-z)) of a pair. The special-function unit gives 16 results a clock and processor,
// and with an exponential and a reciprocal for each value it was the busiest unit (74% of its rate
// in the second pass), so the two values share one reciprocal: 1 / a = b / (a b). Exponents are cut
// at 2^63, so that the product stays finite: below z = -43.7 the result is 2^-63 instead of less.
// Exponential and reciprocal are within two units in the last place of float32. A NaN gives 2^-63
// (the cut drops it), and its product with z is NaN again.
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  const float2 t = mul2(z, both(-1.4426950408889634f));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(fminf(t.x, 63.0f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(fminf(t.y, 63.0f)));
  e = add2(e, both(1.0f));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e.x * e.y));
  return mul2(both(r), make_float2(e.y, e.x));
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
// Blocks give a thread at most kThreadRows rows.
constexpr int kThreadRows = 128;

template <int V>
struct Moments {
  static constexpr int kPairs = Pairs<V>::kCount;
  Pairs<V> pivot, sum, square;  // the pivot is kept negated

  __device__ __forceinline__ void start(const Pairs<V>& v) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) pivot.p[j] = make_float2(-v.p[j].x, -v.p[j].y);
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) pivot.p[j] = sum.p[j] = square.p[j] = both(0.0f);
  }

  __device__ __forceinline__ void add(const Pairs<V>& v) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 d = add2(v.p[j], pivot.p[j]);
      sum.p[j] = add2(sum.p[j], d);
      square.p[j] = fma2(d, d, square.p[j]);
    }
  }

  // Turns the sums of n values into their mean (in sum) and their sum of squared deviations from
  // it (in square). A sum of squares that overflowed stays infinite.
  __device__ __forceinline__ void finish(float n) {
    const float2 inverse = both(n > 0.0f ? __fdividef(1.0f, n) : 0.0f);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 offset = mul2(sum.p[j], inverse);
      const float2 total = square.p[j];
      const float2 s = fma2(make_float2(-offset.x, -offset.y), sum.p[j], total);
      square.p[j].x = total.x < __int_as_float(0x7f800000) ? fmaxf(0.0f, s.x) : total.x;
      square.p[j].y = total.y < __int_as_float(0x7f800000) ? fmaxf(0.0f, s.y) : total.y;
      sum.p[j] = make_float2(offset.x - pivot.p[j].x, offset.y - pivot.p[j].y);
    }
  }

  // Joins the finished moments of n values with those of the lane at a distance:
  //   mean + (mean' - mean) n' / (n + n'),  squares + squares' + (mean' - mean)^2 n n' / (n + n').
  __device__ __forceinline__ void join_lane(int distance, float& n) {
    const float other = __shfl_xor_sync(0xFFFFFFFFu, n, distance);
    const float share = other > 0.0f ? __fdividef(other, n + other) : 0.0f;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      float2 m, q;
      m.x = __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].x, distance);
      q.x = __shfl_xor_sync(0xFFFFFFFFu, square.p[j].x, distance);
      m.y = V > 1 ? __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].y, distance) : 0.0f;
      q.y = V > 1 ? __shfl_xor_sync(0xFFFFFFFFu, square.p[j].y, distance) : 0.0f;
      const float2 d = make_float2(m.x - sum.p[j].x, m.y - sum.p[j].y);
      sum.p[j] = fma2(d, both(share), sum.p[j]);
      square.p[j] = fma2(mul2(d, both(n * share)), d, add2(square.p[j], q));
    }
    n += other;
  }
};

// (count, mean, squared deviations) of some values, and of those joined with others.
struct Moment {
  float n, mean, squares;

  __device__ __forceinline__ void join(const Moment& o) {
    const float share = o.n > 0.0f ? __fdividef(o.n, n + o.n) : 0.0f;
    const float d = o.mean - mean;
    mean = fmaf(d, share, mean);
    squares = fmaf(d * (n * share), d, squares + o.squares);
    n += o.n;
  }
  __device__ __forceinline__ Moment lane(int distance) const {
    return {__shfl_xor_sync(0xFFFFFFFFu, n, distance),
            __shfl_xor_sync(0xFFFFFFFFu, mean, distance),
            __shfl_xor_sync(0xFFFFFFFFu, squares, distance)};
  }
  __device__ __forceinline__ void join_warp() {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) join(lane(d));
  }
};

// NaN or infinite data give NaN statistics (their mean is NaN or infinite).
__device__ __forceinline__ float rstd_of(const Moment& m, float eps) {
  return isfinite(m.mean) ? rsqrtf(m.squares / m.n + eps) : __int_as_float(0x7fc00000);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

// Whether the rows of a warp's threads are joined by shuffles before the block's: the tile's
// columns divide the warp.
__device__ __forceinline__ bool warp_holds_rows() {
  return blockDim.x < 32 && 32 % blockDim.x == 0;
}

// A block's place: a chunk of rows, a tile of columns and a view; and its threads'.
struct NormPlace {
  int view, chunk, rows;
  int col;             // first element of this thread's vector in a row
  int count;           // rows of this thread
  long long first;     // its first row, counted over the views

  __device__ __forceinline__ NormPlace(const NormShape& s, int vec, int v, int tile, int c)
      : view(v), chunk(c) {
    const long long row0 = static_cast<long long>(c) * s.chunk_rows;
    rows = static_cast<int>(min(static_cast<long long>(s.chunk_rows), s.rows - row0));
    const int x = tile * s.tile_cols + threadIdx.x;
    const int y = threadIdx.y;
    col = x * vec;
    count = 0;
    if (x < s.cols && y < rows)
      count = rows == s.chunk_rows
                  ? s.lane_rows
                  : static_cast<int>(static_cast<unsigned int>(rows - y + s.lanes - 1) /
                                     static_cast<unsigned int>(s.lanes));
    first = v * s.rows + row0 + y;
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

  const T* at[Images];       // next row to fetch
  long long stride[Images];  // elements to the thread's row after it
  unsigned int slots;
  int count;

  __device__ __forceinline__ void image(int k, const T* base, long long row, const NormPlace& p,
                                        int lanes) {
    at[k] = base + p.first * row + p.col;
    stride[k] = lanes * row;
  }

  __device__ __forceinline__ void start(void* shared, int rows) {
    slots = static_cast<unsigned int>(__cvta_generic_to_shared(shared)) +
            (threadIdx.y * blockDim.x + threadIdx.x) * static_cast<unsigned int>(sizeof(P));
    count = rows;
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

  __device__ __forceinline__ Pairs<V> load(int u, int k) const {
    return load_pairs<T, V>(load_slot<P>(slots + (u * Images + k) * kSlot));
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
        for (int k = 0; k < Images; ++k) v[k] = load(u, k);
        use(v);
        if (u + Stages < left) fetch(u);
        copy_commit();
      }
    }
  }
};

// The constants of a thread's channels out of a table of one row of `channels` floats: those of
// the columns from `col` on, the channels repeated for each folded pixel.
template <int V>
__device__ __forceinline__ Pairs<V> load_row(const float* row, const NormShape& s, int col) {
  Pairs<V> r;
  if (V == 1) r.p[0].y = 0.0f;
  if (s.fold > 1 || V == 1) {
    int c = s.fold > 1 ? col % s.channels : col;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      r.set(j, row[c]);
      if (++c == s.channels) c = 0;
    }
  } else if constexpr (V == 2) {
    r.p[0] = *reinterpret_cast<const float2*>(row + col);
  } else if constexpr (V > 2) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float4 q = reinterpret_cast<const float4*>(row + col)[j];
      r.p[2 * j] = make_float2(q.x, q.y);
      r.p[2 * j + 1] = make_float2(q.z, q.w);
    }
  }
  return r;
}

// z = (x + shift) scale + bias, the tables that the forward pass leaves: [batch][3][channels].
template <int V>
struct Affine {
  Pairs<V> shift, scale, bias;

  __device__ __forceinline__ void load(const float* table, const NormShape& s, int view, int col) {
    table += static_cast<long long>(view) * 3 * s.channels;
    shift = load_row<V>(table, s, col);
    scale = load_row<V>(table + s.channels, s, col);
    bias = load_row<V>(table + 2 * s.channels, s, col);
  }
};

// The kernels that join the blocks' sums: a block has a run of whole groups of at most 8 channels
// together, or one group, of which it takes 8, 16 or 32 channels at a time (`width`) by as many
// lanes as it has threads for. With 32 channels to every block, two blocks read all the parts of 64
// channels, in 10 us; they are the only work between the two passes.
constexpr int kJoinThreads = 1024;

__host__ __device__ inline int join_run(int group_channels) {
  return group_channels > 8 ? 1 : 8 / group_channels;
}

struct JoinPlace {
  int view, group, channel, channels;  // first group and channel, and its channels
  int width, lanes, x, y;              // channels at a time, and the thread's place

  __device__ __forceinline__ JoinPlace(const NormShape& s, int view0) {
    const int run = join_run(s.group_channels);
    view = view0 + blockIdx.y;
    group = blockIdx.x * run;
    channel = group * s.group_channels;
    channels = min(run, s.groups - group) * s.group_channels;
    const int shift = s.group_channels > 16 ? 5 : s.group_channels > 8 ? 4 : 3;
    width = 1 << shift;
    lanes = kJoinThreads >> shift;
    x = threadIdx.x & (width - 1);
    y = threadIdx.x >> shift;
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

// Cuts views into tiles of at most `most_cols` columns and chunks of rows of about `chunk_bytes`.
inline void cut_norm(NormShape& s, const NormVector& v, long long batch, long long pixels,
                     int channels, int groups, int dtype, long long x_stride,
                     long long grad_stride, int most_cols, long long chunk_bytes) {
  s.batch = batch;
  s.pixels = pixels;
  s.channels = channels;
  s.groups = groups;
  s.group_channels = channels / groups;
  s.fold = v.fold;
  s.rows = pixels / s.fold;
  s.cols = static_cast<int>(static_cast<long long>(channels) * s.fold / v.vec);
  s.x_row = x_stride * s.fold;
  s.grad_row = grad_stride * s.fold;
  s.tiles = (s.cols + most_cols - 1) / most_cols;
  s.tile_cols = (s.cols + s.tiles - 1) / s.tiles;
  s.lanes = kNormThreads / s.tile_cols;
  const long long step = static_cast<long long>(s.tile_cols) * s.lanes * v.vec * dtype_bytes(dtype);
  const long long deep = std::max(1LL, std::min<long long>(chunk_bytes / step, kThreadRows));
  s.lane_rows = static_cast<int>(deep);
  s.chunk_rows = s.lane_rows * s.lanes;
  s.chunks = static_cast<int>((s.rows + s.chunk_rows - 1) / s.chunk_rows);
}

// Views, and pixels of a view, that still leave blocks and rows countable in 32 bits.
inline bool too_large(long long batch, long long pixels) {
  return batch > 0x7FFFFFFFLL || pixels > 0x7FFFFFFFLL;
}

// Blocks for each view of the kernels that join the blocks' sums (see JoinPlace).
inline unsigned int join_runs(const NormShape& s) {
  const int run = join_run(s.group_channels);
  return static_cast<unsigned int>((s.groups + run - 1) / run);
}

// Bytes that both passes over a part of the views may read for the second one to find them in L2.
constexpr long long kPartBytes = 72LL << 20;

#include <cstdlib>
inline long long envv(const char* n, long long d) { const char* e = getenv(n); return e ? atoll(e) : d; }
// Views that are taken together, first pass and second: as many as stay in L2 in between.
inline int views_at_once(long long batch, long long pixels, int channels, int dtype, int images) {
  const long long view = pixels * channels * dtype_bytes(dtype) * images;
  return static_cast<int>(
      std::max(1LL, std::min({batch, 65535LL, (envv("DRX_PART", 72) << 20) / std::max(1LL, view)})));
}

// The plan of a call in passes over memory. A block's start and the join of its sums cost as much
// as 16 rows of its threads, so chunks have about 64 KB (16 rows of 256 vectors); blocks fill the
// processors evenly, up to `resident` to each, or several times over.
inline void plan_passes(NormShape& s, const NormVector& v, long long batch, long long pixels,
                        int channels, int groups, int dtype, long long x_stride,
                        long long grad_stride, int images) {
  const long long view = pixels * channels * dtype_bytes(dtype);
  const long long part = view * views_at_once(batch, pixels, channels, dtype, images);
  const long long processors = 148, resident = images == 1 ? 4 : 3, chunk = envv("DRX_CHUNK", 65536);
  const long long each = (part + processors * chunk / 2) / (processors * chunk);
  const long long blocks = each <= resident ? std::max(1LL, each) * processors
                                            : (each + resident / 2) / resident * resident * processors;
  cut_norm(s, v, batch, pixels, channels, groups, dtype, x_stride, grad_stride, kNormThreads,
           std::max(4096LL, (part + blocks - 1) / blocks));
}

// Workspace: a pair of each channel for each chunk; for the backward pass also one of each view and
// channel, and the table of the second pass.
struct NormSpace {
  size_t parts, sums, table, total;  // offsets, and the end
};

inline NormSpace norm_space(const NormShape& s, bool backward) {
  const size_t channels = static_cast<size_t>(s.batch) * s.channels * sizeof(float2);
  NormSpace w;
  w.parts = 0;
  w.sums = align256(channels * s.chunks);
  w.table = w.sums + (backward ? align256(channels) : 0);
  w.total = w.table + (backward ? align256(channels) : 0);
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
    plan_passes(s, v, batch, pixels, channels, groups, dtype, channels, channels,
                backward ? 2 : 1);
    most = std::max(most, norm_space(s, backward).total);
  }
  return most;
}

// Launches a kernel on a stream, with programmatic dependence on the one before it if `after`.
template <typename... Params, typename... Args>
cudaError_t launch_kernel(void (*kernel)(Params...), dim3 blocks, dim3 threads,
                          size_t shared, cudaStream_t stream, bool after, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = blocks;
  config.blockDim = threads;
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
