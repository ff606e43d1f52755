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
// Where the pixels are no multiple of that, or views do not start on 16 bytes, the rows start at
// the view's first whole vector (`lead` elements in), which turns their channels by as many, and
// the elements before and after the rows are left over for one block of the view, one by one.
// A block's threads are `lanes` rows by the vectors of a tile of columns (threadIdx.y and .x), so
// that a thread keeps its channels, and their constants in registers, for all its rows. Blocks sum
// over channels, whatever their groups, so tiles may cut groups; a small kernel between the two
// passes joins the blocks' sums of each channel and the channels of each group, and leaves the
// constants of each view's channels for the second pass as it reads them.
//
// A row of vectors costs a warp 53 instructions in the first pass, so what a block does once is kept
// small: its shape gives the threads their places without a division, it sums by channel whatever
// the groups, and it reads the channels' constants from tables.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include <cooperative_groups.h>

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
  int turned;        // rows start at the view's first whole vector: V, or 0
  int leftover;      // values of each channel outside the rows
  int cols;          // vectors in a row
  int tile_cols;     // vectors in a tile of columns (the last tile may have fewer)
  int tiles;         // of a row
  int lanes;         // rows of a block's threads
  int chunk_rows;    // rows of one block's work
  int lane_rows;     // of those, rows of each lane
  int chunks;        // of a view
  // Elements between the rows, and between the views, of x and of the output's gradient (those of
  // the contiguous results are out_row and out_view).
  long long x_row, grad_row, out_row;
  long long x_view, grad_view, out_view;

  // Elements of a view before its rows.
  __device__ __forceinline__ int lead(int view) const {
    return turned == 0 ? 0 : static_cast<int>(-(view * out_view) & (turned - 1));
  }
  // The elements left over in a channel of a view with `lead` elements before its rows.
  template <typename Use>
  __device__ __forceinline__ void for_leftovers(int lead, int channel, Use use) const {
    for (int e = channel; e < lead; e += channels) use(static_cast<long long>(e));
    const long long end = lead + rows * out_row;
    const int turn = static_cast<int>(end % channels);
    long long e = end + (channel < turn ? channel - turn + channels : channel - turn);
    for (; e < out_view; e += channels) use(e);
  }
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

__device__ __forceinline__ float power_of_two(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// exp(-z) of a pair. Off by (1.23 |z| + 4) u relative (u = 2^-24), mostly from rounding z / ln 2, which
// moves a function of z like a change of z by as much. Below 2^-126 it is 0.
__device__ __forceinline__ float2 exp_minus(float2 z) {
  const float2 t = mul2(z, both(-1.4426950408889634f));
  return make_float2(power_of_two(t.x), power_of_two(t.y));
}

// 1 / d of a pair. The special-function unit gives 16 results a clock and processor, and an
// exponential and a reciprocal for each value keep it busy for 29 of the 43 us of the second pass over
// four images of 512 x 512 x 64 bfloat16. One reciprocal for both values, 1 / a = b / (a b), takes
// their forward pass from 74 to 70 us and 2 us off the backward pass, but the product leaves the
// range of float32 with exp(-z) above 2^63, and a NaN spoils its neighbour. What it takes to tell
// gives the time back: 79 us with a test of each pair, 74 of each vector, 72 with all rows again after
// a test at their end (in registers that the passes do not have), 73 with exp(-|z|), at most 1, and
// selects.
__device__ __forceinline__ float2 reciprocals(float2 d) {
  return make_float2(reciprocal(d.x), reciprocal(d.y));
}

// The activations: SiLU, z / (1 + exp(-z)), or a clamp from below that is the identity with bound
// -infinity and ReLU with bound 0. The comparisons are written so that NaN passes, as it does
// through all three.
template <bool Silu>
__device__ __forceinline__ float2 activate(float2 z, float bound) {
  if (Silu) return mul2(z, reciprocals(add2(exp_minus(z), both(1.0f))));
  return make_float2(z.x <= bound ? bound : z.x, z.y <= bound ? bound : z.y);
}

// q times the derivative at z: s (1 + z (1 - s)) for SiLU, s the sigmoid. ReLU's is 0 at 0.
//
// 1 - s is formed as exp(-z) s: the difference from an s that is a few units off is wrong by as many,
// and z multiplies them (with z = 1000 the slope came out 6e-5 from 1). Where exp(-z) passes 2^126, s
// is 0 or next to it; the cut keeps 0 times infinity out of the product.
template <bool Silu>
__device__ __forceinline__ float2 activate_grad(float2 q, float2 z, float bound) {
  if (Silu) {
    const float2 e = exp_minus(z), s = reciprocals(add2(e, both(1.0f)));
    const float2 rest = mul2(make_float2(fminf(e.x, 0x1p126f), fminf(e.y, 0x1p126f)), s);
    return mul2(q, mul2(s, fma2(z, rest, both(1.0f))));
  }
  return make_float2(z.x <= bound ? 0.0f : q.x, z.y <= bound ? 0.0f : q.y);
}

// Running moments of V channels. Values are summed as differences from the thread's first value
// k: with n values, sum (x - k)^2 is at most n times their sum of squared deviations from their
// mean (k is one of them), so rounding grows by no more than n, whatever the offset of the data.
// Plans give a thread at most kThreadRows rows.
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

// A sum with what its roundings have left out (Kahan's compensated summation), for the lanes of the
// joins, which may add thousands of chunks one after the other: in plain 32 bits a sum of equal terms
// over 1.5 GB was 250 units in the last place off. (Sums in 64 bits cost the join of a view of 268 MB
// 3 us, most of it for the conversions.)
struct LongSum {
  float sum = 0.0f, lost = 0.0f;

  __device__ __forceinline__ void add(float v) {
    const float term = v - lost, total = sum + term;
    // An infinite sum stays infinite.
    lost = fabsf(total) < __int_as_float(0x7f800000) ? (total - sum) - term : 0.0f;
    sum = total;
  }
};

// The moments of a lane's chunks: Moment::join with long sums.
struct LongMoment {
  float n = 0.0f;
  LongSum mean, squares;

  __device__ __forceinline__ void join(float count, float2 chunk) {
    const float share = count > 0.0f ? __fdividef(count, n + count) : 0.0f;
    const float d = chunk.x - mean.sum;
    mean.add(d * share);
    squares.add(fmaf(d * (n * share), d, chunk.y));
    n += count;
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
__host__ __device__ inline bool warp_holds_rows(int tile_cols) {
  return tile_cols < 32 && 32 % tile_cols == 0;
}

// A block's place: a chunk of rows, a tile of columns and a view; and its threads'.
struct NormPlace {
  int view, chunk, rows;
  int col;             // first element of this thread's vector in a row
  int lead;            // elements before the view's rows
  int count;           // rows of this thread
  long long row;       // its first row

  __device__ __forceinline__ NormPlace(const NormShape& s, int vec, int v, int tile, int c)
      : view(v), chunk(c) {
    const long long row0 = static_cast<long long>(c) * s.chunk_rows;
    rows = static_cast<int>(min(static_cast<long long>(s.chunk_rows), s.rows - row0));
    const int x = tile * s.tile_cols + threadIdx.x;
    const int y = threadIdx.y;
    col = x * vec;
    lead = s.lead(v);
    count = 0;
    if (x < s.cols && y < rows)
      count = rows == s.chunk_rows
                  ? s.lane_rows
                  : static_cast<int>(static_cast<unsigned int>(rows - y + s.lanes - 1) /
                                     static_cast<unsigned int>(s.lanes));
    row = row0 + y;
  }

  // Where this thread's first vector is in an image.
  __device__ __forceinline__ long long at(long long view_size, long long row_size) const {
    return view * view_size + lead + row * row_size + col;
  }
  // The view's first row of chunks and tiles, which takes what is left over.
  __device__ __forceinline__ bool takes_leftovers(const NormShape& s, int tile) const {
    return s.leftover > 0 && chunk == 0 && tile == 0;
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
  else if constexpr (sizeof(P) == 8)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(p.x), "=r"(p.y) : "r"(at) : "memory");
  else if constexpr (sizeof(P) == 4)
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(p) : "r"(at) : "memory");
  else
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(p) : "r"(at) : "memory");
  return p;
}

// A thread's rows on their way to it: it copies its own vectors (of Images images) into its own
// slots of shared memory, Stages rows ahead of the one it works on. No slot is shared, so the
// copies need no barriers, and they hold no registers: with batches of loads in registers instead,
// the sums of the backward pass read memory at 1.9 TB/s, for want of bytes under way; so, at 5.0.
template <typename T, int V, int Images, int Stages>
struct RowRing {
  using P = Packed<T, V>;
  static constexpr unsigned int kSlot = sizeof(P) * kNormThreads;
  static constexpr size_t kBytes = static_cast<size_t>(kSlot) * Images * Stages;

  const T* at[Images];       // next row to fetch
  long long stride[Images];  // elements to the thread's row after it
  unsigned int slots;
  int count;

  __device__ __forceinline__ void image(int k, const T* base, long long view, long long row,
                                        const NormPlace& p, int lanes) {
    at[k] = base + p.at(view, row);
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

  template <typename Use>
  __device__ __forceinline__ void row(int u, Use use) const {
    copy_wait<Stages - 1>();
    Pairs<V> v[Images];
#pragma unroll
    for (int k = 0; k < Images; ++k) v[k] = load(u, k);
    use(v);
  }

  // Calls use(vectors) for the rows in order. While two rounds of the ring are left, nothing is
  // tested.
  template <typename Use>
  __device__ __forceinline__ void for_rows(Use use) {
    int left = count;
    for (; left >= 2 * Stages; left -= Stages) {
#pragma unroll
      for (int u = 0; u < Stages; ++u) {
        row(u, use);
        fetch(u);
        copy_commit();
      }
    }
    for (; left > 0; left -= Stages) {
#pragma unroll
      for (int u = 0; u < Stages; ++u) {
        if (u >= left) break;
        row(u, use);
        if (u + Stages < left) fetch(u);
        copy_commit();
      }
    }
  }
};

// The constants of a thread's channels out of a table of one row of `channels` floats: those of
// the columns from `col` on (`lead` further where rows are turned), the channels repeated for each
// folded pixel.
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
// together, or one group of at most 32, by as many lanes as it has threads for (with 32 channels to
// every block, two blocks read all the parts of 64 channels, 3 us longer; they are the
// only work between the two passes). Of wider groups it has 32 channels, and a second kernel joins the
// channels of each group (the norm of 301 x 301 x 256 float32 in one group takes 61 us so, 116
// us with one block for the group).
constexpr int kJoinThreads = 1024;
constexpr int kJoinChannels = 32;

__host__ __device__ inline int join_channels(int group_channels) {
  if (group_channels > kJoinChannels) return kJoinChannels;
  return group_channels > 8 ? group_channels : 8 / group_channels * group_channels;
}

// log2 of the threads in a row of such a block, at least one for each of its `run` channels.
__host__ __device__ inline int join_shift(int run) { return run > 16 ? 5 : run > 8 ? 4 : 3; }

struct JoinPlace {
  int view, channel, channels;     // first channel, and channels
  int width, lanes, x, y;          // of a row of threads, and the thread's place

  __device__ __forceinline__ JoinPlace(const NormShape& s, int view0) {
    const int run = join_channels(s.group_channels);
    view = view0 + blockIdx.y;
    channel = blockIdx.x * run;
    channels = min(run, s.channels - channel);
    const int shift = join_shift(run);
    width = 1 << shift;
    lanes = blockDim.x >> shift;
    x = threadIdx.x & (width - 1);
    y = threadIdx.x >> shift;
  }
};

// ---- clusters ----------------------------------------------------------------------------------
//
// A slab is a tile of whole groups of one view. Where a cluster of blocks can hold one in shared
// memory, each block copies its share of the rows, sums over it, reads the other blocks' sums of
// each channel from their shared memory, and finishes its rows from its own: one launch, and the
// image is read once and written once. (Larger teams, over all processors and through memory, had
// some 18 us from one slab's copies to its results, and too little shared memory to cover that with
// other slabs: 171 us where the two passes took 74, on four images of 512 x 512 x 64.)

constexpr int kMostCluster = 16;

struct ClusterPlan {
  int size;              // blocks of a cluster
  long long slabs;       // of all views
  int block_rows;        // rows of a block's share
  unsigned int slots;    // bytes of the rows
  unsigned int entries;  // bytes of the joins' entries, after them
  unsigned int shared;   // bytes in all
};

// A thread's place in a tile.
struct TileThread {
  int x, y;    // vector and row
  int thread;  // of the block's
  int threads;
};

// A block's share of a slab.
struct ClusterShare {
  int view, tile, rank, rows;
  int col;           // first element of the thread's vector in a row
  int mine;          // the thread's rows
  int channel;       // first channel of the tile
  int channels;      // of the tile
  long long row;     // the thread's first row
  TileThread at;

  __device__ __forceinline__ ClusterShare(const NormShape& s, const ClusterPlan& t, int vec) {
    at.thread = threadIdx.x;
    at.threads = kNormThreads;
    at.y = threadIdx.x / s.tile_cols;
    at.x = threadIdx.x - at.y * s.tile_cols;
    const unsigned int slab = blockIdx.x / t.size;
    rank = static_cast<int>(blockIdx.x - slab * t.size);
    view = static_cast<int>(slab / s.tiles);
    tile = static_cast<int>(slab - view * static_cast<unsigned int>(s.tiles));
    const long long row0 = static_cast<long long>(rank) * t.block_rows;
    rows = static_cast<int>(max(0LL, min(static_cast<long long>(t.block_rows), s.rows - row0)));
    const int x = tile * s.tile_cols + at.x;
    col = x * vec;
    mine = x < s.cols && at.y < s.lanes && at.y < rows ? (rows - at.y + s.lanes - 1) / s.lanes : 0;
    channel = s.fold > 1 ? 0 : tile * s.tile_cols * vec;
    channels = s.fold > 1 ? s.channels : min(s.tile_cols, s.cols - tile * s.tile_cols) * vec;
    row = row0 + at.y;
  }

  // Where this thread's first vector is in an image.
  __device__ __forceinline__ long long in(long long view_size, long long row_size) const {
    return view * view_size + row * row_size + col;
  }

  // Values of a channel in a rank's share.
  __device__ __forceinline__ float values_of(const NormShape& s, const ClusterPlan& t, int r) const {
    const long long left = s.rows - static_cast<long long>(r) * t.block_rows;
    return static_cast<float>(max(0LL, min(static_cast<long long>(t.block_rows), left))) *
           static_cast<float>(s.fold);
  }
};

// The constants of a thread's channels out of a row of a tile's in shared memory.
template <int V>
__device__ __forceinline__ Pairs<V> load_constants(const float* row, const NormShape& s,
                                                   const ClusterShare& p) {
  Pairs<V> r;
  if (V == 1) r.p[0].y = 0.0f;
  int c = p.col - p.channel;
  if (s.fold > 1) c %= s.channels;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    r.set(j, row[c]);
    if (++c == s.channels && s.fold > 1) c = 0;
  }
  return r;
}

// Lanes (a power of two, at most 32) that a block's threads can give to each of `items`.
__device__ __forceinline__ int lanes_for(int items) {
  if (items >= kNormThreads) return 1;
  return min(32, 1 << (31 - __clz(kNormThreads / items)));
}

// One thread's rows of a slab in shared memory.
template <typename T, int V, int Images>
struct SlabRows {
  using P = Packed<T, V>;
  static constexpr unsigned int kSlot = sizeof(P) * kNormThreads;

  unsigned int slots;
  int count;

  // Starts the copies of rows first, first + lanes, ... of the images, `count` of them.
  __device__ __forceinline__ void fetch(const T* const (&from)[Images],
                                        const long long (&stride)[Images]) {
    const T* at[Images];
#pragma unroll
    for (int k = 0; k < Images; ++k) at[k] = from[k];
    unsigned int to = slots;
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
#pragma unroll
      for (int k = 0; k < Images; ++k) {
        copy_async<sizeof(P)>(to + k * kSlot, at[k]);
        at[k] += stride[k];
      }
      to += Images * kSlot;
    }
    copy_commit();
  }

  template <typename Use>
  __device__ __forceinline__ void for_rows(Use use) const {
    unsigned int at = slots;
#pragma unroll 2
    for (int i = 0; i < count; ++i) {
      Pairs<V> v[Images];
#pragma unroll
      for (int k = 0; k < Images; ++k) v[k] = load_pairs<T, V>(load_slot<P>(at + k * kSlot));
      use(v);
      at += Images * kSlot;
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
  return data != nullptr && (!known_dtype(dtype) || (rows != 1 && rows != batch) ||
                             !aligned_to(data, dtype_bytes(dtype)));
}

inline float norm_bound(int activation) {
  return activation == DR_ACTIVATION_RELU ? 0.0f : -__builtin_huge_valf();
}

// A vector width and a number of folded pixels, which rows may start with at any element.
struct NormVector {
  int vec, fold;
  bool turned;
};

inline int widest_vector(int dtype) { return 16 / dtype_bytes(dtype); }
inline int folded_pixels(int channels, int dtype) {
  return widest_vector(dtype) / greatest_divisor(channels, widest_vector(dtype));
}
// Whether rows of folded pixels have few enough columns, and views a row of them at least.
inline bool can_fold(long long pixels, int channels, int dtype) {
  const long long row = static_cast<long long>(channels) * folded_pixels(channels, dtype);
  return row / widest_vector(dtype) <= kNormThreads &&
         pixels * channels >= row + widest_vector(dtype) - 1;
}

// The widest vectors that the addresses, the strides and the channels allow. Strides are elements
// between the pixels of x and of the output's gradient (`channels` where there is none).
inline NormVector choose_vector(long long pixels, int channels, int dtype, long long x_stride,
                                long long grad_stride,
                                std::initializer_list<const void*> pointers, bool turn) {
  const int size = dtype_bytes(dtype), widest = widest_vector(dtype);
  auto fits = [&](int v) {
    for (const void* p : pointers)
      if (!aligned_to(p, static_cast<size_t>(v) * size)) return false;
    return true;
  };
  auto divides = [&](int v) {
    return channels % v == 0 && x_stride % v == 0 && grad_stride % v == 0;
  };
  if (fits(widest)) {
    if (divides(widest)) return {widest, 1, false};
    const int fold = folded_pixels(channels, dtype);
    if (x_stride == channels && grad_stride == channels && can_fold(pixels, channels, dtype)) {
      if (pixels % fold == 0) return {widest, fold, false};
      if (turn) return {widest, fold, true};
    }
  }
  for (int v : {4, 2})
    if (v < widest && fits(v) && divides(v)) return {v, 1, false};
  return {1, 1, false};
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
  s.turned = v.turned ? v.vec : 0;
  s.rows = v.turned ? (pixels * channels - (v.vec - 1)) / (static_cast<long long>(channels) * v.fold)
                    : pixels / v.fold;
  s.leftover = static_cast<int>(pixels - s.rows * v.fold);
  s.cols = static_cast<int>(static_cast<long long>(channels) * s.fold / v.vec);
  s.x_row = x_stride * s.fold;
  s.grad_row = grad_stride * s.fold;
  s.out_row = static_cast<long long>(channels) * s.fold;
  s.x_view = x_stride * pixels;
  s.grad_view = grad_stride * pixels;
  s.out_view = channels * pixels;
  s.tiles = (s.cols + most_cols - 1) / most_cols;
  s.tile_cols = (s.cols + s.tiles - 1) / s.tiles;
  s.lanes = kNormThreads / s.tile_cols;
  const long long step = static_cast<long long>(s.tile_cols) * s.lanes * v.vec * dtype_bytes(dtype);
  const long long deep = std::max(1LL, std::min<long long>(chunk_bytes / step, kThreadRows));
  s.lane_rows = static_cast<int>(deep);
  s.chunk_rows = s.lane_rows * s.lanes;
  s.chunks = static_cast<int>((s.rows + s.chunk_rows - 1) / s.chunk_rows);
}

// Views, and pixels of a view, that leave blocks and rows countable in 32 bits, and at most 2^48
// elements (more than any device holds), so that no offset or byte count passes 64.
inline bool too_large(long long batch, long long pixels, long long stride) {
  constexpr long long kMost = 1LL << 48;
  return batch > 0x7FFFFFFFLL || pixels > 0x7FFFFFFFLL ||
         (batch > 0 && pixels > 0 && stride > kMost / batch / pixels);
}

// Blocks for each view of the kernels that join the blocks' sums (see JoinPlace), and their
// threads: all or, where a view has few chunks, a warp for each channel (of 64 views of 512 KB each
// the forward pass takes 26 us so and 33 us with 1024 threads to every block).
inline unsigned int join_runs(const NormShape& s) {
  const int run = join_channels(s.group_channels);
  return static_cast<unsigned int>((s.channels + run - 1) / run);
}
inline unsigned int join_threads(const NormShape& s) {
  const int width = 1 << join_shift(join_channels(s.group_channels));
  return static_cast<long long>(s.chunks) * width <= kJoinThreads ? 32 * width : kJoinThreads;
}

constexpr int kMostShared = 220 * 1024;  // dynamic shared memory of a block

// Blocks of a processor that the kernels' registers allow, forward and backward.
constexpr int kResident[2] = {4, 3};

// Largest view that is taken in clusters, both ways. One view of 32 KB (16 x 16 x 64 bfloat16) takes
// 4.8 us forward and 4.5 us backward in clusters, 6.2 and 7.0 us in two passes, and 1024 of them 21
// and 34 us against 47 and 56 us. Four of 256 KB take 7.4 and 8.1 us against 7.8 and 9.4 us, and 256
// of them 43 and 71 us against 46 and 68 us: there the backward pass is even, ahead with few views
// and behind with many. At 512 KB clusters are behind (four: 8.8 and 10.4 us against 8.5 and 10.9 us;
// 256: 79 and 137 us against 75 and 119 us).
constexpr long long kClusterBytes = 1LL << 18;

// The plan of a call in clusters, or false where none fits: tiles of whole groups, and blocks to a
// cluster, by the estimated time in microseconds. A block's own is what is fixed (2, or 3 with a
// cluster, and with clusters the start of all blocks of a wave: sixteen views of 128 KB took 10.7 us
// in 512 blocks of clusters and 6.5 us in 128 without), its bytes at a processor's share of the
// memory, and its rows' instructions, or the cache lines that its warps' copies touch if those are
// slower; the blocks of a processor overlap, as many as its registers and shared memory hold.
//
// The constants: 43.5e3 bytes a microsecond are a processor's share of the measured copy rate (6446
// GB/s by 148); 1.9e3 clocks are a microsecond, and a clock moves one line of 128 bytes between a
// processor and L2 (a warp's copy touches 4, or 32 / cols with rows of fewer vectors); 0.16 and 0.31 us
// are a row of the 8 warps through both loops, some 150 and 290 instructions a warp at four a clock;
// rows of a tile shorter than 64 and 32 bytes waste parts of their 32-byte sectors (1.3 and 2.0). The
// fixed times, 1.0 for joins and constants and 0.01 a block, are set by hand to timings of 1 to 1024
// views of 8 to 512 KB. They choose between plans that are all right, and bound nothing.
inline bool plan_clusters(NormShape& s, ClusterPlan& t, const NormVector& v, long long batch,
                          long long pixels, int channels, int groups, int dtype,
                          long long x_stride, long long grad_stride, int images, int processors) {
  const int d = channels / groups, size = dtype_bytes(dtype);
  const int most_cols = kNormThreads / 2;
  const int row_cols = static_cast<int>(static_cast<long long>(channels) * v.fold / v.vec);
  const int unit = v.fold > 1 ? row_cols : d / greatest_divisor(d, v.vec);
  const long long rows = pixels / v.fold;
  double best = 1e30;
  if (unit > most_cols || pixels * channels * size > kClusterBytes) return false;
  for (int cols = unit; cols <= std::min(row_cols, most_cols); cols *= 2) {
    const long long tiles = (row_cols + cols - 1) / cols;
    const long long slabs = batch * tiles;
    const int lanes = kNormThreads / cols, width = cols * v.vec;
    const int lines = warp_holds_rows(cols) ? kNormThreads / 32 : lanes;
    const long long entries = static_cast<long long>(align256(sizeof(float2) * lines * width));
    const long long extra = entries + static_cast<long long>(align256(20 * width));
    const long long slot = static_cast<long long>(kNormThreads) * v.vec * size * images;
    for (int team = 1; team <= kMostCluster; team *= 2) {
      const long long block_rows = (rows + team - 1) / team;
      const long long lane_rows = (block_rows + lanes - 1) / lanes;
      const long long shared = lane_rows * slot + extra;
      if (shared > kMostShared || slabs * team > 0x7FFFFFFF || lane_rows > kThreadRows) continue;
      const double here = static_cast<double>(
          std::min<long long>(kResident[images - 1], 228 * 1024 / (shared + 2048)));
      const double narrow = tiles == 1 || width * size >= 64 ? 1.0 : width * size >= 32 ? 1.3 : 2.0;
      const double move =
          static_cast<double>(block_rows) * width * size * (images + 1) * narrow / 43.5e3;
      const double lines = 8.0 * (cols < 8 ? 32.0 / cols : 4.0) * (images + 1) / 1.9e3;
      const double row = std::max(images == 1 ? 0.16 : 0.31, lines);
      const double work = static_cast<double>(lane_rows) * row + 1.0;
      const double blocks = static_cast<double>(slabs * team);
      const double fixed =
          team == 1 ? 2.0
                    : (team <= 8 ? 3.0 : 3.5) + 0.01 * std::min(blocks, processors * here);
      const double each = blocks / processors;
      const double waves = std::ceil(each / here);
      const double together = std::min(here, std::ceil(each));
      const double time =
          waves * std::max({move * together, work * together, move + work + fixed});
      if (time >= best) continue;
      best = time;
      t = ClusterPlan{team,
                      slabs,
                      static_cast<int>(block_rows),
                      static_cast<unsigned int>(lane_rows * slot),
                      static_cast<unsigned int>(entries),
                      static_cast<unsigned int>(shared)};
      cut_norm(s, v, batch, pixels, channels, groups, dtype, x_stride, grad_stride, cols, 0);
      s.tiles = static_cast<int>(tiles);
      s.tile_cols = cols;
      s.lanes = lanes;
    }
  }
  return best < 1e30;
}

// Workspace of a backward pass in clusters: the views' sums.
inline size_t cluster_space(const NormShape& s) {
  return sizeof(float2) * static_cast<size_t>(s.batch) * s.channels;
}

// Processors of the current device, looked up once for each.
inline int processors() {
  static std::atomic<int> known[64];
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 148;
  if (device < 64 && (count = known[device].load(std::memory_order_relaxed)) > 0) return count;
  if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 148;
  if (device < 64) known[device].store(count, std::memory_order_relaxed);
  return count;
}

// Launches a kernel of clusters.
template <auto Kernel, typename... Args>
int launch_clusters(const ClusterPlan& t, cudaStream_t stream, Args... args) {
  static std::atomic<unsigned long long> allowed;  // devices where its limits were raised
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return static_cast<int>(err);
  const unsigned long long bit = device < 64 ? 1ull << device : 0;
  if ((allowed.load(std::memory_order_relaxed) & bit) == 0) {
    err = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (err == cudaSuccess)
      err = cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err != cudaSuccess) return static_cast<int>(err);
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned int>(t.slabs * t.size));
  config.blockDim = dim3(kNormThreads);
  config.dynamicSmemBytes = t.shared;
  config.stream = stream;
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = t.size;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = t.size > 1 ? 1 : 0;
  err = cudaLaunchKernelEx(&config, Kernel, args...);
  return err == cudaSuccess ? launch_status() : static_cast<int>(err);
}

// Views of one launch.
inline int views_at_once(long long batch) {
  return static_cast<int>(std::min(batch, 65535LL));
}

// The plan of a call in passes over memory. A block's start and the join of its sums cost as much
// as 16 rows of its threads, and with long blocks the last ones run alone, so a block has about 24
// rows of them (96 KB of 16-byte vectors); blocks fill the processors evenly, up to `resident` to
// each, or several times over. Four images of 512 x 512 x 64 bfloat16, called again and again, take
// 72, 72, 82 and 100 us forward with 16, 24, 48 and 112 rows, and 113, 113, 120 and 135 us backward;
// eight of 128 x 128 x 256 with dropout take 55, 55, 63 and 79 us, and 97, 97, 94 and 151 us.
inline void plan_passes(NormShape& s, const NormVector& v, long long batch, long long pixels,
                        int channels, int groups, int dtype, long long x_stride,
                        long long grad_stride, int images, int processors) {
  const int size = dtype_bytes(dtype), resident = kResident[images - 1];
  const long long bytes = pixels * channels * size * views_at_once(batch);
  const long long row = static_cast<long long>(kNormThreads) * v.vec * size;
  const long long chunk = 24 * row;
  const long long each = (bytes + processors * chunk / 2) / (processors * chunk);
  const long long blocks =
      processors * (each <= resident ? std::max(1LL, each)
                                     : (each + resident / 2) / resident * resident);
  cut_norm(s, v, batch, pixels, channels, groups, dtype, x_stride, grad_stride, kNormThreads,
           std::max(row, (bytes + blocks - 1) / blocks));
}

// Workspace: a pair of each channel for each chunk, and one of each view and channel; for the
// backward pass also the table of the second pass.
struct NormSpace {
  size_t parts, sums, table, total;  // offsets, and the end
};

inline NormSpace norm_space(const NormShape& s, bool backward) {
  const size_t channels = static_cast<size_t>(s.batch) * s.channels * sizeof(float2);
  NormSpace w;
  w.parts = 0;
  w.sums = align256(channels * s.chunks);
  w.table = w.sums + align256(channels);
  w.total = w.table + (backward ? align256(channels) : 0);
  return w;
}

// The larger workspace of all the vector widths that a call may turn out to take.
inline size_t norm_workspace_bytes(long long batch, long long pixels, int channels, int groups,
                                   int dtype, bool backward) {
  const int widest = widest_vector(dtype), images = backward ? 2 : 1;
  const int fold = folded_pixels(channels, dtype);
  size_t most = 0;
  auto passes = [&](const NormVector& v) {
    NormShape s;
    plan_passes(s, v, batch, pixels, channels, groups, dtype, channels, channels, images,
                processors());
    most = std::max(most, norm_space(s, backward).total);
  };
  for (NormVector v : {NormVector{widest, fold, false}, NormVector{4, 1, false},
                       NormVector{2, 1, false}, NormVector{1, 1, false}}) {
    if (v.fold > 1 && (pixels % fold != 0 || !can_fold(pixels, channels, dtype))) continue;
    if (v.fold == 1 && (channels % v.vec != 0 || v.vec > widest)) continue;
    NormShape s;
    ClusterPlan t;
    if (plan_clusters(s, t, v, batch, pixels, channels, groups, dtype, channels, channels, images,
                      processors())) {
      if (backward) most = std::max(most, cluster_space(s));
      continue;
    }
    passes(v);
    if (fold > 1 && pixels % fold != 0 && can_fold(pixels, channels, dtype))
      passes({widest, fold, true});
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
    if (vec == 4) return flags(type, std::integral_constant<int, 4>());
    if (vec == 2) return flags(type, std::integral_constant<int, 2>());
    return flags(type, std::integral_constant<int, 1>());
  };
  if (dtype == DR_FLOAT16) return half(Variant<__half, 0, false, false>());
  if (dtype == DR_BFLOAT16) return half(Variant<__nv_bfloat16, 0, false, false>());
  if (vec == 4) return flags(Variant<float, 0, false, false>(), std::integral_constant<int, 4>());
  if (vec == 2) return flags(Variant<float, 0, false, false>(), std::integral_constant<int, 2>());
  return flags(Variant<float, 0, false, false>(), std::integral_constant<int, 1>());
}

}  // namespace dr
