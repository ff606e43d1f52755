// Group normalisation with an activation and optional dropout: the forward pass (the formulas and
// the way views are cut up are in group_norm.cuh).
#include "group_norm.cuh"

namespace dr {
namespace {

constexpr int kStages = 8;  // rows that a thread has under way

// Joins the threads' moments of a block's rows into those of the tile's groups: within a thread
// over the neighbouring channels of a group, then over the rows, then over a group's columns (and
// folded pixels).
template <int V>
constexpr size_t join_bytes() {
  return sizeof(float2) * kNormThreads * (V + (V + 1) / 2);
}

template <int V, typename Done>
__device__ __forceinline__ void join_block(Moments<V>& moments, const TileThread& t,
                                           const NormShape& s, const NormTile& tile, int rows,
                                           void* shared, Done done) {
  auto* entry = static_cast<float2*>(shared);   // [kNormThreads * V]
  float2* column = entry + kNormThreads * V;    // [kNormThreads * V / 2]
  __shared__ float counts[kNormThreads];  // rows of each line of entries
  __syncthreads();
  const int d = s.group_channels;
  // Channels folded within a thread: all that its vector has of a group, where vectors do not
  // straddle groups.
  int q = d % V == 0 ? V : V % d == 0 ? d : 1;
  const int per = V / q, width = tile.cols * per;
  const int mine = t.active && t.lane < rows ? (rows - t.lane + t.lanes - 1) / t.lanes : 0;
  int lines = t.lanes, line = t.lane;
  bool write = t.active;
  float n = static_cast<float>(mine);
  if (tile.cols < 32 && 32 % tile.cols == 0) {
    // A tile's columns divide the warp: its rows are joined first.
    moments.move_pivot(threadIdx.x % tile.cols, n);
    for (int d = tile.cols; d < 32; d *= 2) {
      moments.add_lane(d);
      n += __shfl_xor_sync(0xFFFFFFFFu, n, d);
    }
    lines = kNormThreads / 32;
    line = threadIdx.x / 32;
    write = threadIdx.x % 32 < tile.cols;
  }
  if (write && t.col == 0) counts[line] = n;
  if (write) {
    const float inverse = n > 0.0f ? 1.0f / n : 0.0f;
    float2* to = entry + (line * tile.cols + t.col) * per;
    auto fold = [&](auto count) {
      constexpr int Q = decltype(count)::value;
#pragma unroll
      for (int j = 0; j < V / Q; ++j)
        to[j] = n > 0.0f ? fold_channels<Q>(moments, j * Q, n, inverse) : both(0.0f);
    };
    if (q == V) {
      fold(std::integral_constant<int, V>());
    } else if constexpr (V > 1) {
      if (q == 1) fold(std::integral_constant<int, 1>());
      if constexpr (V > 2) {
        if (q == 2) fold(std::integral_constant<int, 2>());
      }
      if constexpr (V > 4) {
        if (q == 4) fold(std::integral_constant<int, 4>());
      }
    }
  }
  __syncthreads();
  const int members = (s.pieces > 1 ? tile.cols * V : s.fold * d) / q;  // columns of a group
  const float weight = static_cast<float>(q);
  if (members == 1) {
    join_moments(
        width, lines,
        [&](int item, int i, float2& v) {
          v = entry[i * width + item];
          return weight * counts[i];
        },
        done);
    return;
  }
  const float2* from = entry;
  if (lines > 1) {
    join_moments(
        width, lines,
        [&](int item, int i, float2& v) {
          v = entry[i * width + item];
          return weight * counts[i];
        },
        [&](int item, float mean, float squares) { column[item] = make_float2(mean, squares); });
    __syncthreads();
    from = column;
  }
  const int span = s.fold > 1 ? d / q : members;  // neighbouring columns of a group
  join_moments(
      tile.groups, members,
      [&](int item, int i, float2& v) {
        const int f = s.fold > 1 ? i / span : 0;
        v = from[f * (s.channels / q) + item * span + i - f * span];
        return weight * static_cast<float>(rows);
      },
      done);
}

// First pass: the statistics of one chunk of rows in one tile of columns.
// parts [batch][groups][pieces][chunks].
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 4) norm_stats_kernel(const T* __restrict__ x,
                                                                     NormShape s, int view0,
                                                                     float2* __restrict__ parts) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormBlock b = norm_block(s, V, view0, blockIdx.x);
  const TileThread t(b.tile.cols);
  RowRing<T, V, 1, kStages> ring;
  ring.at[0] = x + b.first * s.x_row + (b.tile.col + t.col) * V;
  ring.stride[0] = s.x_row;
  ring.start(shared, t, b.rows);
  Moments<V> moments;
  bool first = true;
#pragma unroll
  for (int j = 0; j < Pairs<V>::kCount; ++j)
    moments.pivot.p[j] = moments.sum.p[j] = moments.square.p[j] = both(0.0f);
  ring.for_rows([&](const Pairs<V> (&v)[1]) {
    if (first) moments.start(v[0]);
    first = false;
    moments.add(v[0]);
  });
  join_block<V>(moments, t, s, b.tile, b.rows, shared, [&](int item, float mean, float squares) {
    const long long group = static_cast<long long>(b.view) * s.groups + b.tile.group + item;
    parts[(group * s.pieces + b.piece) * s.chunks + b.chunk] = make_float2(mean, squares);
  });
  wait_for_kernel_before();
}

// Sums over a block, for all of its threads.
__device__ __forceinline__ float block_sum(float v, float* shared) {
  v = lane_sum(v, 32);
  __syncthreads();
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < kNormThreads / 32; ++i) total += shared[i];
  return total;
}

// Joins the parts of one view and group: kJoin of them for each thread at a time, kept in registers
// between the sum that gives their mean and the sum of squares about it; then with those before.
constexpr int kJoin = 4;

template <int V>
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const float2* parts,
                                                                 NormShape s, int view0, float eps,
                                                                 float* __restrict__ mean,
                                                                 float* __restrict__ rstd) {
  __shared__ float shared[kNormThreads / 32];
  let_next_kernel_start();
  wait_for_kernel_before();
  const long long group = static_cast<long long>(view0) * s.groups + blockIdx.x;
  const int count = s.pieces * s.chunks;
  parts += group * count;
  const float2 pivot = parts[0];
  float all = 0.0f, all_mean = 0.0f, all_squares = 0.0f;
  for (int base = 0; base < count; base += kJoin * kNormThreads) {
    float2 v[kJoin];
    float n[kJoin];
    float total_n = 0.0f, total = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      const int i = base + k * kNormThreads + threadIdx.x;
      v[k] = pivot;
      n[k] = 0.0f;
      if (i < count) {
        v[k] = parts[i];
        const int piece = s.pieces > 1 ? i / s.chunks : 0, chunk = i - piece * s.chunks;
        const long long rows = min(static_cast<long long>(s.chunk_rows),
                                   s.rows - static_cast<long long>(chunk) * s.chunk_rows);
        const int width = s.pieces > 1
                              ? min(s.tile_cols, s.group_cols - piece * s.tile_cols) * V
                              : s.group_channels * s.fold;
        n[k] = static_cast<float>(rows) * static_cast<float>(width);
      }
    }
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      total_n += n[k];
      total = fmaf(n[k], v[k].x - pivot.x, total);
    }
    total_n = block_sum(total_n, shared);
    total = block_sum(total, shared);
    const float m = total / total_n;  // about the pivot
    float squares = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      const float d = v[k].x - pivot.x - m;
      squares += n[k] > 0.0f ? fmaf(n[k] * d, d, v[k].y) : 0.0f;
    }
    squares = block_sum(squares, shared);
    const float sum_n = all + total_n, d = m - all_mean;
    all_squares += squares + d * d * (all * (total_n / sum_n));
    all_mean += d * (total_n / sum_n);
    all = sum_n;
  }
  if (threadIdx.x == 0) {
    const float m = pivot.x + all_mean;
    const float values = static_cast<float>(s.pixels) * static_cast<float>(s.group_channels);
    mean[group] = m;
    rstd[group] = rsqrtf(variance_of(m, all_squares, values) + eps);
  }
}

// Second pass: normalise, scale, activate and drop one chunk of rows in one tile of columns. Blocks
// run from the end of the views to their start: what the first pass read last is still in L2.
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, 4) norm_apply_kernel(
    const T* __restrict__ x, NormShape s, int view0, NormParam weight, NormParam bias, float bound,
    DropKey key, const float* mean, const float* rstd, T* __restrict__ y) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormBlock b = norm_block(s, V, view0, gridDim.x - 1 - blockIdx.x);
  const TileThread t(b.tile.cols);
  const int col = (b.tile.col + t.col) * V;
  RowRing<T, V, 1, kStages> ring;
  ring.at[0] = x + b.first * s.x_row + col;
  ring.stride[0] = s.x_row;
  ring.start(shared, t, b.rows);
  wait_for_kernel_before();
  if (!t.active) return;
  Pairs<V> m, a, c;  // z = (x + m) a + c
  if (V == 1) m.p[0].y = a.p[0].y = c.p[0].y = 0.0f;
  ChannelWalk walk(s, col);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const long long group = static_cast<long long>(b.view) * s.groups + walk.group;
    m.set(j, -mean[group]);
    a.set(j, rstd[group] * load_scale(weight, b.view, walk.channel));
    c.set(j, load_shift(bias, b.view, walk.channel));
    walk.next();
  }
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  const long long out_row = static_cast<long long>(s.channels) * s.fold;
  long long at = (b.first + t.lane) * out_row + col;
  const long long step = t.lanes * out_row;
  ring.for_rows([&](const Pairs<V> (&v)[1]) {
    Pairs<V> z;
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j)
      z.p[j] = activate<Silu>(fma2(add2(v[0].p[j], m.p[j]), a.p[j], c.p[j]), bound);
    if (Drop) apply_dropout<V>(z, at, key, seed);
    __stcs(reinterpret_cast<Packed<T, V>*>(y + at), pack_pairs<T, V>(z));
    at += step;
  });
}

template <typename T, int V, bool Silu, bool Drop>
int passes(const void* x, const NormShape& s, int dtype, const NormParam& weight,
           const NormParam& bias, float eps, float bound, const DropKey& key, void* y, float* mean,
           float* rstd, float2* parts, cudaStream_t stream) {
  const T* in = static_cast<const T*>(x);
  T* out = static_cast<T*>(y);
  const int most = views_at_once(s, dtype, 1);
  constexpr size_t ring = RowRing<T, V, 1, kStages>::kBytes;
  constexpr size_t shared = std::max(ring, join_bytes<V>());
  for (int view0 = 0; view0 < s.batch; view0 += most) {
    const int views = static_cast<int>(std::min<long long>(most, s.batch - view0));
    const unsigned int blocks = static_cast<unsigned int>(views) * s.tiles * s.chunks;
    const unsigned int groups = static_cast<unsigned int>(views) * s.groups;
    cudaError_t err = launch_kernel(norm_stats_kernel<T, V>, blocks, kNormThreads, shared, stream,
                                    view0 > 0, in, s, view0, parts);
    if (err == cudaSuccess)
      err = launch_kernel(norm_join_kernel<V>, groups, kNormThreads, 0, stream, true, parts, s,
                          view0, eps, mean, rstd);
    if (err == cudaSuccess)
      err = launch_kernel(norm_apply_kernel<T, V, Silu, Drop>, blocks, kNormThreads, ring, stream,
                          true, in, s, view0, weight, bias, bound, key, mean, rstd, out);
    if (err != cudaSuccess) return static_cast<int>(err);
  }
  return launch_status();
}

}  // namespace
}  // namespace dr

using namespace dr;

extern "C" size_t dr_group_norm_workspace_bytes(int64_t batch, int64_t pixels, int32_t channels,
                                                int32_t groups, int32_t dtype, int32_t backward) {
  if (bad_norm_sizes(batch, pixels, channels, groups, dtype)) return 0;
  return norm_workspace_bytes(batch, pixels, channels, groups, dtype, backward != 0);
}

extern "C" int dr_group_norm_fwd(const void* x, int64_t x_stride, int32_t dtype, int64_t batch,
                                 int64_t pixels, int32_t channels, int32_t groups,
                                 const void* weight, int32_t weight_dtype, int64_t weight_batch,
                                 const void* bias, int32_t bias_dtype, int64_t bias_batch,
                                 float eps, int32_t activation, int32_t drop_threshold,
                                 const int64_t* seed, int64_t seed_value, int64_t layer, void* y,
                                 float* mean, float* rstd, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (bad_norm_sizes(batch, pixels, channels, groups, dtype) || x_stride < channels ||
      bad_norm_param(weight, weight_dtype, weight_batch, batch) ||
      bad_norm_param(bias, bias_dtype, bias_batch, batch) || activation < DR_ACTIVATION_NONE ||
      activation > DR_ACTIVATION_SILU || bad_drop(drop_threshold, layer))
    return DR_ERR_INVALID_ARGUMENT;
  if (batch == 0 || pixels == 0) return DR_OK;
  if (x == nullptr || y == nullptr || mean == nullptr || rstd == nullptr)
    return DR_ERR_INVALID_ARGUMENT;
  NormShape s;
  NormVector v = choose_vector(pixels, channels, dtype, x_stride, channels, {x, y});
  if (batch > kMaxNormBlocks ||
      !plan_passes(s, v, batch, pixels, channels, groups, dtype, x_stride, channels))
    return DR_ERR_TOO_LARGE;
  if (workspace == nullptr || workspace_bytes < norm_space(s, false).total)
    return DR_ERR_WORKSPACE_TOO_SMALL;
  const NormParam w{weight, weight_dtype, weight_batch > 1 ? channels : 0};
  const NormParam b{bias, bias_dtype, bias_batch > 1 ? channels : 0};
  const DropKey key = drop_key(seed, seed_value, layer, drop_threshold);
  const float bound = norm_bound(activation);
  return with_variant(dtype, v.vec, activation, drop_threshold, [&](auto k) {
    using K = decltype(k);
    return passes<typename K::Type, K::kVec, K::kSilu, K::kDrop>(
        x, s, dtype, w, b, eps, bound, key, y, mean, rstd, static_cast<float2*>(workspace),
        as_stream(stream));
  });
}
