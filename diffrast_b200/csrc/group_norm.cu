// Group normalisation with an activation and optional dropout: the forward pass (the formulas and
// the way views are cut up are in group_norm.cuh).
#include "group_norm.cuh"

namespace dr {
namespace {

constexpr int kUnroll = 4;  // vectors a thread has under way

// Reads the rows first, first + step, ... below `end` of a column of vectors, kUnroll of them at a
// time, and gives each to `use(vector, row)`.
template <typename T, int V, typename Use>
__device__ __forceinline__ void for_rows(const T* __restrict__ x, long long stride, int first,
                                         int step, int end, Use use) {
  using P = Packed<T, V>;
  for (int row = first; row < end; row += kUnroll * step) {
    P p[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (row + u * step < end)
        p[u] = *reinterpret_cast<const P*>(x + (row + u * step) * stride);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (row + u * step < end) use(p[u], row + u * step);
  }
}

// Statistics of one chunk of rows in one tile of columns: per-thread moments per channel, joined
// over the block's rows, then over the channels (and folded pixels) of each group.
// parts [batch][groups][chunks * group_tiles] of (mean, squared deviations).
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(const T* __restrict__ x,
                                                                  NormShape s,
                                                                  float2* __restrict__ parts) {
  __shared__ float2 entry[kNormThreads * V];
  __shared__ float2 channel[kNormThreads * V];
  long long block = blockIdx.x;
  const int chunk = static_cast<int>(block % s.chunks);
  block /= s.chunks;
  const int tile_index = static_cast<int>(block % s.tiles);
  const long long view = block / s.tiles;
  const NormTile tile = norm_tile(s, V, tile_index);
  const int lanes = kNormThreads / tile.cols;
  const int col = threadIdx.x % tile.cols, lane = threadIdx.x / tile.cols;
  const long long row0 = chunk * s.chunk_rows;
  const int rows = static_cast<int>(min(s.chunk_rows, s.rows - row0));
  const int width = tile.cols * V;
  if (lane < lanes) {
    Moments<V> moments;
    const T* base = x + (view * s.rows + row0) * s.x_row + (tile.col + col) * V;
    for_rows<T, V>(base, s.x_row, lane, lanes, rows, [&](const Packed<T, V>& p, int) {
      float v[V];
      unpack<T, V>(p, v);
      moments.add(v);
    });
#pragma unroll
    for (int j = 0; j < V; ++j) entry[lane * width + col * V + j] = moments.get(j);
  }
  __syncthreads();
  join_moments(
      width, lanes, kNormThreads,
      [&](int item, int i, float2& v) {
        v = entry[i * width + item];
        return static_cast<float>((rows - i + lanes - 1) / lanes);
      },
      [&](int item, float mean, float squares) { channel[item] = make_float2(mean, squares); });
  __syncthreads();
  const int d = s.group_tiles > 1 ? width : s.group_channels;
  const int part_count = s.chunks * s.group_tiles;
  join_moments(
      tile.groups, s.fold * d, kNormThreads,
      [&](int item, int i, float2& v) {
        const int f = i / d;
        v = channel[f * s.channels + item * d + i - f * d];
        return static_cast<float>(rows);
      },
      [&](int item, float mean, float squares) {
        const long long at = (view * s.groups + tile.group + item) * part_count;
        const int piece = s.group_tiles > 1 ? tile_index % s.group_tiles : 0;
        parts[at + chunk * s.group_tiles + piece] = make_float2(mean, squares);
      });
}

// Joins the chunks' statistics: one warp for each view and group.
template <int V>
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const float2* __restrict__ parts,
                                                                 NormShape s, float eps,
                                                                 float* __restrict__ mean,
                                                                 float* __restrict__ rstd) {
  constexpr int kWarps = kNormThreads / 32;
  const long long first = blockIdx.x * static_cast<long long>(kWarps);
  const long long total = s.batch * s.groups;
  const int part_count = s.chunks * s.group_tiles;
  join_moments(
      static_cast<int>(min(static_cast<long long>(kWarps), total - first)), part_count, kNormThreads,
      [&](int item, int i, float2& v) {
        v = parts[(first + item) * part_count + i];
        const int chunk = i / s.group_tiles, piece = i - chunk * s.group_tiles;
        const int rows = static_cast<int>(min(s.chunk_rows, s.rows - chunk * s.chunk_rows));
        const int width = s.group_tiles > 1 ? min(s.tile_cols, s.group_cols - piece * s.tile_cols) * V
                                            : s.group_channels * s.fold;
        return static_cast<float>(rows) * static_cast<float>(width);
      },
      [&](int item, float m, float squares) {
        const float count = static_cast<float>(s.pixels) * static_cast<float>(s.group_channels);
        mean[first + item] = m;
        rstd[first + item] = rsqrtf(variance_of(m, squares, count) + eps);
      });
}

// Normalise, scale, activate and drop: one chunk of rows in one tile of columns.
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(
    const T* __restrict__ x, NormShape s, NormParam weight, NormParam bias, float bound,
    DropKey key, const float* __restrict__ mean, const float* __restrict__ rstd,
    T* __restrict__ y) {
  long long block = blockIdx.x;
  const int chunk = static_cast<int>(block % s.chunks);
  block /= s.chunks;
  const NormTile tile = norm_tile(s, V, static_cast<int>(block % s.tiles));
  const long long view = block / s.tiles;
  const int lanes = kNormThreads / tile.cols;
  const int col = threadIdx.x % tile.cols, lane = threadIdx.x / tile.cols;
  if (lane >= lanes) return;
  const long long row0 = chunk * s.chunk_rows;
  const int rows = static_cast<int>(min(s.chunk_rows, s.rows - row0));
  float m[V], a[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = ((tile.col + col) * V + j) % s.channels;
    const long long group = view * s.groups + c / s.group_channels;
    const float w = weight.data ? load_param(weight.data, weight.dtype, view * weight.view + c) : 1.0f;
    m[j] = mean[group];
    a[j] = rstd[group] * w;
    b[j] = bias.data ? load_param(bias.data, bias.dtype, view * bias.view + c) : 0.0f;
  }
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  const long long out_row = static_cast<long long>(s.channels) * s.fold;
  const long long offset = (view * s.rows + row0) * out_row + (tile.col + col) * V;
  const T* base = x + (view * s.rows + row0) * s.x_row + (tile.col + col) * V;
  for_rows<T, V>(base, s.x_row, lane, lanes, rows, [&](const Packed<T, V>& p, int row) {
    float v[V];
    unpack<T, V>(p, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = activate<Silu>(fmaf(v[j] - m[j], a[j], b[j]), bound);
    const long long at = offset + row * out_row;
    if (Drop) apply_dropout<V>(v, at, key, seed);
    *reinterpret_cast<Packed<T, V>*>(y + at) = pack<T, V>(v);
  });
}

template <typename T, int V>
int run(const void* x, const NormShape& s, const NormParam& weight, const NormParam& bias,
        float eps, int activation, const DropKey& key, void* y, float* mean, float* rstd,
        float2* parts, cudaStream_t stream) {
  const T* in = static_cast<const T*>(x);
  T* out = static_cast<T*>(y);
  const unsigned int blocks = static_cast<unsigned int>(s.batch * s.tiles * s.chunks);
  norm_stats_kernel<T, V><<<blocks, kNormThreads, 0, stream>>>(in, s, parts);
  norm_join_kernel<V><<<blocks_for(s.batch * s.groups, kNormThreads / 32), kNormThreads, 0,
                        stream>>>(parts, s, eps, mean, rstd);
  const float bound = norm_bound(activation);
  auto launch = [&](auto kernel) {
    kernel<<<blocks, kNormThreads, 0, stream>>>(in, s, weight, bias, bound, key, mean, rstd, out);
  };
  const bool drop = key.threshold != 0;
  if (activation == DR_ACTIVATION_SILU)
    drop ? launch(norm_apply_kernel<T, V, true, true>) : launch(norm_apply_kernel<T, V, true, false>);
  else
    drop ? launch(norm_apply_kernel<T, V, false, true>)
         : launch(norm_apply_kernel<T, V, false, false>);
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
  if (!cut_norm(s, v, batch, pixels, channels, groups, dtype, x_stride, channels,
                norm_chunk_bytes(batch, pixels, channels, dtype)))
    return DR_ERR_TOO_LARGE;
  if (workspace == nullptr || workspace_bytes < norm_forward_bytes(s))
    return DR_ERR_WORKSPACE_TOO_SMALL;
  const NormParam w{weight, weight_dtype, weight_batch > 1 ? channels : 0};
  const NormParam b{bias, bias_dtype, bias_batch > 1 ? channels : 0};
  const DropKey key = drop_key(seed, seed_value, layer, drop_threshold);
  auto* parts = static_cast<float2*>(workspace);
  return with_vector(dtype, v.vec, [&](auto type, auto width) {
    return run<typename decltype(type)::type, decltype(width)::value>(
        x, s, w, b, eps, activation, key, y, mean, rstd, parts, as_stream(stream));
  });
}
