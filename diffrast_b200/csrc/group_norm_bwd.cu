// Group normalisation with an activation and optional dropout: the backward pass (the formulas and
// the way views are cut up are in group_norm.cuh). Nothing of the forward pass is kept but the
// image, the means and the reciprocal standard deviations: z, its derivative and the dropout's
// mask are computed again.
#include "group_norm.cuh"

namespace dr {
namespace {

constexpr int kUnroll = 2;  // vectors of x, and as many of the gradient, a thread has under way

// Constants of a thread's channels.
template <int V>
struct Channels {
  float mean[V], rstd[V], weight[V], bias[V];

  __device__ __forceinline__ void load(const NormShape& s, long long view, int first,
                                       const NormParam& w, const NormParam& b,
                                       const float* means, const float* rstds) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (first + j) % s.channels;
      const long long group = view * s.groups + c / s.group_channels;
      mean[j] = __ldg(means + group);
      rstd[j] = __ldg(rstds + group);
      weight[j] = w.data ? load_param(w.data, w.dtype, view * w.view + c) : 1.0f;
      bias[j] = b.data ? load_param(b.data, b.dtype, view * b.view + c) : 0.0f;
    }
  }
};

// Runs use(vector of x, vector of the gradient, row) over the rows first, first + step, ... < end.
template <typename T, int V, typename Use>
__device__ __forceinline__ void for_rows(const T* __restrict__ x, long long x_row,
                                         const T* __restrict__ grad, long long grad_row, int first,
                                         int step, int end, Use use) {
  using P = Packed<T, V>;
  for (int row = first; row < end; row += kUnroll * step) {
    P p[kUnroll], g[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (row + u * step < end) {
        p[u] = *reinterpret_cast<const P*>(x + (row + u * step) * x_row);
        g[u] = *reinterpret_cast<const P*>(grad + (row + u * step) * grad_row);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (row + u * step < end) use(p[u], g[u], row + u * step);
  }
}

// Sums of q and q (x - m) of each channel over one chunk of rows in one tile of columns.
// parts [batch][chunks][channels].
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads) norm_sums_kernel(
    const T* __restrict__ x, const T* __restrict__ grad, NormShape s, NormParam weight,
    NormParam bias, float bound, DropKey key, const float* __restrict__ mean,
    const float* __restrict__ rstd, float2* __restrict__ parts) {
  __shared__ float2 entry[kNormThreads * V];
  long long block = blockIdx.x;
  const int chunk = static_cast<int>(block % s.chunks);
  block /= s.chunks;
  const NormTile tile = norm_tile(s, V, static_cast<int>(block % s.tiles));
  const long long view = block / s.tiles;
  const int lanes = kNormThreads / tile.cols;
  const int col = threadIdx.x % tile.cols, lane = threadIdx.x / tile.cols;
  const long long row0 = chunk * s.chunk_rows;
  const int rows = static_cast<int>(min(s.chunk_rows, s.rows - row0));
  const int width = tile.cols * V;
  if (lane < lanes) {
    Channels<V> c;
    c.load(s, view, (tile.col + col) * V, weight, bias, mean, rstd);
    const unsigned long long seed = Drop ? load_seed(key) : 0;
    const long long out_row = static_cast<long long>(s.channels) * s.fold;
    const long long offset = (view * s.rows + row0) * out_row + (tile.col + col) * V;
    float sum[V], dot[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f, dot[j] = 0.0f;
    for_rows<T, V>(x + (view * s.rows + row0) * s.x_row + (tile.col + col) * V, s.x_row,
                   grad + (view * s.rows + row0) * s.grad_row + (tile.col + col) * V, s.grad_row,
                   lane, lanes, rows, [&](const Packed<T, V>& p, const Packed<T, V>& g, int row) {
      float v[V], q[V];
      unpack<T, V>(p, v);
      unpack<T, V>(g, q);
      if (Drop) apply_dropout<V>(q, offset + row * out_row, key, seed);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[j] - c.mean[j];
        const float z = fmaf(d, c.rstd[j] * c.weight[j], c.bias[j]);
        const float t = q[j] * activate_grad<Silu>(z, bound);
        sum[j] += t;
        dot[j] = fmaf(t, d, dot[j]);
      }
    });
#pragma unroll
    for (int j = 0; j < V; ++j)
      entry[lane * width + col * V + j] = make_float2(sum[j], dot[j]);
  }
  __syncthreads();
  const int items = s.fold > 1 ? s.channels : width;
  const int first = s.fold > 1 ? 0 : tile.col * V;
  join_sums(
      items, lanes * s.fold, kNormThreads,
      [&](int item, int i) { return entry[i * items + item]; },
      [&](int item, float2 total) {
        parts[(view * s.chunks + chunk) * s.channels + first + item] = total;
      });
}

// Per view: the channels' sums over the chunks, then the groups' two means. One block for each
// view and each run of groups (`run_groups` of them).
__global__ void __launch_bounds__(kNormThreads) norm_means_kernel(
    const float2* __restrict__ parts, NormShape s, NormParam weight, int runs, int run_groups,
    const float* __restrict__ rstd, float2* __restrict__ sums, float2* __restrict__ means) {
  const long long view = blockIdx.x / runs;
  const int group0 = static_cast<int>(blockIdx.x % runs) * run_groups;
  const int groups = min(run_groups, s.groups - group0);
  const int d = s.group_channels, first = group0 * d;
  join_sums(
      groups * d, s.chunks, kNormThreads,
      [&](int item, int i) { return parts[(view * s.chunks + i) * s.channels + first + item]; },
      [&](int item, float2 total) {
        total.y *= rstd[view * s.groups + (first + item) / d];
        sums[view * s.channels + first + item] = total;
      });
  __syncthreads();
  const float count = static_cast<float>(s.pixels) * static_cast<float>(d);
  join_sums(
      groups, d, kNormThreads,
      [&](int item, int i) {
        const int c = first + item * d + i;
        const float w =
            weight.data ? load_param(weight.data, weight.dtype, view * weight.view + c) : 1.0f;
        const float2 v = sums[view * s.channels + c];
        return make_float2(v.x * w, v.y * w);
      },
      [&](int item, float2 total) {
        means[view * s.groups + group0 + item] = make_float2(total.x / count, total.y / count);
      });
}

// grad x = r (q w - A - h B) over one chunk of rows in one tile of columns.
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads) norm_grad_kernel(
    const T* __restrict__ x, const T* __restrict__ grad, NormShape s, NormParam weight,
    NormParam bias, float bound, DropKey key, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float2* __restrict__ means, T* __restrict__ grad_x) {
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
  Channels<V> c;
  c.load(s, view, (tile.col + col) * V, weight, bias, mean, rstd);
  float shift[V], slope[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int channel = ((tile.col + col) * V + j) % s.channels;
    const float2 m = __ldg(means + view * s.groups + channel / s.group_channels);
    shift[j] = -c.rstd[j] * m.x;
    slope[j] = -c.rstd[j] * c.rstd[j] * m.y;
  }
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  const long long out_row = static_cast<long long>(s.channels) * s.fold;
  const long long offset = (view * s.rows + row0) * out_row + (tile.col + col) * V;
  for_rows<T, V>(x + (view * s.rows + row0) * s.x_row + (tile.col + col) * V, s.x_row,
                 grad + (view * s.rows + row0) * s.grad_row + (tile.col + col) * V, s.grad_row,
                 lane, lanes, rows, [&](const Packed<T, V>& p, const Packed<T, V>& g, int row) {
    float v[V], q[V];
    unpack<T, V>(p, v);
    unpack<T, V>(g, q);
    const long long at = offset + row * out_row;
    if (Drop) apply_dropout<V>(q, at, key, seed);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = v[j] - c.mean[j];
      const float a = c.rstd[j] * c.weight[j];
      const float t = q[j] * activate_grad<Silu>(fmaf(d, a, c.bias[j]), bound);
      v[j] = fmaf(t, a, fmaf(d, slope[j], shift[j]));
    }
    *reinterpret_cast<Packed<T, V>*>(grad_x + at) = pack<T, V>(v);
  });
}

// Gradients of weight and bias: sums over the views (or each view's own), 32 channels a block.
__global__ void __launch_bounds__(kNormThreads) norm_params_kernel(
    const float2* __restrict__ sums, long long batch, int channels, void* grad_weight,
    int weight_dtype, bool weight_views, void* grad_bias, int bias_dtype, bool bias_views) {
  constexpr int kLanes = kNormThreads / 32;
  __shared__ float2 entry[kLanes][32];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
  float2 total = make_float2(0.0f, 0.0f);
  if (c < channels) {
    for (long long n = lane; n < batch; n += kLanes) {
      const float2 v = sums[n * channels + c];
      if (grad_weight != nullptr && weight_views)
        store_param(grad_weight, weight_dtype, n * channels + c, v.y);
      if (grad_bias != nullptr && bias_views)
        store_param(grad_bias, bias_dtype, n * channels + c, v.x);
      total.x += v.x;
      total.y += v.y;
    }
  }
  entry[lane][threadIdx.x % 32] = total;
  __syncthreads();
  if (lane != 0 || c >= channels) return;
  for (int i = 1; i < kLanes; ++i) {
    total.x += entry[i][threadIdx.x].x;
    total.y += entry[i][threadIdx.x].y;
  }
  if (grad_weight != nullptr && !weight_views) store_param(grad_weight, weight_dtype, c, total.y);
  if (grad_bias != nullptr && !bias_views) store_param(grad_bias, bias_dtype, c, total.x);
}

template <typename T, int V>
int run(const void* x, const void* grad, const NormShape& s, const NormParam& weight,
        const NormParam& bias, int activation, const DropKey& key, const float* mean,
        const float* rstd, void* grad_x, void* grad_weight, bool weight_views, void* grad_bias,
        bool bias_views, unsigned char* workspace, cudaStream_t stream) {
  const size_t views = static_cast<size_t>(s.batch) * s.channels * sizeof(float2);
  auto* parts = reinterpret_cast<float2*>(workspace);
  auto* sums = reinterpret_cast<float2*>(workspace + align256(views * s.chunks));
  auto* means = reinterpret_cast<float2*>(workspace + align256(views * s.chunks) + align256(views));
  const T* in = static_cast<const T*>(x);
  const T* dy = static_cast<const T*>(grad);
  const unsigned int blocks = static_cast<unsigned int>(s.batch * s.tiles * s.chunks);
  const float bound = norm_bound(activation);
  const bool drop = key.threshold != 0, silu = activation == DR_ACTIVATION_SILU;
  auto add = [&](auto kernel) {
    kernel<<<blocks, kNormThreads, 0, stream>>>(in, dy, s, weight, bias, bound, key, mean, rstd,
                                                parts);
  };
  if (silu)
    drop ? add(norm_sums_kernel<T, V, true, true>) : add(norm_sums_kernel<T, V, true, false>);
  else
    drop ? add(norm_sums_kernel<T, V, false, true>) : add(norm_sums_kernel<T, V, false, false>);
  const int run_groups = std::max(1, std::min(s.groups, 32 / s.group_channels));
  const int runs = (s.groups + run_groups - 1) / run_groups;
  norm_means_kernel<<<static_cast<unsigned int>(s.batch * runs), kNormThreads, 0, stream>>>(
      parts, s, weight, runs, run_groups, rstd, sums, means);
  if (grad_x != nullptr) {
    auto apply = [&](auto kernel) {
      kernel<<<blocks, kNormThreads, 0, stream>>>(in, dy, s, weight, bias, bound, key, mean, rstd,
                                                  means, static_cast<T*>(grad_x));
    };
    if (silu)
      drop ? apply(norm_grad_kernel<T, V, true, true>) : apply(norm_grad_kernel<T, V, true, false>);
    else
      drop ? apply(norm_grad_kernel<T, V, false, true>)
           : apply(norm_grad_kernel<T, V, false, false>);
  }
  if (grad_weight != nullptr || grad_bias != nullptr)
    norm_params_kernel<<<blocks_for(s.channels, 32), kNormThreads, 0, stream>>>(
        sums, s.batch, s.channels, grad_weight, weight.dtype, weight_views, grad_bias, bias.dtype,
        bias_views);
  return launch_status();
}

}  // namespace
}  // namespace dr

using namespace dr;

extern "C" int dr_group_norm_bwd(const void* x, int64_t x_stride, const void* grad_y,
                                 int64_t grad_stride, int32_t dtype, int64_t batch, int64_t pixels,
                                 int32_t channels, int32_t groups, const void* weight,
                                 int32_t weight_dtype, int64_t weight_batch, const void* bias,
                                 int32_t bias_dtype, int64_t bias_batch, const float* mean,
                                 const float* rstd, int32_t activation, int32_t drop_threshold,
                                 const int64_t* seed, int64_t seed_value, int64_t layer,
                                 void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (bad_norm_sizes(batch, pixels, channels, groups, dtype) || x_stride < channels ||
      grad_stride < channels || bad_norm_param(weight, weight_dtype, weight_batch, batch) ||
      bad_norm_param(bias, bias_dtype, bias_batch, batch) || activation < DR_ACTIVATION_NONE ||
      activation > DR_ACTIVATION_SILU || bad_drop(drop_threshold, layer) ||
      (grad_weight != nullptr && weight == nullptr) || (grad_bias != nullptr && bias == nullptr))
    return DR_ERR_INVALID_ARGUMENT;
  if (batch == 0 || pixels == 0) return DR_OK;
  if (x == nullptr || grad_y == nullptr || mean == nullptr || rstd == nullptr)
    return DR_ERR_INVALID_ARGUMENT;
  NormShape s;
  NormVector v = choose_vector(pixels, channels, dtype, x_stride, grad_stride,
                               {x, grad_y, grad_x});
  if (!cut_norm(s, v, batch, pixels, channels, groups, dtype, x_stride, grad_stride,
                norm_chunk_bytes(batch, pixels, channels, dtype)))
    return DR_ERR_TOO_LARGE;
  if (workspace == nullptr || workspace_bytes < norm_backward_bytes(s))
    return DR_ERR_WORKSPACE_TOO_SMALL;
  const NormParam w{weight, weight_dtype, weight_batch > 1 ? channels : 0};
  const NormParam b{bias, bias_dtype, bias_batch > 1 ? channels : 0};
  const DropKey key = drop_key(seed, seed_value, layer, drop_threshold);
  return with_vector(dtype, v.vec, [&](auto type, auto width) {
    return run<typename decltype(type)::type, decltype(width)::value>(
        x, grad_y, s, w, b, activation, key, mean, rstd, grad_x, grad_weight, weight_batch > 1,
        grad_bias, bias_batch > 1, static_cast<unsigned char*>(workspace), as_stream(stream));
  });
}
