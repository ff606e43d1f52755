// Group normalisation with an activation and optional dropout: the backward pass (the formulas and
// the way views are cut up are in group_norm.cuh). Nothing of the forward pass is kept but the
// image, the means and the reciprocal standard deviations: z, its derivative and the dropout's
// mask are computed again.
#include "group_norm.cuh"

namespace dr {
namespace {

constexpr int kStages = 4;  // rows of x and of the gradient that a thread has under way

// Constants of a thread's channels: z = (x + shift) scale + bias.
template <int V>
struct Channels {
  Pairs<V> shift, scale, bias;

  __device__ __forceinline__ void load(const NormShape& s, long long view, int first,
                                       const NormParam& w, const NormParam& b,
                                       const float* means, const float* rstds) {
    if (V == 1) shift.p[0].y = scale.p[0].y = bias.p[0].y = 0.0f;
    ChannelWalk c(s, first);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const long long group = view * s.groups + c.group;
      shift.set(j, -__ldg(means + group));
      scale.set(j, __ldg(rstds + group) * load_scale(w, view, c.channel));
      bias.set(j, load_shift(b, view, c.channel));
      c.next();
    }
  }
};

// Joins the threads' sums of a block's rows: over the rows of a warp where a tile's columns divide
// it, then over the rows (and folded pixels) that are left. `done` gets the channel within the
// tile.
template <int V, typename Done>
__device__ __forceinline__ void join_block(Pairs<V>& sum, Pairs<V>& dot, const TileThread& t,
                                           const NormShape& s, const NormTile& tile, void* shared,
                                           Done done) {
  auto* entry = static_cast<float2*>(shared);  // [kNormThreads * V]
  __syncthreads();
  const int width = tile.cols * V;
  int rows = t.lanes, row = t.lane;
  bool write = t.active;
  if (tile.cols < 32 && 32 % tile.cols == 0) {
    for (int d = tile.cols; d < 32; d *= 2) {
#pragma unroll
      for (int j = 0; j < Pairs<V>::kCount; ++j) {
        sum.p[j].x += __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].x, d);
        dot.p[j].x += __shfl_xor_sync(0xFFFFFFFFu, dot.p[j].x, d);
        if (V > 1) {
          sum.p[j].y += __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].y, d);
          dot.p[j].y += __shfl_xor_sync(0xFFFFFFFFu, dot.p[j].y, d);
        }
      }
    }
    rows = kNormThreads / 32;
    row = threadIdx.x / 32;
    write = threadIdx.x % 32 < tile.cols;
  }
  if (write) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      entry[row * width + t.col * V + j] = make_float2(sum.get(j), dot.get(j));
  }
  __syncthreads();
  const int items = s.fold > 1 ? s.channels : width;
  join_sums(items, rows * s.fold, [&](int item, int i) { return entry[i * items + item]; }, done);
}

// First pass: sums of q and q (x - m) of each channel over one chunk of rows in one tile of columns.
// parts [batch][chunks][channels].
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, 3) norm_sums_kernel(
    const T* __restrict__ x, const T* __restrict__ grad, NormShape s, int view0, NormParam weight,
    NormParam bias, float bound, DropKey key, const float* __restrict__ mean,
    const float* __restrict__ rstd, float2* __restrict__ parts) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormBlock b = norm_block(s, V, view0, blockIdx.x);
  const TileThread t(b.tile.cols);
  const int col = (b.tile.col + t.col) * V;
  RowRing<T, V, 2, kStages> ring;
  ring.at[0] = x + b.first * s.x_row + col;
  ring.at[1] = grad + b.first * s.grad_row + col;
  ring.stride[0] = s.x_row;
  ring.stride[1] = s.grad_row;
  ring.start(shared, t, b.rows);
  Pairs<V> sum, dot;
#pragma unroll
  for (int j = 0; j < Pairs<V>::kCount; ++j) sum.p[j] = dot.p[j] = both(0.0f);
  if (t.active) {
    Channels<V> c;
    c.load(s, b.view, col, weight, bias, mean, rstd);
    const unsigned long long seed = Drop ? load_seed(key) : 0;
    const long long out_row = static_cast<long long>(s.channels) * s.fold;
    long long at = (b.first + t.lane) * out_row + col;
    const long long step = t.lanes * out_row;
    ring.for_rows([&](Pairs<V> (&v)[2]) {
      if (Drop) apply_dropout<V>(v[1], at, key, seed);
      at += step;
#pragma unroll
      for (int j = 0; j < Pairs<V>::kCount; ++j) {
        const float2 d = add2(v[0].p[j], c.shift.p[j]);
        const float2 z = fma2(d, c.scale.p[j], c.bias.p[j]);
        const float2 u = activate_grad<Silu>(v[1].p[j], z, bound);
        sum.p[j] = add2(sum.p[j], u);
        dot.p[j] = fma2(u, d, dot.p[j]);
      }
    });
  }
  const int first = s.fold > 1 ? 0 : b.tile.col * V;
  join_block<V>(sum, dot, t, s, b.tile, shared, [&](int item, float2 total) {
    parts[(static_cast<long long>(b.view) * s.chunks + b.chunk) * s.channels + first + item] = total;
  });
  wait_for_kernel_before();
}

// Joins the parts of a view's channels, 32 of them at a time by 32 lanes each, and forms the two
// means of their groups. A block has a run of whole groups of at most 32 channels, or one group.
constexpr int kMeansThreads = 1024;

__global__ void __launch_bounds__(kMeansThreads) norm_means_kernel(
    const float2* parts, NormShape s, int view0, NormParam weight, int runs,
    int run_groups, const float* __restrict__ rstd, float2* __restrict__ sums,
    float2* __restrict__ means) {
  __shared__ float2 entry[32][33];
  __shared__ float2 scaled[32];
  let_next_kernel_start();
  wait_for_kernel_before();
  const long long view = view0 + blockIdx.x / runs;
  const int d = s.group_channels;
  const int group0 = static_cast<int>(blockIdx.x % runs) * run_groups;
  const int channel0 = group0 * d;
  const int channels = min(run_groups, s.groups - group0) * d;
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const float inverse = 1.0f / (static_cast<float>(s.pixels) * static_cast<float>(d));
  float2 group = make_float2(0.0f, 0.0f);  // of a group wider than 32 channels
  for (int base = 0; base < channels; base += 32) {
    const int c = channel0 + base + x;
    float2 total = make_float2(0.0f, 0.0f);
    if (base + x < channels) {
      const float2* from = parts + view * s.chunks * s.channels + c;
#pragma unroll 8
      for (int i = y; i < s.chunks; i += 32) {
        const float2 v = from[static_cast<long long>(i) * s.channels];
        total.x += v.x;
        total.y += v.y;
      }
    }
    entry[y][x] = total;
    __syncthreads();
    // Channel y of the 32 is summed by warp y.
    total = entry[x][y];
    total.x = lane_sum(total.x, 32);
    total.y = lane_sum(total.y, 32);
    if (x == 0) {
      const int channel = channel0 + base + y;
      float2 w = make_float2(0.0f, 0.0f);
      if (base + y < channels) {
        total.y *= rstd[view * s.groups + channel / d];
        sums[view * s.channels + channel] = total;
        const float scale = load_scale(weight, view, channel);
        w = make_float2(total.x * scale, total.y * scale);
      }
      scaled[y] = w;
    }
    __syncthreads();
    if (d > 32) {
      if (y == 0) {
        group.x += lane_sum(scaled[x].x, 32);
        group.y += lane_sum(scaled[x].y, 32);
      }
    } else if (threadIdx.x < channels / d) {
      for (int i = 0; i < d; ++i) {
        group.x += scaled[threadIdx.x * d + i].x;
        group.y += scaled[threadIdx.x * d + i].y;
      }
    }
  }
  if (threadIdx.x < (d > 32 ? 1 : channels / d))
    means[view * s.groups + group0 + threadIdx.x] =
        make_float2(group.x * inverse, group.y * inverse);
}

// Second pass: grad x = r (q w - A - h B) over one chunk of rows in one tile of columns, from the
// end of the views to their start (what the first pass read last is still in L2).
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, 3) norm_grad_kernel(
    const T* __restrict__ x, const T* __restrict__ grad, NormShape s, int view0, NormParam weight,
    NormParam bias, float bound, DropKey key, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float2* means, T* __restrict__ grad_x) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormBlock b = norm_block(s, V, view0, gridDim.x - 1 - blockIdx.x);
  const TileThread t(b.tile.cols);
  const int col = (b.tile.col + t.col) * V;
  RowRing<T, V, 2, kStages> ring;
  ring.at[0] = x + b.first * s.x_row + col;
  ring.at[1] = grad + b.first * s.grad_row + col;
  ring.stride[0] = s.x_row;
  ring.stride[1] = s.grad_row;
  ring.start(shared, t, b.rows);
  Channels<V> c;
  if (t.active) c.load(s, b.view, col, weight, bias, mean, rstd);
  wait_for_kernel_before();
  if (!t.active) return;
  Pairs<V> base, slope;  // grad x = u scale + d slope + base
  if (V == 1) base.p[0].y = slope.p[0].y = 0.0f;
  ChannelWalk walk(s, col);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const long long group = static_cast<long long>(b.view) * s.groups + walk.group;
    const float r = __ldg(rstd + group);
    const float2 m = means[group];
    base.set(j, -r * m.x);
    slope.set(j, -r * r * m.y);
    walk.next();
  }
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  const long long out_row = static_cast<long long>(s.channels) * s.fold;
  long long at = (b.first + t.lane) * out_row + col;
  const long long step = t.lanes * out_row;
  ring.for_rows([&](Pairs<V> (&v)[2]) {
    if (Drop) apply_dropout<V>(v[1], at, key, seed);
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j) {
      const float2 d = add2(v[0].p[j], c.shift.p[j]);
      const float2 z = fma2(d, c.scale.p[j], c.bias.p[j]);
      const float2 u = activate_grad<Silu>(v[1].p[j], z, bound);
      v[0].p[j] = fma2(u, c.scale.p[j], fma2(d, slope.p[j], base.p[j]));
    }
    __stcs(reinterpret_cast<Packed<T, V>*>(grad_x + at), pack_pairs<T, V>(v[0]));
    at += step;
  });
}

// Gradients of weight and bias: sums over the views (or each view's own), 32 channels a block.
__global__ void __launch_bounds__(kNormThreads) norm_params_kernel(
    const float2* sums, long long batch, int channels, void* grad_weight,
    int weight_dtype, bool weight_views, void* grad_bias, int bias_dtype, bool bias_views) {
  constexpr int kLanes = kNormThreads / 32;
  __shared__ float2 entry[kLanes][32];
  let_next_kernel_start();
  wait_for_kernel_before();
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

struct Gradients {
  void *x, *weight, *bias;
  int weight_dtype, bias_dtype;
  bool weight_views, bias_views;
};

template <typename T, int V, bool Silu, bool Drop>
int passes(const void* x, const void* grad, const NormShape& s, int dtype, const NormParam& weight,
           const NormParam& bias, float bound, const DropKey& key, const float* mean,
           const float* rstd, const Gradients& out, unsigned char* workspace,
           cudaStream_t stream) {
  const NormSpace space = norm_space(s, true);
  auto* parts = reinterpret_cast<float2*>(workspace + space.parts);
  auto* sums = reinterpret_cast<float2*>(workspace + space.sums);
  auto* means = reinterpret_cast<float2*>(workspace + space.means);
  const T* in = static_cast<const T*>(x);
  const T* dy = static_cast<const T*>(grad);
  const int run_groups = std::max(1, std::min(s.groups, 32 / s.group_channels));
  const int runs = (s.groups + run_groups - 1) / run_groups;
  const int most = views_at_once(s, dtype, 2);
  constexpr size_t ring = RowRing<T, V, 2, kStages>::kBytes;
  constexpr size_t shared = std::max(ring, sizeof(float2) * kNormThreads * V);
  cudaError_t err = cudaSuccess;
  for (int view0 = 0; view0 < s.batch; view0 += most) {
    const int views = static_cast<int>(std::min<long long>(most, s.batch - view0));
    const unsigned int blocks = static_cast<unsigned int>(views) * s.tiles * s.chunks;
    err = launch_kernel(norm_sums_kernel<T, V, Silu, Drop>, blocks, kNormThreads, shared, stream,
                        view0 > 0, in, dy, s, view0, weight, bias, bound, key, mean, rstd, parts);
    if (err == cudaSuccess)
      err = launch_kernel(norm_means_kernel, static_cast<unsigned int>(views) * runs,
                          kMeansThreads, 0, stream, true, parts, s, view0, weight, runs, run_groups,
                          rstd, sums, means);
    if (err == cudaSuccess && out.x != nullptr)
      err = launch_kernel(norm_grad_kernel<T, V, Silu, Drop>, blocks, kNormThreads, ring, stream, true,
                          in, dy, s, view0, weight, bias, bound, key, mean, rstd, means,
                          static_cast<T*>(out.x));
    if (err != cudaSuccess) return static_cast<int>(err);
  }
  if (out.weight != nullptr || out.bias != nullptr)
    err = launch_kernel(norm_params_kernel, blocks_for(s.channels, 32), kNormThreads, 0, stream, true,
                        sums, s.batch, s.channels, out.weight, out.weight_dtype, out.weight_views,
                        out.bias, out.bias_dtype, out.bias_views);
  return err == cudaSuccess ? launch_status() : static_cast<int>(err);
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
  if (batch > kMaxNormBlocks ||
      !plan_passes(s, v, batch, pixels, channels, groups, dtype, x_stride, grad_stride))
    return DR_ERR_TOO_LARGE;
  if (workspace == nullptr || workspace_bytes < norm_space(s, true).total)
    return DR_ERR_WORKSPACE_TOO_SMALL;
  const NormParam w{weight, weight_dtype, weight_batch > 1 ? channels : 0};
  const NormParam b{bias, bias_dtype, bias_batch > 1 ? channels : 0};
  const DropKey key = drop_key(seed, seed_value, layer, drop_threshold);
  const Gradients out{grad_x,      grad_weight,      grad_bias,     weight_dtype,
                      bias_dtype,  weight_batch > 1, bias_batch > 1};
  const float bound = norm_bound(activation);
  return with_variant(dtype, v.vec, activation, drop_threshold, [&](auto k) {
    using K = decltype(k);
    return passes<typename K::Type, K::kVec, K::kSilu, K::kDrop>(
        x, grad_y, s, dtype, w, b, bound, key, mean, rstd, out,
        static_cast<unsigned char*>(workspace), as_stream(stream));
  });
}
