// Group normalisation with an activation and optional dropout: the backward pass (the formulas and
// the way views are cut up are in group_norm.cuh). Nothing of the forward pass is kept but the
// image and the table of its channels' constants: z, its derivative and the dropout's mask are
// computed again.
#include "group_norm.cuh"

namespace dr {
namespace {

constexpr int kStages = 4;  // rows of x and of the gradient that a thread has under way

// Joins the threads' sums of a block's rows into those of each channel: over the rows of a warp
// where the tile's columns divide it, then over the lines of rows that are left. `valid` is the
// tile's channels (with folded pixels: the view's), `turn` the elements before the view's rows.
template <int V, typename Done>
__device__ __forceinline__ void join_block(Pairs<V>& sum, Pairs<V>& dot, const TileThread& t,
                                           const NormShape& s, int valid, int turn, float2* entry,
                                           Done done) {
  int lines = s.lanes, line = t.y;
  bool write = t.y < s.lanes;
  if (warp_holds_rows(s.tile_cols)) {
    for (int d = s.tile_cols; d < 32; d *= 2) {
#pragma unroll
      for (int j = 0; j < Pairs<V>::kCount; ++j) {
        float2 a, b;
        a.x = __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].x, d);
        b.x = __shfl_xor_sync(0xFFFFFFFFu, dot.p[j].x, d);
        a.y = V > 1 ? __shfl_xor_sync(0xFFFFFFFFu, sum.p[j].y, d) : 0.0f;
        b.y = V > 1 ? __shfl_xor_sync(0xFFFFFFFFu, dot.p[j].y, d) : 0.0f;
        sum.p[j] = add2(sum.p[j], a);
        dot.p[j] = add2(dot.p[j], b);
      }
    }
    lines = kNormThreads / 32;
    line = t.thread / 32;
    write = t.thread % 32 < s.tile_cols;
  }
  const int width = s.tile_cols * V;
  __syncthreads();
  if (write) {
    float2* to = entry + line * width + t.x * V;
#pragma unroll
    for (int j = 0; j < V; ++j) to[j] = make_float2(sum.get(j), dot.get(j));
  }
  __syncthreads();
  // Channel by channel. With more than 16 parts to a channel and threads to spare, several threads
  // take some of its parts each, and one of them adds what they have.
  const int items = s.fold > 1 ? s.channels : width, parts = lines * s.fold;
  const int sharers = parts > 16 ? max(1, min(parts / 4, t.threads / valid)) : 1;
  auto add_parts = [&](int item, int first_part) {
    // Channel `item` is `lead` columns on in turned rows.
    const int at = item < turn ? item - turn + s.channels : item - turn;
    float2 total = make_float2(0.0f, 0.0f);
    for (int i = first_part; i < parts; i += sharers) total = add2(total, entry[i * items + at]);
    return total;
  };
  if (sharers == 1) {
    for (int item = t.thread; item < valid; item += t.threads) done(item, add_parts(item, 0));
    return;
  }
  __shared__ float2 shares[kNormThreads];
  const int item = t.thread / sharers;
  if (item < valid) shares[t.thread] = add_parts(item, t.thread - item * sharers);
  __syncthreads();
  if (t.thread < valid) {
    float2 total = shares[t.thread * sharers];
    for (int i = 1; i < sharers; ++i) total = add2(total, shares[t.thread * sharers + i]);
    done(t.thread, total);
  }
}

// One element outside the rows: x - m and q.
struct Leftover {
  float d, u;
};

template <typename T, bool Silu, bool Drop>
__device__ __forceinline__ Leftover leftover_at(const T* x, const T* grad, long long at,
                                                const float* row, int channels, int channel,
                                                float bound, const DropKey& key,
                                                unsigned long long seed) {
  const float d = to_float(x[at]) + row[channel];
  const float z = fmaf(d, row[channels + channel], row[2 * channels + channel]);
  Pairs<1> q;
  q.p[0] = make_float2(to_float(grad[at]), 0.0f);
  if (Drop) apply_dropout<1>(q, at, key, seed);
  return {d, activate_grad<Silu>(q.p[0], make_float2(z, 0.0f), bound).x};
}

// First pass: sums of q and q (x - m) of each channel over one chunk of rows in one tile of columns.
// parts [batch][chunks][channels]. Bound by memory: 268 MB (x and the gradient of four images of 512
// x 512 x 64 bfloat16) in 57 us, 4.7 TB/s; a warp has 117 instructions for each of its rows of
// vectors, 55% of the rate at which it could issue them, and 16 results of the special-function unit.
// With dropout the generator's registers leave room for two blocks, and both passes are bound by
// their instructions (64% of the rate, with 23% of the warps that a processor can hold).
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, Drop ? 2 : 3) norm_sums_kernel(
    const T* __restrict__ x, const T* __restrict__ grad, NormShape s, int view0,
    const float* __restrict__ table, float bound, DropKey key, float2* __restrict__ parts) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormPlace p(s, V, view0 + blockIdx.z, blockIdx.y, blockIdx.x);
  RowRing<T, V, 2, kStages> ring;
  ring.image(0, x, s.x_view, s.x_row, p, s.lanes);
  ring.image(1, grad, s.grad_view, s.grad_row, p, s.lanes);
  ring.start(shared, p.count);
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  Pairs<V> sum, dot;
#pragma unroll
  for (int j = 0; j < Pairs<V>::kCount; ++j) sum.p[j] = dot.p[j] = both(0.0f);
  if (p.count > 0) {
    Affine<V> c;
    c.load(table, s, p.view, p.col + p.lead);
    long long at = p.at(s.out_view, s.out_row);
    const long long step = s.lanes * s.out_row;
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
  parts += (static_cast<long long>(p.view) * s.chunks + p.chunk) * s.channels;
  if (s.fold == 1) parts += blockIdx.y * s.tile_cols * V;
  const int tile_col = blockIdx.y * s.tile_cols;
  const int valid = s.fold > 1 ? s.channels : min(s.tile_cols, s.cols - tile_col) * V;
  const TileThread t = {static_cast<int>(threadIdx.x), static_cast<int>(threadIdx.y),
                        static_cast<int>(threadIdx.y * blockDim.x + threadIdx.x),
                        static_cast<int>(blockDim.x * blockDim.y)};
  const bool more = p.takes_leftovers(s, blockIdx.y);
  const float* row = table + static_cast<long long>(p.view) * 3 * s.channels;
  join_block<V>(sum, dot, t, s, valid, p.lead % s.channels, reinterpret_cast<float2*>(shared),
                [&](int item, float2 total) {
    if (more)
      s.for_leftovers(p.lead, item, [&](long long e) {
        const long long at = p.view * s.out_view + e;
        const Leftover l = leftover_at<T, Silu, Drop>(x, grad, at, row, s.channels, item, bound, key, seed);
        total = make_float2(total.x + l.u, fmaf(l.u, l.d, total.y));
      });
    parts[item] = total;
  });
  wait_for_kernel_before();
}

// The constants of the second pass that a group's sums of q w r and q h w r leave: table
// [batch][2][channels] of -r A and -r^2 B.
__device__ __forceinline__ void write_constants(float* table, const NormShape& s, int view,
                                                int channel, float2 group, float r) {
  const float inverse =
      1.0f / (static_cast<float>(s.pixels) * static_cast<float>(s.group_channels));
  table += static_cast<long long>(view) * 2 * s.channels + channel;
  table[0] = -group.x * inverse;
  table[s.channels] = -group.y * inverse * r;
}

// Joins the parts of a view's channels into sums [batch][channels] of q and q h, and the channels of
// its groups where a block has them all; the others are left to norm_group_means_kernel. Bound by
// latency: 8 us for four views of 64 channels.
__global__ void __launch_bounds__(kJoinThreads) norm_means_kernel(
    const float2* parts, NormShape s, int view0, const float* __restrict__ affine,
    const float* __restrict__ rstd, float2* __restrict__ sums, float* __restrict__ table) {
  __shared__ float2 entry[kJoinThreads + kJoinThreads / 8];
  __shared__ float2 scaled[kJoinChannels];
  let_next_kernel_start();
  const JoinPlace p(s, view0);
  const int d = s.group_channels;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // rstd * weight of the channels
  affine += (static_cast<long long>(p.view) * 3 + 1) * s.channels + p.channel;
  rstd += static_cast<long long>(p.view) * s.groups;
  parts += static_cast<long long>(p.view) * s.chunks * s.channels + p.channel;
  sums += static_cast<long long>(p.view) * s.channels + p.channel;
  wait_for_kernel_before();
  // This lane's chunks of channel x.
  LongSum sum, dot;
  if (p.x < p.channels) {
#pragma unroll 8
    for (int i = p.y; i < s.chunks; i += p.lanes) {
      const float2 v = parts[static_cast<long long>(i) * s.channels + p.x];
      sum.add(v.x);
      dot.add(v.y);
    }
  }
  entry[p.y * (p.width + 1) + p.x] = make_float2(sum.sum, dot.sum);
  __syncthreads();
  // A warp a channel, from its lanes.
  for (int c = warp; c < p.channels; c += blockDim.x / 32) {
    float2 total = make_float2(0.0f, 0.0f);
    for (int i = lane; i < p.lanes; i += 32) total = add2(total, entry[i * (p.width + 1) + c]);
    total.x = warp_sum(total.x);
    total.y = warp_sum(total.y);
    if (lane == 0) {
      const float r = rstd[(p.channel + c) / d], scale = affine[c];
      sums[c] = make_float2(total.x, total.y * r);
      scaled[c] = make_float2(total.x * scale, total.y * r * scale);
    }
  }
  __syncthreads();
  if (warp != 0 || lane >= p.channels || d > kJoinChannels) return;
  const int g = lane / d;
  float2 group = scaled[g * d];
  for (int i = 1; i < d; ++i) group = add2(group, scaled[g * d + i]);
  write_constants(table, s, p.view, p.channel + lane, group, rstd[p.channel / d + g]);
}

// Joins the channels of one group of a view (groups wider than a block of norm_means_kernel).
__global__ void __launch_bounds__(kNormThreads) norm_group_means_kernel(
    const float2* sums, NormShape s, int view0, const float* __restrict__ affine,
    const float* __restrict__ rstd, float* __restrict__ table) {
  __shared__ float2 warps[kNormThreads / 32];
  let_next_kernel_start();
  wait_for_kernel_before();
  const int view = view0 + blockIdx.y, first = blockIdx.x * s.group_channels;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const float* scales = affine + (static_cast<long long>(view) * 3 + 1) * s.channels + first;
  float2 total = make_float2(0.0f, 0.0f);
  for (int i = threadIdx.x; i < s.group_channels; i += kNormThreads) {
    const float2 v = sums[static_cast<long long>(view) * s.channels + first + i];
    total = make_float2(fmaf(v.x, scales[i], total.x), fmaf(v.y, scales[i], total.y));
  }
  total.x = warp_sum(total.x);
  total.y = warp_sum(total.y);
  if (lane == 0) warps[warp] = total;
  __syncthreads();
  total = warps[0];
  for (int i = 1; i < kNormThreads / 32; ++i) total = add2(total, warps[i]);
  const float r = rstd[static_cast<long long>(view) * s.groups + blockIdx.x];
  for (int i = threadIdx.x; i < s.group_channels; i += kNormThreads)
    write_constants(table, s, view, first + i, total, r);
}

// Second pass: grad x = r (q w - A - h B) over one chunk of rows in one tile of columns, from the
// end of the views to their start (what the first pass read last is still in L2: of four images of
// 512 x 512 x 64 bfloat16 a fifth is). Bound by memory: 60 us for those, 403 MB read and written.
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, Drop ? 2 : 3) norm_grad_kernel(
    const T* __restrict__ x, const T* __restrict__ grad, NormShape s, int view0,
    const float* __restrict__ affine, const float* table, float bound, DropKey key,
    T* __restrict__ grad_x) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormPlace p(s, V, view0 + gridDim.z - 1 - blockIdx.z, gridDim.y - 1 - blockIdx.y,
                    gridDim.x - 1 - blockIdx.x);
  RowRing<T, V, 2, kStages> ring;
  ring.image(0, x, s.x_view, s.x_row, p, s.lanes);
  ring.image(1, grad, s.grad_view, s.grad_row, p, s.lanes);
  ring.start(shared, p.count);
  Affine<V> c;
  if (p.count > 0) c.load(affine, s, p.view, p.col + p.lead);
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  wait_for_kernel_before();
  table += static_cast<long long>(p.view) * 2 * s.channels;
  if (p.takes_leftovers(s, gridDim.y - 1 - blockIdx.y)) {
    const float* row = affine + static_cast<long long>(p.view) * 3 * s.channels;
    for (int ch = threadIdx.y * blockDim.x + threadIdx.x; ch < s.channels;
         ch += blockDim.x * blockDim.y)
      s.for_leftovers(p.lead, ch, [&](long long e) {
        const long long own = p.view * s.out_view + e;
        const Leftover l = leftover_at<T, Silu, Drop>(x, grad, own, row, s.channels, ch, bound, key, seed);
        grad_x[own] = from_float<T>(
            fmaf(l.u, row[s.channels + ch], fmaf(l.d, table[s.channels + ch], table[ch])));
      });
  }
  if (p.count == 0) return;
  const Pairs<V> base = load_row<V>(table, s, p.col + p.lead);
  const Pairs<V> slope = load_row<V>(table + s.channels, s, p.col + p.lead);
  long long at = p.at(s.out_view, s.out_row);
  const long long step = s.lanes * s.out_row;
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

// Gradients of weight and bias: sums over the views (or each view's own), 8 channels a block. The
// sums are held in 64 bits: a lane may add thousands of views one after the other, which in 32 bits
// left 131077 equal views 1e-4 off. Bound by latency (3 us; its launch overlaps the second pass).
constexpr int kParamChannels = 8;

__global__ void __launch_bounds__(kNormThreads) norm_params_kernel(
    const float2* sums, long long batch, int channels, void* grad_weight,
    int weight_dtype, bool weight_views, void* grad_bias, int bias_dtype, bool bias_views) {
  constexpr int kLanes = kNormThreads / kParamChannels;
  __shared__ double2 entry[kLanes][kParamChannels];
  let_next_kernel_start();
  wait_for_kernel_before();
  const int x = threadIdx.x % kParamChannels, lane = threadIdx.x / kParamChannels;
  const int c = blockIdx.x * kParamChannels + x;
  double2 total = make_double2(0.0, 0.0);
  if (c < channels) {
#pragma unroll 4
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
  entry[lane][x] = total;
  __syncthreads();
  if (lane != 0 || c >= channels) return;
  const int lanes = static_cast<int>(min(batch, static_cast<long long>(kLanes)));
  for (int i = 1; i < lanes; ++i) {
    total.x += entry[i][x].x;
    total.y += entry[i][x].y;
  }
  if (grad_weight != nullptr && !weight_views)
    store_param(grad_weight, weight_dtype, c, static_cast<float>(total.y));
  if (grad_bias != nullptr && !bias_views)
    store_param(grad_bias, bias_dtype, c, static_cast<float>(total.x));
}

struct Gradients {
  void *x, *weight, *bias;
  int weight_dtype, bias_dtype;
  bool weight_views, bias_views;
};

// The whole pass by clusters of blocks (see "clusters" in group_norm.cuh). The gradients of weight
// and bias are written here where they are sums of one view (`direct`); otherwise the views' sums
// are left for norm_params_kernel. Bound by latency: 4.5 us for one 16 x 16 x 64 bfloat16 view.
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, Drop ? 2 : 3) norm_cluster_bwd_kernel(
    const T* __restrict__ x, const T* __restrict__ grad, NormShape s, ClusterPlan t,
    const float* __restrict__ affine, const float* __restrict__ rstd, float bound, DropKey key,
    Gradients out, bool direct, float2* __restrict__ sums) {
  extern __shared__ uint4 shared[];
  auto* bytes = reinterpret_cast<unsigned char*>(shared);
  auto* entry = reinterpret_cast<float2*>(bytes + t.slots);
  const int width = s.tile_cols * V;
  auto* channel = reinterpret_cast<float2*>(bytes + t.slots + t.entries);  // [width]
  auto* constants = reinterpret_cast<float*>(channel + width);             // [2][width]
  T* grad_x = static_cast<T*>(out.x);
  const ClusterShare p(s, t, V);
  SlabRows<T, V, 2> rows;
  rows.slots = static_cast<unsigned int>(__cvta_generic_to_shared(shared)) +
               threadIdx.x * static_cast<unsigned int>(sizeof(Packed<T, V>));
  rows.count = p.mine;
  rows.fetch({x + p.in(s.x_view, s.x_row), grad + p.in(s.grad_view, s.grad_row)},
             {s.lanes * s.x_row, s.lanes * s.grad_row});
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  const long long start = p.in(s.out_view, s.out_row), stride = s.lanes * s.out_row;
  Affine<V> c;
  Pairs<V> sum, dot;
#pragma unroll
  for (int j = 0; j < Pairs<V>::kCount; ++j) sum.p[j] = dot.p[j] = both(0.0f);
  if (p.mine > 0) c.load(affine, s, p.view, p.col);
  copy_wait<0>();
  long long at = start;
  rows.for_rows([&](Pairs<V> (&v)[2]) {
    if (Drop) apply_dropout<V>(v[1], at, key, seed);
    at += stride;
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j) {
      const float2 e = add2(v[0].p[j], c.shift.p[j]);
      const float2 z = fma2(e, c.scale.p[j], c.bias.p[j]);
      const float2 u = activate_grad<Silu>(v[1].p[j], z, bound);
      sum.p[j] = add2(sum.p[j], u);
      dot.p[j] = fma2(u, e, dot.p[j]);
    }
  });
  join_block<V>(sum, dot, p.at, s, p.channels, 0, entry,
                [&](int item, float2 total) { channel[item] = total; });
  const int d = s.group_channels;
  float2* joined = channel;
  if (t.size > 1) {
    auto cluster = cooperative_groups::this_cluster();
    cluster.sync();
    joined = entry;  // its readers are behind the cluster's barrier
    for (int item = threadIdx.x; item < p.channels; item += kNormThreads) {
      float2 v[kMostCluster];
#pragma unroll
      for (int r = 0; r < kMostCluster; ++r)
        if (r < t.size) v[r] = *cluster.map_shared_rank(channel + item, r);
      float2 total = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int r = 0; r < kMostCluster; ++r)
        if (r < t.size) total = add2(total, v[r]);
      joined[item] = total;
    }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  }
  __syncthreads();
  // The groups' means, and from them the channels' constants of grad x.
  const int groups = p.channels / d;
  const int lanes = lanes_for(groups), lane = threadIdx.x & (lanes - 1);
  const int step = kNormThreads / lanes;
  const float inverse = 1.0f / (static_cast<float>(s.pixels) * static_cast<float>(d));
  const float* scales = affine + (static_cast<long long>(p.view) * 3 + 1) * s.channels + p.channel;
  const float* rs = rstd + static_cast<long long>(p.view) * s.groups + p.channel / d;
  for (int base = 0; base < groups; base += step) {
    const int g = base + threadIdx.x / lanes;
    float2 total = make_float2(0.0f, 0.0f);
    float r = 0.0f;
    if (g < groups) {
      r = __ldg(rs + g);
      for (int i = lane; i < d; i += lanes) {
        const float2 v = joined[g * d + i];
        const float scale = __ldg(scales + g * d + i);
        total = add2(total, make_float2(v.x * scale, v.y * r * scale));
      }
    }
    for (int e = 1; e < lanes; e *= 2) {
      total.x += __shfl_xor_sync(0xFFFFFFFFu, total.x, e);
      total.y += __shfl_xor_sync(0xFFFFFFFFu, total.y, e);
    }
    if (g < groups) {
      for (int i = lane; i < d; i += lanes) {
        const int item = g * d + i;
        constants[item] = -total.x * inverse;
        constants[width + item] = -total.y * inverse * r;
        if (p.rank == 0) {
          const float2 v = joined[item];
          const long long own = static_cast<long long>(p.view) * s.channels + p.channel + item;
          if (!direct) {
            sums[own] = make_float2(v.x, v.y * r);
          } else {
            if (out.weight != nullptr) store_param(out.weight, out.weight_dtype, own, v.y * r);
            if (out.bias != nullptr) store_param(out.bias, out.bias_dtype, own, v.x);
          }
        }
      }
    }
  }
  __syncthreads();
  if (p.mine > 0 && grad_x != nullptr) {
    const Pairs<V> base = load_constants<V>(constants, s, p);
    const Pairs<V> slope = load_constants<V>(constants + width, s, p);
    at = start;
    rows.for_rows([&](Pairs<V> (&v)[2]) {
      if (Drop) apply_dropout<V>(v[1], at, key, seed);
#pragma unroll
      for (int j = 0; j < Pairs<V>::kCount; ++j) {
        const float2 e = add2(v[0].p[j], c.shift.p[j]);
        const float2 z = fma2(e, c.scale.p[j], c.bias.p[j]);
        const float2 u = activate_grad<Silu>(v[1].p[j], z, bound);
        v[0].p[j] = fma2(u, c.scale.p[j], fma2(e, slope.p[j], base.p[j]));
      }
      __stcs(reinterpret_cast<Packed<T, V>*>(grad_x + at), pack_pairs<T, V>(v[0]));
      at += stride;
    });
  }
  // No block ends while another may still read its sums.
  if (t.size > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

int params(const NormShape& s, const float2* sums, const Gradients& out, cudaStream_t stream,
           bool after) {
  if (out.weight == nullptr && out.bias == nullptr) return DR_OK;
  return static_cast<int>(launch_kernel(
      norm_params_kernel, blocks_for(s.channels, kParamChannels), kNormThreads, 0, stream, after, sums,
      s.batch, s.channels, out.weight, out.weight_dtype, out.weight_views, out.bias,
      out.bias_dtype, out.bias_views));
}

template <typename T, int V, bool Silu, bool Drop>
int clusters(const void* x, const void* grad, const NormShape& s, const ClusterPlan& t,
             const float* affine, const float* rstd, float bound, const DropKey& key,
             const Gradients& out, float2* sums, cudaStream_t stream) {
  const bool direct = s.batch == 1 || ((out.weight == nullptr || out.weight_views) &&
                                       (out.bias == nullptr || out.bias_views));
  const int status = launch_clusters<norm_cluster_bwd_kernel<T, V, Silu, Drop>>(
      t, stream, static_cast<const T*>(x), static_cast<const T*>(grad), s, t, affine, rstd, bound,
      key, out, direct, sums);
  return status != DR_OK || direct ? status : params(s, sums, out, stream, false);
}

template <typename T, int V, bool Silu, bool Drop>
int passes(const void* x, const void* grad, const NormShape& s, const float* affine,
           const float* rstd, float bound, const DropKey& key, const Gradients& out,
           unsigned char* workspace, cudaStream_t stream) {
  const NormSpace space = norm_space(s, true);
  auto* parts = reinterpret_cast<float2*>(workspace + space.parts);
  auto* sums = reinterpret_cast<float2*>(workspace + space.sums);
  auto* table = reinterpret_cast<float*>(workspace + space.table);
  const T* in = static_cast<const T*>(x);
  const T* dy = static_cast<const T*>(grad);
  const int most = views_at_once(s.batch);
  const unsigned int runs = join_runs(s);
  const dim3 threads(s.tile_cols, s.lanes);
  constexpr size_t ring = RowRing<T, V, 2, kStages>::kBytes;
  constexpr size_t shared = std::max(ring, sizeof(float2) * kNormThreads * V);
  cudaError_t err = cudaSuccess;
  for (long long view0 = 0; view0 < s.batch && err == cudaSuccess; view0 += most) {
    const int views = static_cast<int>(std::min<long long>(most, s.batch - view0));
    const dim3 blocks(s.chunks, s.tiles, views);
    err = launch_kernel(norm_sums_kernel<T, V, Silu, Drop>, blocks, threads, shared, stream,
                        view0 > 0, in, dy, s, view0, affine, bound, key, parts);
    if (err == cudaSuccess)
      err = launch_kernel(norm_means_kernel, dim3(runs, views), join_threads(s), 0, stream, true,
                          parts, s, view0, affine, rstd, sums, table);
    if (err == cudaSuccess && out.x != nullptr && s.group_channels > kJoinChannels)
      err = launch_kernel(norm_group_means_kernel, dim3(s.groups, views), kNormThreads, 0, stream,
                          true, sums, s, view0, affine, rstd, table);
    if (err == cudaSuccess && out.x != nullptr)
      err = launch_kernel(norm_grad_kernel<T, V, Silu, Drop>, blocks, threads, ring, stream, true,
                          in, dy, s, view0, affine, table, bound, key, static_cast<T*>(out.x));
  }
  return err == cudaSuccess ? params(s, sums, out, stream, true) : static_cast<int>(err);
}

}  // namespace
}  // namespace dr

using namespace dr;

extern "C" int dr_group_norm_bwd(const void* x, int64_t x_stride, const void* grad_y,
                                 int64_t grad_stride, int32_t dtype, int64_t batch, int64_t pixels,
                                 int32_t channels, int32_t groups, const float* state,
                                 int32_t activation, int32_t drop_threshold, const int64_t* seed,
                                 int64_t seed_value, int64_t layer, void* grad_x,
                                 void* grad_weight, int32_t weight_dtype, int64_t weight_batch,
                                 void* grad_bias, int32_t bias_dtype, int64_t bias_batch,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_norm_sizes(batch, pixels, channels, groups, dtype) || x_stride < channels ||
      grad_stride < channels || bad_norm_param(grad_weight, weight_dtype, weight_batch, batch) ||
      bad_norm_param(grad_bias, bias_dtype, bias_batch, batch) ||
      activation < DR_ACTIVATION_NONE || activation > DR_ACTIVATION_SILU ||
      bad_drop(drop_threshold, layer))
    return DR_ERR_INVALID_ARGUMENT;
  if (batch == 0 || pixels == 0) return DR_OK;
  const size_t size = dtype_bytes(dtype);
  if (x == nullptr || grad_y == nullptr || state == nullptr || !aligned_to(state, 16) ||
      !aligned_to(workspace, 16) || !aligned_to(seed, sizeof(int64_t)) || !aligned_to(x, size) ||
      !aligned_to(grad_y, size) || !aligned_to(grad_x, size))
    return DR_ERR_INVALID_ARGUMENT;
  if (too_large(batch, pixels, std::max(x_stride, grad_stride))) return DR_ERR_TOO_LARGE;
  NormShape s;
  ClusterPlan t;
  NormVector v = choose_vector(pixels, channels, dtype, x_stride, grad_stride,
                               {x, grad_y, grad_x}, false);
  const bool small = plan_clusters(s, t, v, batch, pixels, channels, groups, dtype, x_stride,
                                   grad_stride, 2, processors());
  if (!small) {
    v = choose_vector(pixels, channels, dtype, x_stride, grad_stride, {x, grad_y, grad_x}, true);
    plan_passes(s, v, batch, pixels, channels, groups, dtype, x_stride, grad_stride, 2,
                processors());
  }
  const size_t need = small ? cluster_space(s) : norm_space(s, true).total;
  if (workspace == nullptr || workspace_bytes < need) return DR_ERR_WORKSPACE_TOO_SMALL;
  const DropKey key = drop_key(seed, seed_value, layer, drop_threshold);
  const Gradients out{grad_x,      grad_weight,      grad_bias,     weight_dtype,
                      bias_dtype,  weight_batch > 1, bias_batch > 1};
  const float bound = norm_bound(activation);
  const float* rstd = state + static_cast<size_t>(batch) * 3 * channels;
  return with_variant(dtype, v.vec, activation, drop_threshold, [&](auto k) {
    using K = decltype(k);
    if (small)
      return clusters<typename K::Type, K::kVec, K::kSilu, K::kDrop>(
          x, grad_y, s, t, state, rstd, bound, key, out, static_cast<float2*>(workspace),
          as_stream(stream));
    return passes<typename K::Type, K::kVec, K::kSilu, K::kDrop>(
        x, grad_y, s, state, rstd, bound, key, out,
        static_cast<unsigned char*>(workspace), as_stream(stream));
  });
}
