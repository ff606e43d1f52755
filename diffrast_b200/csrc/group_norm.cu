// Group normalisation with an activation and optional dropout: the forward pass (the formulas and
// the way views are cut up are in group_norm.cuh).
#include "group_norm.cuh"

namespace dr {
namespace {

constexpr int kStages = 8;  // rows that a thread has under way

// Joins the threads' moments of a block's rows into those of each channel: over the rows of a warp
// where the tile's columns divide it, then over the lines of rows that are left. `n` is the
// thread's count, `valid` the tile's channels (with folded pixels: the view's), `turn` the elements
// before the view's rows. `done` gets the channel, counted from the tile's first, and its moment.
template <int V, typename Done>
__device__ __forceinline__ void join_block(Moments<V>& m, float n, const TileThread& t,
                                           const NormShape& s, int valid, int turn, float2* entry,
                                           Done done) {
  __shared__ float counts[kNormThreads];  // of the lines
  m.finish(n);
  int lines = s.lanes, line = t.y;
  bool write = t.y < s.lanes;
  if (warp_holds_rows(s.tile_cols)) {
    for (int d = s.tile_cols; d < 32; d *= 2) m.join_lane(d, n);
    lines = kNormThreads / 32;
    line = t.thread / 32;
    write = t.thread % 32 < s.tile_cols;
  }
  const int width = s.tile_cols * V;
  __syncthreads();
  if (write) {
    float2* to = entry + line * width + t.x * V;
#pragma unroll
    for (int j = 0; j < V; ++j) to[j] = make_float2(m.sum.get(j), m.square.get(j));
    if (t.x == 0) counts[line] = n;
  }
  __syncthreads();
  // Channel by channel. With more than 16 parts to a channel and threads to spare, several threads
  // take some of its parts each, and one of them joins what they have.
  const int items = s.fold > 1 ? s.channels : width, parts = lines * s.fold;
  const int sharers = parts > 16 ? max(1, min(parts / 4, t.threads / valid)) : 1;
  auto join_parts = [&](int item, int first_part) {
    // Channel `item` is `lead` columns on in turned rows.
    const int at = item < turn ? item - turn + s.channels : item - turn;
    Moment c = {0.0f, 0.0f, 0.0f};
    for (int i = first_part; i < parts; i += sharers) {
      const float2 v = entry[i * items + at];
      c.join({counts[s.fold > 1 ? i / s.fold : i], v.x, v.y});
    }
    return c;
  };
  if (sharers == 1) {
    for (int item = t.thread; item < valid; item += t.threads) done(item, join_parts(item, 0));
    return;
  }
  __shared__ Moment shares[kNormThreads];
  const int item = t.thread / sharers;
  if (item < valid) shares[t.thread] = join_parts(item, t.thread - item * sharers);
  __syncthreads();
  if (t.thread < valid) {
    Moment c = shares[t.thread * sharers];
    for (int i = 1; i < sharers; ++i) c.join(shares[t.thread * sharers + i]);
    done(t.thread, c);
  }
}

// First pass: the moments of each channel over one chunk of rows in one tile of columns.
// parts [batch][chunks][channels] of (mean, squared deviations). Bound by memory, less what a
// block's start and join leave idle: 134 MB (four images of 512 x 512 x 64 bfloat16) in 32 us, 4.2
// TB/s, and 268 MB in 54 us, 5.0 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 4) norm_stats_kernel(const T* __restrict__ x,
                                                                     NormShape s, int view0,
                                                                     float2* __restrict__ parts) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormPlace p(s, V, view0 + blockIdx.z, blockIdx.y, blockIdx.x);
  RowRing<T, V, 1, kStages> ring;
  ring.image(0, x, s.x_view, s.x_row, p, s.lanes);
  ring.start(shared, p.count);
  Moments<V> m;
  m.clear();
  bool first = true;
  ring.for_rows([&](const Pairs<V> (&v)[1]) {
    if (first) m.start(v[0]);
    first = false;
    m.add(v[0]);
  });
  parts += (static_cast<long long>(p.view) * s.chunks + p.chunk) * s.channels;
  if (s.fold == 1) parts += blockIdx.y * s.tile_cols * V;
  const int tile_col = blockIdx.y * s.tile_cols;
  const int valid = s.fold > 1 ? s.channels : min(s.tile_cols, s.cols - tile_col) * V;
  const TileThread t = {static_cast<int>(threadIdx.x), static_cast<int>(threadIdx.y),
                        static_cast<int>(threadIdx.y * blockDim.x + threadIdx.x),
                        static_cast<int>(blockDim.x * blockDim.y)};
  const bool more = p.takes_leftovers(s, blockIdx.y);
  join_block<V>(m, static_cast<float>(p.count), t, s, valid, p.lead % s.channels,
                reinterpret_cast<float2*>(shared), [&](int item, Moment c) {
    if (more)
      s.for_leftovers(p.lead, item, [&](long long e) {
        c.join({1.0f, to_float(x[p.view * s.out_view + e]), 0.0f});
      });
    parts[item] = make_float2(c.mean, c.squares);
  });
  wait_for_kernel_before();
}

// The constants of the second pass that a group's moment leaves: table [batch][3][channels] of
// -mean, rstd * weight and bias.
__device__ __forceinline__ void write_constants(float* table, const NormShape& s, int view,
                                                int channel, float mean, float scale,
                                                float offset) {
  table += static_cast<long long>(view) * 3 * s.channels + channel;
  table[0] = -mean;
  table[s.channels] = scale;
  table[2 * s.channels] = offset;
}

// Joins the parts of a view's channels, and the channels of its groups where a block has them all;
// otherwise leaves (mean, squares) of the channels for norm_group_kernel. Bound by latency: 8 us for
// four views of 64 channels.
__global__ void __launch_bounds__(kJoinThreads) norm_join_kernel(
    const float2* parts, NormShape s, int view0, NormParam weight, NormParam bias, float eps,
    float* __restrict__ rstd, float* __restrict__ table, float2* __restrict__ channels) {
  __shared__ float2 entry[kJoinThreads + kJoinThreads / 8];
  __shared__ Moment channel[kJoinChannels];
  let_next_kernel_start();
  const JoinPlace p(s, view0);
  const int d = s.group_channels;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float scale = 1.0f, offset = 0.0f;  // weight and bias of channel `lane`, before the wait
  if (warp == 0 && lane < p.channels) {
    scale = load_scale(weight, p.view, p.channel + lane);
    offset = load_shift(bias, p.view, p.channel + lane);
  }
  wait_for_kernel_before();
  parts += static_cast<long long>(p.view) * s.chunks * s.channels + p.channel;
  const float fold = static_cast<float>(s.fold);
  const float chunk_count = static_cast<float>(s.chunk_rows) * fold;
  const float last_count =
      static_cast<float>(s.rows - static_cast<long long>(s.chunks - 1) * s.chunk_rows) * fold;
  auto count_of = [&](int chunk) {
    return (chunk + 1 < s.chunks ? chunk_count : last_count) +
           (chunk == 0 ? static_cast<float>(s.leftover) : 0.0f);
  };
  // This lane's chunks of channel x.
  LongMoment own;
  if (p.x < p.channels) {
#pragma unroll 8
    for (int i = p.y; i < s.chunks; i += p.lanes)
      own.join(count_of(i), parts[static_cast<long long>(i) * s.channels + p.x]);
  }
  entry[p.y * (p.width + 1) + p.x] = make_float2(own.mean.sum, own.squares.sum);
  __syncthreads();
  // A warp a channel, from its lanes; lane i has ceil((chunks - i) / lanes) chunks.
  for (int c = warp; c < p.channels; c += blockDim.x / 32) {
    Moment m = {0.0f, 0.0f, 0.0f};
    for (int i = lane; i < p.lanes; i += 32) {
      const float2 v = entry[i * (p.width + 1) + c];
      const int own = i < s.chunks ? (s.chunks - i + p.lanes - 1) / p.lanes : 0;
      const bool last = own > 0 && (s.chunks - 1) % p.lanes == i;
      float n = chunk_count * static_cast<float>(own - (last ? 1 : 0)) + (last ? last_count : 0.0f);
      if (i == 0) n += static_cast<float>(s.leftover);
      m.join({n, v.x, v.y});
    }
    m.join_warp();
    if (lane == 0) channel[c] = m;
  }
  __syncthreads();
  if (warp != 0 || lane >= p.channels) return;
  if (d > kJoinChannels) {
    const Moment c = channel[lane];
    channels[static_cast<long long>(p.view) * s.channels + p.channel + lane] =
        make_float2(c.mean, c.squares);
    return;
  }
  const int g = lane / d;
  Moment group = channel[g * d];
  for (int i = 1; i < d; ++i) group.join(channel[g * d + i]);
  const float r = rstd_of(group, eps);
  if (lane == g * d) rstd[static_cast<long long>(p.view) * s.groups + p.channel / d + g] = r;
  write_constants(table, s, p.view, p.channel + lane, group.mean, r * scale, offset);
}

// Joins the channels of one group of a view (groups wider than a block of norm_join_kernel).
__global__ void __launch_bounds__(kNormThreads) norm_group_kernel(
    const float2* channels, NormShape s, int view0, NormParam weight, NormParam bias, float eps,
    float* __restrict__ rstd, float* __restrict__ table) {
  __shared__ Moment warps[kNormThreads / 32];
  let_next_kernel_start();
  wait_for_kernel_before();
  const int view = view0 + blockIdx.y, first = blockIdx.x * s.group_channels;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const float pixels = static_cast<float>(s.pixels);
  Moment m = {0.0f, 0.0f, 0.0f};
  for (int i = threadIdx.x; i < s.group_channels; i += kNormThreads) {
    const float2 v = channels[static_cast<long long>(view) * s.channels + first + i];
    m.join({pixels, v.x, v.y});
  }
  m.join_warp();
  if (lane == 0) warps[warp] = m;
  __syncthreads();
  m = warps[0];
  for (int i = 1; i < kNormThreads / 32; ++i) m.join(warps[i]);
  const float r = rstd_of(m, eps);
  if (threadIdx.x == 0) rstd[static_cast<long long>(view) * s.groups + blockIdx.x] = r;
  for (int i = threadIdx.x; i < s.group_channels; i += kNormThreads)
    write_constants(table, s, view, first + i, m.mean, r * load_scale(weight, view, first + i),
                    load_shift(bias, view, first + i));
}

// Second pass: normalise, scale, activate and drop one chunk of rows in one tile of columns. Blocks
// run from the end of the views to their start: what the first pass read last is still in L2 (of
// four images of 512 x 512 x 64 bfloat16 a third is). For those it takes 43 us, 268 MB read and
// written at 6.2 TB/s, a third of it in L2; the special-function unit is busy for 29 us of it, and no
// unit is saturated. With dropout the generator's registers leave room for three blocks, and the
// pass is bound by its instructions: of eight images of 128 x 128 x 256 it issues one in 65% of the
// clocks, with 31% of the warps that a processor can hold, and moves only 1.8 TB/s of DRAM.
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, Drop ? 3 : 4) norm_apply_kernel(
    const T* __restrict__ x, NormShape s, int view0, const float* table, float bound, DropKey key,
    T* __restrict__ y) {
  extern __shared__ uint4 shared[];
  let_next_kernel_start();
  const NormPlace p(s, V, view0 + gridDim.z - 1 - blockIdx.z, gridDim.y - 1 - blockIdx.y,
                    gridDim.x - 1 - blockIdx.x);
  RowRing<T, V, 1, kStages> ring;
  ring.image(0, x, s.x_view, s.x_row, p, s.lanes);
  ring.start(shared, p.count);
  wait_for_kernel_before();
  const unsigned long long seed = Drop ? load_seed(key) : 0;
  if (p.takes_leftovers(s, gridDim.y - 1 - blockIdx.y)) {
    const float* row = table + static_cast<long long>(p.view) * 3 * s.channels;
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < s.channels;
         c += blockDim.x * blockDim.y)
      s.for_leftovers(p.lead, c, [&](long long e) {
        const long long at = p.view * s.out_view + e;
        const float z = fmaf(to_float(x[at]) + row[c], row[s.channels + c], row[2 * s.channels + c]);
        Pairs<1> v;
        v.p[0] = activate<Silu>(make_float2(z, 0.0f), bound);
        if (Drop) apply_dropout<1>(v, at, key, seed);
        y[at] = from_float<T>(v.p[0].x);
      });
  }
  if (p.count == 0) return;
  Affine<V> c;
  c.load(table, s, p.view, p.col + p.lead);
  long long at = p.at(s.out_view, s.out_row);
  const long long step = s.lanes * s.out_row;
  ring.for_rows([&](const Pairs<V> (&v)[1]) {
    Pairs<V> z;
#pragma unroll
    for (int j = 0; j < Pairs<V>::kCount; ++j)
      z.p[j] = activate<Silu>(fma2(add2(v[0].p[j], c.shift.p[j]), c.scale.p[j], c.bias.p[j]),
                              bound);
    if (Drop) apply_dropout<V>(z, at, key, seed);
    __stcs(reinterpret_cast<Packed<T, V>*>(y + at), pack_pairs<T, V>(z));
    at += step;
  });
}

// The whole pass by clusters of blocks (see "clusters" in group_norm.cuh). Bound by latency, of the
// copies, the joins and the cluster's barrier: 4.8 us for one 16 x 16 x 64 bfloat16 view. With many
// views (256 of 256 KB: 43 us, 3.1 TB/s) a block's copies, sums, joins and stores still follow one
// another, and the two or three blocks of a processor do not cover them.
template <typename T, int V, bool Silu, bool Drop>
__global__ void __launch_bounds__(kNormThreads, Drop ? 3 : 4) norm_cluster_kernel(
    const T* __restrict__ x, NormShape s, ClusterPlan t, NormParam weight, NormParam bias,
    float eps, float bound, DropKey key, T* __restrict__ y, float* __restrict__ table,
    float* __restrict__ rstd) {
  extern __shared__ uint4 shared[];
  auto* bytes = reinterpret_cast<unsigned char*>(shared);
  auto* entry = reinterpret_cast<float2*>(bytes + t.slots);
  const int width = s.tile_cols * V;
  auto* channel = reinterpret_cast<float2*>(bytes + t.slots + t.entries);  // [width]
  auto* constants = reinterpret_cast<float*>(channel + width);             // [3][width]
  const ClusterShare p(s, t, V);
  SlabRows<T, V, 1> rows;
  rows.slots = static_cast<unsigned int>(__cvta_generic_to_shared(shared)) +
               threadIdx.x * static_cast<unsigned int>(sizeof(Packed<T, V>));
  rows.count = p.mine;
  rows.fetch({x + p.in(s.x_view, s.x_row)}, {s.lanes * s.x_row});
  // Weight and bias, while the rows are on their way.
  for (int item = threadIdx.x; item < p.channels; item += kNormThreads) {
    constants[width + item] = load_scale(weight, p.view, p.channel + item);
    constants[2 * width + item] = load_shift(bias, p.view, p.channel + item);
  }
  copy_wait<0>();
  Moments<V> m;
  m.clear();
  bool first = true;
  rows.for_rows([&](const Pairs<V> (&v)[1]) {
    if (first) m.start(v[0]);
    first = false;
    m.add(v[0]);
  });
  join_block<V>(m, static_cast<float>(p.mine), p.at, s, p.channels, 0, entry,
                [&](int item, const Moment& c) { channel[item] = make_float2(c.mean, c.squares); });
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
      Moment c = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < kMostCluster; ++r)
        if (r < t.size) c.join({p.values_of(s, t, r), v[r].x, v[r].y});
      joined[item] = make_float2(c.mean, c.squares);
    }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  }
  __syncthreads();
  // The groups' moments, and from them the channels' constants.
  const int groups = p.channels / d;
  const int lanes = lanes_for(groups), lane = threadIdx.x & (lanes - 1);
  const int step = kNormThreads / lanes;
  const float all = static_cast<float>(s.pixels);
  for (int base = 0; base < groups; base += step) {
    const int g = base + threadIdx.x / lanes;
    Moment c = {0.0f, 0.0f, 0.0f};
    if (g < groups) {
      for (int i = lane; i < d; i += lanes) {
        const float2 v = joined[g * d + i];
        c.join({all, v.x, v.y});
      }
    }
    for (int e = 1; e < lanes; e *= 2) c.join(c.lane(e));
    const int leader = (threadIdx.x & 31) & ~(lanes - 1);
    const float mean = __shfl_sync(0xFFFFFFFFu, c.mean, leader);
    const float r = __shfl_sync(0xFFFFFFFFu, rstd_of(c, eps), leader);
    if (g < groups) {
      for (int i = lane; i < d; i += lanes) {
        const int item = g * d + i;
        const float scale = r * constants[width + item], offset = constants[2 * width + item];
        constants[item] = -mean;
        constants[width + item] = scale;
        if (p.rank == 0) {
          float* row = table + static_cast<long long>(p.view) * 3 * s.channels + p.channel + item;
          row[0] = -mean;
          row[s.channels] = scale;
          row[2 * s.channels] = offset;
        }
      }
      if (p.rank == 0 && lane == 0)
        rstd[static_cast<long long>(p.view) * s.groups + p.channel / d + g] = r;
    }
  }
  __syncthreads();
  if (p.mine > 0) {
    const Pairs<V> shift = load_constants<V>(constants, s, p);
    const Pairs<V> scale = load_constants<V>(constants + width, s, p);
    const Pairs<V> offset = load_constants<V>(constants + 2 * width, s, p);
    const unsigned long long seed = Drop ? load_seed(key) : 0;
    long long at = p.in(s.out_view, s.out_row);
    const long long stride = s.lanes * s.out_row;
    rows.for_rows([&](const Pairs<V> (&v)[1]) {
      Pairs<V> z;
#pragma unroll
      for (int j = 0; j < Pairs<V>::kCount; ++j)
        z.p[j] = activate<Silu>(fma2(add2(v[0].p[j], shift.p[j]), scale.p[j], offset.p[j]), bound);
      if (Drop) apply_dropout<V>(z, at, key, seed);
      __stcs(reinterpret_cast<Packed<T, V>*>(y + at), pack_pairs<T, V>(z));
      at += stride;
    });
  }
  // No block ends while another may still read its sums.
  if (t.size > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T, int V, bool Silu, bool Drop>
int passes(const void* x, const NormShape& s, const NormParam& weight, const NormParam& bias,
           float eps, float bound, const DropKey& key, void* y, float* table,
           float* rstd, unsigned char* workspace, cudaStream_t stream) {
  const NormSpace space = norm_space(s, false);
  auto* parts = reinterpret_cast<float2*>(workspace + space.parts);
  auto* channels = reinterpret_cast<float2*>(workspace + space.sums);
  const T* in = static_cast<const T*>(x);
  T* out = static_cast<T*>(y);
  const int most = views_at_once(s.batch);
  const unsigned int runs = join_runs(s);
  const dim3 threads(s.tile_cols, s.lanes);
  constexpr size_t ring = RowRing<T, V, 1, kStages>::kBytes;
  constexpr size_t shared = std::max(ring, sizeof(float2) * kNormThreads * V);
  cudaError_t err = cudaSuccess;
  for (long long view0 = 0; view0 < s.batch && err == cudaSuccess; view0 += most) {
    const int views = static_cast<int>(std::min<long long>(most, s.batch - view0));
    const dim3 blocks(s.chunks, s.tiles, views);
    err = launch_kernel(norm_stats_kernel<T, V>, blocks, threads, shared, stream, view0 > 0, in, s,
                        view0, parts);
    if (err == cudaSuccess)
      err = launch_kernel(norm_join_kernel, dim3(runs, views), join_threads(s), 0, stream, true,
                          parts, s, view0, weight, bias, eps, rstd, table, channels);
    if (err == cudaSuccess && s.group_channels > kJoinChannels)
      err = launch_kernel(norm_group_kernel, dim3(s.groups, views), kNormThreads, 0, stream, true,
                          channels, s, view0, weight, bias, eps, rstd, table);
    if (err == cudaSuccess)
      err = launch_kernel(norm_apply_kernel<T, V, Silu, Drop>, blocks, threads, ring, stream, true,
                          in, s, view0, table, bound, key, out);
  }
  return err == cudaSuccess ? launch_status() : static_cast<int>(err);
}

}  // namespace
}  // namespace dr

using namespace dr;

extern "C" size_t dr_group_norm_state_floats(int64_t batch, int32_t channels, int32_t groups) {
  return batch < 0 || channels < 1 || groups < 1
             ? 0
             : static_cast<size_t>(batch) * (3 * static_cast<size_t>(channels) + groups);
}

extern "C" size_t dr_group_norm_workspace_bytes(int64_t batch, int64_t pixels, int32_t channels,
                                                int32_t groups, int32_t dtype, int32_t backward) {
  if (bad_norm_sizes(batch, pixels, channels, groups, dtype) || too_large(batch, pixels, channels))
    return 0;
  return norm_workspace_bytes(batch, pixels, channels, groups, dtype, backward != 0);
}

extern "C" int dr_group_norm_fwd(const void* x, int64_t x_stride, int32_t dtype, int64_t batch,
                                 int64_t pixels, int32_t channels, int32_t groups,
                                 const void* weight, int32_t weight_dtype, int64_t weight_batch,
                                 const void* bias, int32_t bias_dtype, int64_t bias_batch,
                                 float eps, int32_t activation, int32_t drop_threshold,
                                 const int64_t* seed, int64_t seed_value, int64_t layer, void* y,
                                 float* state, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (bad_norm_sizes(batch, pixels, channels, groups, dtype) || x_stride < channels ||
      bad_norm_param(weight, weight_dtype, weight_batch, batch) ||
      bad_norm_param(bias, bias_dtype, bias_batch, batch) || activation < DR_ACTIVATION_NONE ||
      activation > DR_ACTIVATION_SILU || bad_drop(drop_threshold, layer))
    return DR_ERR_INVALID_ARGUMENT;
  if (batch == 0 || pixels == 0) return DR_OK;
  const size_t size = dtype_bytes(dtype);
  if (x == nullptr || y == nullptr || state == nullptr || !aligned_to(state, 16) ||
      !aligned_to(workspace, 16) || !aligned_to(seed, sizeof(int64_t)) || !aligned_to(x, size) ||
      !aligned_to(y, size))
    return DR_ERR_INVALID_ARGUMENT;
  if (too_large(batch, pixels, x_stride)) return DR_ERR_TOO_LARGE;
  NormShape s;
  ClusterPlan t;
  NormVector v = choose_vector(pixels, channels, dtype, x_stride, channels, {x, y}, false);
  const bool clusters = plan_clusters(s, t, v, batch, pixels, channels, groups, dtype, x_stride,
                                      channels, 1, processors());
  if (!clusters) {
    v = choose_vector(pixels, channels, dtype, x_stride, channels, {x, y}, true);
    plan_passes(s, v, batch, pixels, channels, groups, dtype, x_stride, channels, 1, processors());
    if (workspace == nullptr || workspace_bytes < norm_space(s, false).total)
      return DR_ERR_WORKSPACE_TOO_SMALL;
  }
  auto param = [&](const void* data, int32_t type, int64_t rows) {
    return data != nullptr ? NormParam{data, true, type, rows > 1 ? channels : 0}
                           : NormParam{state, false, DR_FLOAT32, 0};
  };
  const NormParam w = param(weight, weight_dtype, weight_batch);
  const NormParam b = param(bias, bias_dtype, bias_batch);
  const DropKey key = drop_key(seed, seed_value, layer, drop_threshold);
  const float bound = norm_bound(activation);
  float* rstd = state + static_cast<size_t>(batch) * 3 * channels;
  return with_variant(dtype, v.vec, activation, drop_threshold, [&](auto k) {
    using K = decltype(k);
    using T = typename K::Type;
    if (clusters)
      return launch_clusters<norm_cluster_kernel<T, K::kVec, K::kSilu, K::kDrop>>(
          t, as_stream(stream), static_cast<const T*>(x), s, t, w, b, eps, bound, key,
          static_cast<T*>(y), state, rstd);
    return passes<T, K::kVec, K::kSilu, K::kDrop>(
        x, s, w, b, eps, bound, key, y, state, rstd, static_cast<unsigned char*>(workspace),
        as_stream(stream));
  });
}
