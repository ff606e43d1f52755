// Host-only check of how group norm cuts views up: for many sizes, the plans of a call in clusters
// and in passes give a thread at most kThreadRows rows (the statistics' rounding grows with them),
// cover every row, and fit shared memory. Prints the plans checked, or the first that is wrong.
#include <cstdio>

#include "group_norm.cuh"

using namespace dr;

namespace {

long long checked = 0;

bool check(long long batch, long long pixels, int channels, int groups, int dtype, long long x_stride,
           const NormVector& v, int images) {
  NormShape s;
  ClusterPlan t;
  const bool clusters = plan_clusters(s, t, v, batch, pixels, channels, groups, dtype, x_stride,
                                      channels, images, 148);
  long long rows = s.lane_rows;
  bool good = true;
  if (clusters) {
    rows = (t.block_rows + s.lanes - 1) / s.lanes;
    good = t.shared <= kMostShared && static_cast<long long>(t.block_rows) * t.size >= s.rows &&
           t.slabs == batch * s.tiles;
  } else {
    plan_passes(s, v, batch, pixels, channels, groups, dtype, x_stride, channels, images, 148);
    rows = s.lane_rows;
    good = static_cast<long long>(s.chunk_rows) * s.chunks >= s.rows;
  }
  ++checked;
  if (good && rows <= kThreadRows) return true;
  std::printf("wrong: %lld views of %lld pixels of %d channels in %d groups, type %d, stride %lld, "
              "vectors of %d, %d folded, %d images, %s: %lld rows to a thread\n",
              batch, pixels, channels, groups, dtype, x_stride, v.vec, v.fold, images,
              clusters ? "clusters" : "passes", rows);
  return false;
}

}  // namespace

int main() {
  const int channel_counts[] = {1, 2, 3, 4, 6, 7, 8, 12, 16, 24, 30, 32, 48, 64, 96, 100, 128, 130, 256, 500};
  for (long long batch : {1LL, 2LL, 7LL, 64LL, 148LL, 1024LL, 16384LL, 100000LL})
    for (long long pixels = 1; pixels <= 200000; pixels += 1 + pixels / 7)
      for (int channels : channel_counts)
        for (int groups : {1, 2, channels / 2, channels})
          for (int dtype : {DR_FLOAT32, DR_FLOAT16})
            for (int images : {1, 2}) {
              if (groups < 1 || channels % groups != 0) continue;
              // Aligned and contiguous, a slice with an odd stride, and 4- or 8-byte vectors.
              const int widest = widest_vector(dtype), fold = folded_pixels(channels, dtype);
              if (!check(batch, pixels, channels, groups, dtype, channels + 1, {1, 1, false}, images))
                return 1;
              for (int vec : {2, 4, widest})
                if (channels % vec == 0 && vec <= widest &&
                    !check(batch, pixels, channels, groups, dtype, channels, {vec, 1, false}, images))
                  return 1;
              if (fold > 1 && pixels % fold == 0 && can_fold(pixels, channels, dtype) &&
                  !check(batch, pixels, channels, groups, dtype, channels, {widest, fold, false}, images))
                return 1;
            }
  std::printf("%lld plans\n", checked);
  return 0;
}
