// What the launchers of the attention over a paged cache share.
#pragma once

#include <cuda_runtime.h>

#include "../../include/splash_sm100.h"

namespace splash {

struct CachedArgs;

// How a call is cut: rows per tile, tiles of rows per (sequence, kv head), CTAs, cost of a unit in tiles, and where the workspace's parts begin.
struct CachedPlan {
  int row_cap, row_tiles, ctas, unit_cost;
  int64_t part_o, part_ml, bytes;
};

template <int D, bool BF16>
int launch_cached(const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream);

}  // namespace splash
