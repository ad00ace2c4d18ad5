#include "cached_launch.cuh"

namespace splash {
template int launch_cached<64, true>(const SplashCachedParams&, const CachedPlan&, const CachedArgs&, cudaStream_t);
template int launch_cached<64, false>(const SplashCachedParams&, const CachedPlan&, const CachedArgs&, cudaStream_t);
}  // namespace splash
