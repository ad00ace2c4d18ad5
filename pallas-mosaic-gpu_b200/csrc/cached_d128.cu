#include "cached_launch.cuh"

namespace splash {
template int launch_cached<128, true>(const SplashCachedParams&, const CachedPlan&, const CachedArgs&, cudaStream_t);
template int launch_cached<128, false>(const SplashCachedParams&, const CachedPlan&, const CachedArgs&, cudaStream_t);
}  // namespace splash
