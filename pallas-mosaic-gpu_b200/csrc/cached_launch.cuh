// Host launcher of the attention over a paged cache; included by the translation units that instantiate it.
#pragma once

#include "cached_dispatch.h"
#include "cached_few_kernel.cuh"
#include "cached_kernel.cuh"
#include "host_common.cuh"

namespace splash {

// Maps of the cache, and a kernel's room.
template <class L, int D, typename Kernel>
int cached_maps(Kernel kernel, const SplashCachedParams& p, CUtensorMap& tm_k, CUtensorMap& tm_v) {
  const uint64_t kv_rows = static_cast<uint64_t>(p.num_pages) * p.kv_heads * p.page_size;
  const uint32_t box_rows = p.page_size < kCachedTile ? p.page_size : kCachedTile;
  const CUtensorMapDataType dt = p.quantized ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : tmap_dtype(p.dtype);
  const CUtensorMapSwizzle swz = L::kBoxBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (int rc = make_tmap_2d(&tm_k, p.k_cache, dt, L::kItem, kv_rows, D, box_rows, L::kBoxElems, swz)) return rc;
  if (int rc = make_tmap_2d(&tm_v, p.v_cache, dt, L::kItem, kv_rows, D, box_rows, L::kBoxElems, swz)) return rc;
  return opt_in_smem(kernel, L::kSmem);
}

template <int D, bool BF16, bool QUANT, int KG>
int launch_cached_form(const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream) {
  using L = CachedLayout<D, BF16, QUANT, KG>;
  auto kernel = cached_kernel<D, BF16, QUANT, KG>;
  CUtensorMap tm_q, tm_k, tm_v;
  if (int rc = cached_maps<L, D>(kernel, p, tm_k, tm_v)) return rc;
  if (QUANT) tm_q = tm_k;  // (Q is read and split by a warp)
  else if (int rc = make_tmap_2d(&tm_q, p.q, tmap_dtype(p.dtype), 2, static_cast<uint64_t>(p.batch) * p.heads * p.n, D, L::kRows, 64,
                                 CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  kernel<<<plan.ctas, kCachedThreads, L::kSmem, stream>>>(tm_q, tm_k, tm_v, a);
  SPLASH_CUDA_CHECK(cudaGetLastError());
  return SPLASH_OK;
}

template <int D, bool BF16, int R>
int launch_cached_few(const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream) {
  using L = CachedFewLayout<D, BF16, R>;
  auto kernel = cached_few_kernel<D, BF16, R>;
  CUtensorMap tm_k, tm_v;
  if (int rc = cached_maps<L, D>(kernel, p, tm_k, tm_v)) return rc;
  kernel<<<plan.ctas, kCachedThreads, L::kSmem, stream>>>(tm_k, tm_v, a);
  SPLASH_CUDA_CHECK(cudaGetLastError());
  return SPLASH_OK;
}

template <int D, bool BF16>
int launch_cached(const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream) {
  if (p.quantized) {
    if (plan.row_cap == 8) return launch_cached_few<D, BF16, 8>(p, plan, a, stream);
    if (plan.row_cap == 16) return launch_cached_few<D, BF16, 16>(p, plan, a, stream);
    if (plan.row_cap == 32) return launch_cached_form<D, BF16, true, 4>(p, plan, a, stream);
    if (plan.row_cap == 64) return launch_cached_form<D, BF16, true, 2>(p, plan, a, stream);
    return launch_cached_form<D, BF16, true, 1>(p, plan, a, stream);
  }
  if (plan.row_cap == 32) return launch_cached_form<D, BF16, false, 4>(p, plan, a, stream);
  if (plan.row_cap == 64) return launch_cached_form<D, BF16, false, 2>(p, plan, a, stream);
  return launch_cached_form<D, BF16, false, 1>(p, plan, a, stream);
}

}  // namespace splash
