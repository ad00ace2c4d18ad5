// Host launcher of the attention over a paged cache; included by the translation units that instantiate it.
#pragma once

#include "cached_dispatch.h"
#include "cached_few_kernel.cuh"
#include "cached_kernel.cuh"
#include "host_common.cuh"

namespace splash {

template <class L, int D, bool QUANT, int Q_ROWS, typename Kernel>
int launch_cached_kernel(Kernel kernel, const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream) {
  CUtensorMap tm_q, tm_k, tm_v;
  int rc;
  const uint64_t kv_rows = static_cast<uint64_t>(p.num_pages) * p.kv_heads * p.page_size;
  const uint32_t box_rows = p.page_size < kCachedTile ? p.page_size : kCachedTile;
  const CUtensorMapDataType dt = QUANT ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : tmap_dtype(p.dtype);
  const CUtensorMapSwizzle swz = L::kBoxBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if ((rc = make_tmap_2d(&tm_k, p.k_cache, dt, L::kItem, kv_rows, D, box_rows, L::kBoxElems, swz))) return rc;
  if ((rc = make_tmap_2d(&tm_v, p.v_cache, dt, L::kItem, kv_rows, D, box_rows, L::kBoxElems, swz))) return rc;
  if (QUANT) tm_q = tm_k;  // (Q is read and split by a warp)
  else if ((rc = make_tmap_2d(&tm_q, p.q, dt, 2, static_cast<uint64_t>(p.batch) * p.heads * p.n, D, Q_ROWS, 64, swz))) return rc;
  if ((rc = opt_in_smem(kernel, L::kSmem))) return rc;
  kernel<<<plan.ctas, kCachedThreads, L::kSmem, stream>>>(tm_q, tm_k, tm_v, a);
  SPLASH_CUDA_CHECK(cudaGetLastError());
  return SPLASH_OK;
}

template <int D, bool BF16, bool QUANT, int KG>
int launch_cached_form(const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream) {
  using L = CachedLayout<D, BF16, QUANT, KG>;
  return launch_cached_kernel<L, D, QUANT, L::kRows>(cached_kernel<D, BF16, QUANT, KG>, p, plan, a, stream);
}

template <int D, bool BF16, bool QUANT, int R>
int launch_cached_few(const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream) {
  using L = CachedFewLayout<D, BF16, QUANT, R>;
  return launch_cached_kernel<L, D, QUANT, R>(cached_few_kernel<D, BF16, QUANT, R>, p, plan, a, stream);
}

template <int D, bool BF16>
int launch_cached(const SplashCachedParams& p, const CachedPlan& plan, const CachedArgs& a, cudaStream_t stream) {
  if (p.quantized) {
    if (plan.row_cap == 8) return launch_cached_few<D, BF16, true, 8>(p, plan, a, stream);
    if (plan.row_cap == 16) return launch_cached_few<D, BF16, true, 16>(p, plan, a, stream);
    if (plan.row_cap == 32) return launch_cached_form<D, BF16, true, 4>(p, plan, a, stream);
    if (plan.row_cap == 64) return launch_cached_form<D, BF16, true, 2>(p, plan, a, stream);
    return launch_cached_form<D, BF16, true, 1>(p, plan, a, stream);
  }
  if (plan.row_cap == 16) return launch_cached_few<D, BF16, false, 16>(p, plan, a, stream);
  if (plan.row_cap == 32) return launch_cached_form<D, BF16, false, 4>(p, plan, a, stream);
  if (plan.row_cap == 64) return launch_cached_form<D, BF16, false, 2>(p, plan, a, stream);
  return launch_cached_form<D, BF16, false, 1>(p, plan, a, stream);
}

}  // namespace splash
