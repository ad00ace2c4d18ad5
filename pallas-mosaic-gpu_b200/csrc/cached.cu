// Entry points of the attention over a paged cache, and its second pass.
#include "cached_dispatch.h"
#include "cached_kernel.cuh"
#include "host_common.cuh"

namespace splash {

// Second pass: units that several CTAs shared,
//   m = max_i m_i, w_i = 2^(m_i - m), l = sum_i w_i l_i, out = sum_i w_i O_i / l, lse = (m + log2 l) ln 2,
// and zeros for units whose rows see no key at all.  One block per unit (most have nothing to do and leave), one warp per
// row, the parts in the order of the keys.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) cached_finish_kernel(const CachedArgs a, int grid) {
  if (a.status[0] != 0) return;  // a wait ran out: the parts are not to be read
  const int unit = blockIdx.x;
  const int entry = unit / a.kv_heads, head = unit - entry * a.kv_heads;
  const int begin = a.starts[entry], all = a.starts[entry + 1] - begin, total = a.starts[a.batch * a.row_tiles];
  const int tiles = all / a.kv_heads, ctas = min(grid, total);
  const int us = begin + head * tiles, ue = us + tiles;
  int c0 = 0, c1 = -1;
  if (tiles > 0) {
    // The CTA whose share holds tile x: the last c with floor(c * total / ctas) <= x.
    c0 = static_cast<int>(((us + 1ll) * ctas - 1) / total);
    c1 = static_cast<int>((static_cast<long long>(ue) * ctas - 1) / total);
    if (c0 == c1) return;
  }
  const int b = entry / a.row_tiles, rt = entry - b * a.row_tiles;
  const int rows = min(a.row_cap, a.rows - rt * a.row_cap);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = cached_geom(a, entry).count;
  const long long row0 = static_cast<long long>(b * a.kv_heads + head) * a.rows + rt * a.row_cap;
  for (int r = warp; r < rows; r += 8) {
    const bool live = (rt * a.row_cap + r) % a.n < count;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live && tiles > 0) {
      auto part = [&](int c) {
        return (2ll * c + (cached_share(c, total, ctas) < us ? 1 : 0)) * a.row_cap + r;
      };
      for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, a.part_ml[part(c)].x);
#pragma unroll
      for (int d = 16; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
#pragma unroll 4
      for (int c = c0; c <= c1; ++c) {
        const long long at = part(c);
        const float2 ml = a.part_ml[at];
        const float w = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : ex2_approx(ml.x - m);  // (a NaN sum stays one)
        if (lane < D / 4) {
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * D + lane * 4);
          o.x = fmaf(x.x, w, o.x);
          o.y = fmaf(x.y, w, o.y);
          o.z = fmaf(x.z, w, o.z);
          o.w = fmaf(x.w, w, o.w);
        }
        l = fmaf(ml.y, w, l);
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    if (lane < D / 4)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (row0 + r) * D + lane * 4) =
          make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
    if (a.lse_out && lane == 0) a.lse_out[row0 + r] = l != 0.f ? (m + lg2_approx(l)) * kCachedLn2 : a.mask_value;
  }
}

static int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

static int check_cached(const SplashCachedParams* p) {
  if (!p) return fail(SPLASH_INVALID_ARGUMENT, "params is null");
  if (p->dtype != SPLASH_DTYPE_BF16 && p->dtype != SPLASH_DTYPE_F16) return fail(SPLASH_UNSUPPORTED, "Only bf16/f16 are supported");
  if (p->head_dim != 64 && p->head_dim != 128) return fail(SPLASH_UNSUPPORTED, "attention over the cache supports head dims 64 and 128");
  if (p->batch <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->n <= 0 || p->num_pages <= 0 || p->table_width < 0)
    return fail(SPLASH_INVALID_ARGUMENT, "sizes must be positive");
  if (p->heads % p->kv_heads) return fail(SPLASH_INVALID_ARGUMENT, "heads not a multiple of kv_heads");
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128 && p->page_size != 256)
    return fail(SPLASH_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256");
  if (p->parents && p->n > kCachedMaxTree) return fail(SPLASH_UNSUPPORTED, "a tree has at most 128 nodes");
  if (p->num_sinks < 0) return fail(SPLASH_INVALID_ARGUMENT, "num_sinks must not be negative");
  const int64_t limit = 1ll << 31;
  const int64_t rows = static_cast<int64_t>(p->heads / p->kv_heads) * p->n;
  const int64_t capacity = static_cast<int64_t>(p->table_width) * p->page_size;
  if (static_cast<int64_t>(p->num_pages) * p->kv_heads * p->page_size >= limit)
    return fail(SPLASH_INVALID_ARGUMENT, "num_pages * kv_heads * page_size must fit in 31 bits");
  if (capacity >= (1ll << 30)) return fail(SPLASH_INVALID_ARGUMENT, "a page table may hold at most 2^30 tokens");
  if (rows >= (1ll << 30) || static_cast<int64_t>(p->batch) * p->kv_heads * rows >= limit)
    return fail(SPLASH_INVALID_ARGUMENT, "batch * heads * new tokens must fit in 31 bits");
  const int64_t units = (rows + 31) / 32 * p->batch * p->kv_heads;
  if (units * (capacity / kCachedTile + 2) >= limit)
    return fail(SPLASH_INVALID_ARGUMENT, "batch * kv heads * tiles of rows * tiles of keys must fit in 31 bits");
  return SPLASH_OK;
}

// Rows per tile: as few as hold the call's, since the other copies of few rows share the softmax (see the kernel).
static CachedPlan cached_plan(const SplashCachedParams& p) {
  CachedPlan plan;
  const int64_t rows = static_cast<int64_t>(p.heads / p.kv_heads) * p.n;
  plan.row_cap = rows <= 32 ? 32 : (rows <= 64 || p.quantized) ? 64 : 128;
  plan.row_tiles = static_cast<int>((rows + plan.row_cap - 1) / plan.row_cap);
  const int64_t entries = static_cast<int64_t>(p.batch) * plan.row_tiles;
  const int64_t capacity = static_cast<int64_t>(p.table_width) * p.page_size;
  const int64_t most = entries * p.kv_heads * ((capacity + kCachedTile - 1) / kCachedTile);  // tiles there can be
  plan.ctas = static_cast<int>(most < 1 ? 1 : most < sm_count() ? most : sm_count());
  plan.part_o = round16((entries + 1) * 4);
  plan.part_ml = plan.part_o + static_cast<int64_t>(2) * plan.ctas * plan.row_cap * p.head_dim * 4;
  plan.bytes = plan.part_ml + static_cast<int64_t>(2) * plan.ctas * plan.row_cap * 8;
  return plan;
}

}  // namespace splash

using namespace splash;

extern "C" int64_t splash_cached_workspace_bytes(const SplashCachedParams* p) {
  return check_cached(p) ? 0 : cached_plan(*p).bytes;
}

extern "C" int splash_cached_fwd(const SplashCachedParams* p, void* workspace, int64_t bytes, void* stream) {
  if (int rc = check_cached(p)) return rc;
  if (!p->q || !p->k_cache || !p->v_cache || !p->lengths || !p->out || !p->status || (!p->page_table && p->table_width > 0))
    return fail(SPLASH_INVALID_ARGUMENT, "q, the cache, page_table, lengths, out and status must be non-null");
  if (p->quantized && (!p->k_exponent || !p->v_exponent)) return fail(SPLASH_INVALID_ARGUMENT, "an 8-bit cache needs its exponents");
  if ((reinterpret_cast<uintptr_t>(p->k_exponent) | reinterpret_cast<uintptr_t>(p->v_exponent) |
       reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out)) & 15)
    return fail(SPLASH_INVALID_ARGUMENT, "q, out and the exponents must be 16-byte aligned");
  const CachedPlan plan = cached_plan(*p);
  if (!workspace || bytes < plan.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(SPLASH_INVALID_ARGUMENT, "the workspace is null, too small or not 16-byte aligned");
  CachedArgs a;
  a.q = p->q;
  a.k_exponent = p->k_exponent;
  a.v_exponent = p->v_exponent;
  a.page_table = p->page_table;
  a.lengths = p->lengths;
  a.counts = p->counts;
  a.parents = p->parents;
  a.out = p->out;
  a.lse_out = p->lse_out;
  a.status = p->status;
  a.starts = static_cast<int32_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.part_o);
  a.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + plan.part_ml);
  a.table_stride = p->table_stride;
  a.parents_stride = p->parents_stride;
  a.batch = p->batch;
  a.heads = p->heads;
  a.kv_heads = p->kv_heads;
  a.n = p->n;
  a.rows = p->heads / p->kv_heads * p->n;
  a.row_tiles = plan.row_tiles;
  a.row_cap = plan.row_cap;
  a.num_pages = p->num_pages;
  a.page_size = p->page_size;
  a.table_width = p->table_width;
  a.window = p->window_left < 0 ? -1 : p->window_left < (1 << 30) ? p->window_left : (1 << 30);
  a.sinks = p->num_sinks < (1 << 30) ? p->num_sinks : (1 << 30);
  a.mask_value = p->mask_value;
  a.soft_cap = p->soft_cap;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = p->dtype == SPLASH_DTYPE_BF16;
  const int rc = p->head_dim == 64 ? (bf16 ? launch_cached<64, true>(*p, plan, a, st) : launch_cached<64, false>(*p, plan, a, st))
                                   : (bf16 ? launch_cached<128, true>(*p, plan, a, st) : launch_cached<128, false>(*p, plan, a, st));
  if (rc) return rc;
  auto finish = p->head_dim == 64 ? (bf16 ? cached_finish_kernel<64, true> : cached_finish_kernel<64, false>)
                                  : (bf16 ? cached_finish_kernel<128, true> : cached_finish_kernel<128, false>);
  finish<<<static_cast<unsigned>(static_cast<int64_t>(p->batch) * plan.row_tiles * p->kv_heads), 256, 0, st>>>(a, plan.ctas);
  SPLASH_CUDA_CHECK(cudaGetLastError());
  return SPLASH_OK;
}
