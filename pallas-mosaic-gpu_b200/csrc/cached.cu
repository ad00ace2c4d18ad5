// Entry points of the attention over a paged cache, and its second pass.
#include "cached_dispatch.h"
#include "cached_common.cuh"
#include "host_common.cuh"

namespace splash {

// Second pass: units that several CTAs shared,
//   m = max_i m_i, w_i = 2^(m_i - m), l = sum_i w_i l_i, out = sum_i w_i O_i / l, lse = (m + log2 l) ln 2.
// A block per cut between two CTAs and 8 rows; the first cut of a unit has the work, the parts in the order of the keys,
// a warp per row.  Bound by latency: the weights of up to 32 parts come first, a lane each, then the rows of O together.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) cached_finish_kernel(const CachedArgs a, int ctas) {
  wait_for_prerequisites();
  const int c = blockIdx.x + 1, lane = threadIdx.x & 31;
  const int4 before = a.cuts[c - 1], cut = a.cuts[c];
  if (a.status[0] != 0) return;  // a wait ran out: the parts are not to be read
  if (cut.x < 0 || cut.z == 0) return;  // no unit goes on here
  const bool same = before.x == cut.x && before.y == cut.y;
  if (same && before.z > 0) return;     // not its first cut
  int last = c;  // the CTA that has the unit's end
  for (int c0 = c + 1; c0 < ctas; c0 += 32) {
    bool goes_on = false;
    if (c0 + lane < ctas) {
      const int4 x = a.cuts[c0 + lane];
      goes_on = x.x == cut.x && x.y == cut.y && x.z > 0;
    }
    const uint32_t ends = ~__ballot_sync(0xffffffffu, goes_on);
    if (ends) {
      last = c0 + __ffs(ends) - 2;
      break;
    }
    last = c0 + 31;
  }
  const int b = cut.x / a.row_tiles, rt = cut.x - b * a.row_tiles;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (r >= min(a.row_cap, a.rows - rt * a.row_cap)) return;
  const long long row = static_cast<long long>(b * a.kv_heads + cut.y) * a.rows + rt * a.row_cap + r;
  const bool live = (rt * a.row_cap + r) % a.n < cached_geom(a, cut.x).count;
  const int parts = last - c + 2;
  // Where part i lies: what CTA c - 1 began is its first or its last segment, the others' are their first.
  auto place = [&](int i) { return (2ll * (c - 1 + i) + (i == 0 && !same ? 1 : 0)) * a.row_cap + r; };
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    for (int i0 = 0; i0 < parts; i0 += 32) {
      const int n = min(32, parts - i0);
      const float2 ml = lane < n ? a.part_ml[place(i0 + lane)] : make_float2(-INFINITY, 0.f);
      float top = ml.x;
#pragma unroll
      for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float m_new = fmaxf(m, top);
      const float scale = m == -INFINITY ? (l == l ? 0.f : l) : ex2_approx(m - m_new);  // (a NaN sum stays one)
      float w = ml.x == -INFINITY ? (ml.y == ml.y ? 0.f : ml.y) : ex2_approx(ml.x - m_new);
      float sum = ml.y * w;
#pragma unroll
      for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      m = m_new;
      l = l * scale + sum;
      o.x *= scale; o.y *= scale; o.z *= scale; o.w *= scale;
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        if (lane < D / 4) {
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + place(i0 + i) * D + lane * 4);
          o.x = fmaf(x.x, wi, o.x);
          o.y = fmaf(x.y, wi, o.y);
          o.z = fmaf(x.z, wi, o.z);
          o.w = fmaf(x.w, wi, o.w);
        }
      }
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  if (lane < D / 4)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * D + lane * 4) =
        make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
  if (a.lse_out && lane == 0) a.lse_out[row] = l != 0.f ? (m + lg2_approx(l)) * kCachedLn2 : a.mask_value;
}

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
  const int64_t units = (rows + 7) / 8 * p->batch * p->kv_heads;
  if (units * (capacity / kCachedTile + 2 + kCachedMostUnitCost) >= limit)
    return fail(SPLASH_INVALID_ARGUMENT, "batch * kv heads * tiles of rows * tiles of keys must fit in 31 bits");
  return SPLASH_OK;
}

// Rows per tile: as few as hold the call's.  8-bit caches take the kernel whose MMA rows are keys (cached_few_kernel.cuh) with up
// to 16 rows, above which the other (cached_kernel.cuh) has at most 4 copies.  us with 16 rows in bf16, few | copies, from L2
// flushed: 32 sequences of 8192 keys, 8 kv heads 129 | 170 (head_dim 64: 115 | 141), 64 of 100 to 3000 keys 86 | 98 (78 | 82),
// 64 windows of 4096 keys with a soft-cap 160 | 186.
static CachedPlan cached_plan(const SplashCachedParams& p) {
  CachedPlan plan;
  const int64_t rows = static_cast<int64_t>(p.heads / p.kv_heads) * p.n;
  const int64_t capacity = static_cast<int64_t>(p.table_width) * p.page_size;
  const bool few = p.quantized && rows <= 16;
  plan.row_cap = few ? (rows <= 8 ? 8 : 16) : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  // A unit stands in the line by as many tiles more as its start and the sum of its parts take.  us for 64 sequences of 100 to
  // 3000 keys, 8 kv heads, head_dim 128, with a cost of 2 | 4 | 8 | 12: 4 rows 80 | 80 | 82 | 86, 128 rows 138 | 124 | 113 |
  // 113; 8 bit, with L2 flushed: 4 rows 78 | 68 | 67 | 70 (6: 66), 16 rows 100 | 90 | 82 | 84 (6: 84), 32 rows 109 | 98 | 100 | 109,
  // 64 rows 162 | 139 | 135 | 141, 128 rows 277 | 238 | 229 | 238.  Contexts of 8192 keys and more move by 3 % at most.
  plan.unit_cost = plan.row_cap == 128 || (p.quantized && plan.row_cap == 64) ? 8 : few ? 6 : 4;
  plan.row_tiles = static_cast<int>((rows + plan.row_cap - 1) / plan.row_cap);
  const int64_t entries = static_cast<int64_t>(p.batch) * plan.row_tiles;
  const int64_t most = entries * p.kv_heads * ((capacity + kCachedTile - 1) / kCachedTile);  // tiles there can be
  plan.ctas = static_cast<int>(most < 1 ? 1 : most < sm_count() ? most : sm_count());
  plan.part_o = static_cast<int64_t>(plan.ctas) * 16;
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
  a.status_host = p->status_host;
  a.cuts = static_cast<int4*>(workspace);
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
  a.unit_cost = plan.unit_cost;
  a.num_pages = p->num_pages;
  for (a.page_shift = 4; (1 << a.page_shift) < p->page_size; ++a.page_shift) {}
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
  if (plan.ctas == 1) return SPLASH_OK;  // nothing is cut
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(plan.ctas - 1, ((a.rows < plan.row_cap ? a.rows : plan.row_cap) + 7) / 8);
  config.blockDim = dim3(256);
  config.stream = st;
  cudaLaunchAttribute dependent[1];
  dependent[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  dependent[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = dependent;
  config.numAttrs = 1;
  SPLASH_CUDA_CHECK(cudaLaunchKernelEx(&config, finish, a, plan.ctas));
  SPLASH_CUDA_CHECK(cudaGetLastError());
  return SPLASH_OK;
}
