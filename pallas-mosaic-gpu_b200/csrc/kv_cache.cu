// A paged cache of keys and values, [pages, kv_heads, page_size, head_dim]: writing new tokens into it and reading
// sequences out of it, as 16-bit numbers or as e4m3 codes with one power-of-two scale per (token, head).
//
//   e = the smallest whole number in [-64, 120] with max|x| <= 448 * 2^e,   code = e4m3(x * 2^-e),   x' = code * 2^e
// The scale is a power of two because a floating-point code loses nothing by that (its relative step is the same
// everywhere) and everything after the one rounding of 2^-4 is exact: the product with the scale, and the 16-bit number
// it gives.  A row with an infinity or NaN has exponent -128 and reads back as NaN throughout.
//
// Bound: HBM for long writes and reads, launch latency for single tokens.  head_dim / 8 lanes take a row, 16 bytes of
// 16-bit numbers a lane; a row's largest magnitude is an integer maximum over the lanes (bits of |x| order like |x|,
// NaN above infinity).
#include "host_common.cuh"
#include "ptx.cuh"

namespace splash {

constexpr int kCacheThreads = 256;
constexpr int kMinExponent = -64, kMaxExponent = 120, kBadExponent = -128;

// Slot of token `index` of sequence b for head h, in rows of the cache; -1 where the sequence has no such page.
__device__ __forceinline__ long long cache_row(const SplashCacheParams& p, int b, long long index, int h) {
  const long long entry = index / p.page_size;
  if (index < 0 || entry >= p.table_width) return -1;
  const int page = p.page_table[static_cast<long long>(b) * p.table_stride + entry];
  if (page < 0 || page >= p.num_pages) return -1;
  return (static_cast<long long>(page) * p.kv_heads + h) * p.page_size + (index - entry * p.page_size);
}

__device__ __forceinline__ float pow2(int e) {  // e in [-126, 127]
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Two f32 to two e4m3 codes, `lo` in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <bool BF16>
__device__ __forceinline__ float2 wide2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// LPR lanes per row of head_dim = 8 * LPR numbers; blockIdx.y: 0 keys, 1 values.
template <int LPR, bool BF16, bool QUANT>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const SplashCacheParams p) {
  const long long id = static_cast<long long>(blockIdx.x) * (kCacheThreads / LPR) + threadIdx.x / LPR;
  const int sub = threadIdx.x % LPR;
  const bool is_v = blockIdx.y != 0;
  const long long per_head = p.len;
  const long long bh = id / per_head;
  const int t = static_cast<int>(id - bh * per_head);
  const int b = static_cast<int>(bh / p.kv_heads);
  const int h = static_cast<int>(bh - static_cast<long long>(b) * p.kv_heads);
  bool live = b < p.batch;
  long long row = -1;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (live && (!p.counts || t < p.counts[b])) row = cache_row(p, b, static_cast<long long>(p.lengths[b]) + t, h);
  live = live && row >= 0;
  if (live) {
    const int64_t* st = is_v ? p.v_stride : p.k_stride;
    const uint16_t* src = static_cast<const uint16_t*>(is_v ? p.v : p.k) + b * st[0] + h * st[1] + t * st[2];
    x = *reinterpret_cast<const uint4*>(src + sub * 8);
  }
  if constexpr (!QUANT) {
    if (live) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + row * (16 * LPR) + sub * 16) = x;
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
#pragma unroll
    for (int d = LPR / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (!live) return;  // (after the shuffles, in which every lane of the warp takes part)
    const bool bad = top >= (BF16 ? 0x7f80u : 0x7c00u);
    int e = kMinExponent;
    if (top != 0) {
      const uint32_t bits = __float_as_uint(wide2<BF16>(top).x);
      // |x| = 1.f * 2^E: 448 = 1.75 * 2^8.
      e = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
      e = min(max(e, kMinExponent), kMaxExponent);
    }
    const float scale = pow2(-e);
    uint32_t code[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = wide2<BF16>(w[i]);
      code[i] = bad ? 0x7f7fu : to_e4m3x2(f.x * scale, f.y * scale);
    }
    uint8_t* dst = static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + row * (8 * LPR) + sub * 8;
    *reinterpret_cast<uint2*>(dst) = make_uint2(code[0] | (code[1] << 16), code[2] | (code[3] << 16));
    if (sub == 0) (is_v ? p.v_exponent : p.k_exponent)[row] = static_cast<int8_t>(bad ? kBadExponent : e);
  }
}

template <int LPR, bool BF16, bool QUANT>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const SplashCacheParams p) {
  const long long id = static_cast<long long>(blockIdx.x) * (kCacheThreads / LPR) + threadIdx.x / LPR;
  const int sub = threadIdx.x % LPR;
  const bool is_v = blockIdx.y != 0;
  const long long bh = id / p.len;
  const int t = static_cast<int>(id - bh * p.len);
  const int b = static_cast<int>(bh / p.kv_heads);
  const int h = static_cast<int>(bh - static_cast<long long>(b) * p.kv_heads);
  if (b >= p.batch) return;
  const long long row = t < p.lengths[b] ? cache_row(p, b, t, h) : -1;
  uint4 y = make_uint4(0, 0, 0, 0);
  if (row >= 0) {
    const uint8_t* src = static_cast<const uint8_t*>(is_v ? p.v_cache : p.k_cache);
    if constexpr (!QUANT) {
      y = *reinterpret_cast<const uint4*>(src + row * (16 * LPR) + sub * 16);
    } else {
      const uint2 c = *reinterpret_cast<const uint2*>(src + row * (8 * LPR) + sub * 8);
      const int e = (is_v ? p.v_exponent : p.k_exponent)[row];
      const float scale = e == kBadExponent ? __uint_as_float(0x7fc00000u) : pow2(e);
      uint32_t* w = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = from_e4m3x2(((i < 2 ? c.x : c.y) >> (16 * (i & 1))) & 0xffffu);
        w[i] = pack2<BF16>(f.x * scale, f.y * scale);
      }
    }
  }
  uint16_t* dst = static_cast<uint16_t*>(is_v ? p.v_out : p.k_out) + id * (8 * LPR) + sub * 8;
  *reinterpret_cast<uint4*>(dst) = y;
}

static int check_cache(const SplashCacheParams* p) {
  if (!p) return fail(SPLASH_INVALID_ARGUMENT, "params is null");
  if (p->dtype != SPLASH_DTYPE_BF16 && p->dtype != SPLASH_DTYPE_F16) return fail(SPLASH_UNSUPPORTED, "Only bf16/f16 are supported");
  if (p->head_dim != 64 && p->head_dim != 128) return fail(SPLASH_UNSUPPORTED, "the cache supports head dims 64 and 128");
  if (p->batch < 0 || p->len < 0 || p->kv_heads <= 0 || p->page_size <= 0 || p->num_pages < 0 || p->table_width < 0)
    return fail(SPLASH_INVALID_ARGUMENT, "sizes must not be negative");
  if (p->batch == 0 || p->len == 0) return SPLASH_OK;
  if (!p->k_cache || !p->v_cache || !p->lengths || (!p->page_table && p->table_width > 0))
    return fail(SPLASH_INVALID_ARGUMENT, "the cache, page_table and lengths must be non-null");
  if (p->quantized && (!p->k_exponent || !p->v_exponent)) return fail(SPLASH_INVALID_ARGUMENT, "an 8-bit cache needs its exponents");
  if ((reinterpret_cast<uintptr_t>(p->k_cache) | reinterpret_cast<uintptr_t>(p->v_cache)) & 15)
    return fail(SPLASH_INVALID_ARGUMENT, "the cache must be 16-byte aligned");
  return SPLASH_OK;
}

static int cache_grid(const SplashCacheParams& p, dim3& grid) {
  const long long rows = static_cast<long long>(p.batch) * p.kv_heads * p.len;
  const int per_block = kCacheThreads / (p.head_dim / 8);
  const long long blocks = (rows + per_block - 1) / per_block;
  if (blocks >= (1ll << 31)) return fail(SPLASH_INVALID_ARGUMENT, "too many tokens for one call");
  grid = dim3(static_cast<unsigned>(blocks), 2);
  return SPLASH_OK;
}

#define SPLASH_CACHE_LAUNCH(KERNEL)                                                                               \
  const bool bf16 = p->dtype == SPLASH_DTYPE_BF16;                                                                \
  auto kernel = p->head_dim == 64                                                                                 \
                    ? (p->quantized ? (bf16 ? KERNEL<8, true, true> : KERNEL<8, false, true>)                     \
                                    : (bf16 ? KERNEL<8, true, false> : KERNEL<8, false, false>))                  \
                    : (p->quantized ? (bf16 ? KERNEL<16, true, true> : KERNEL<16, false, true>)                   \
                                    : (bf16 ? KERNEL<16, true, false> : KERNEL<16, false, false>));               \
  kernel<<<grid, kCacheThreads, 0, static_cast<cudaStream_t>(stream)>>>(*p);                                      \
  SPLASH_CUDA_CHECK(cudaGetLastError());                                                                          \
  return SPLASH_OK

}  // namespace splash

using namespace splash;

extern "C" int splash_cache_write(const SplashCacheParams* p, void* stream) {
  if (int rc = check_cache(p)) return rc;
  if (p->batch == 0 || p->len == 0) return SPLASH_OK;
  if (!p->k || !p->v) return fail(SPLASH_INVALID_ARGUMENT, "k and v must be non-null");
  for (int i = 0; i < 3; ++i)
    if (p->k_stride[i] % 8 || p->v_stride[i] % 8) return fail(SPLASH_INVALID_ARGUMENT, "rows of k and v must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15)
    return fail(SPLASH_INVALID_ARGUMENT, "rows of k and v must be 16-byte aligned");
  dim3 grid;
  if (int rc = cache_grid(*p, grid)) return rc;
  SPLASH_CACHE_LAUNCH(cache_write_kernel);
}

extern "C" int splash_cache_read(const SplashCacheParams* p, void* stream) {
  if (int rc = check_cache(p)) return rc;
  if (p->batch == 0 || p->len == 0) return SPLASH_OK;
  if (!p->k_out || !p->v_out) return fail(SPLASH_INVALID_ARGUMENT, "k_out and v_out must be non-null");
  if ((reinterpret_cast<uintptr_t>(p->k_out) | reinterpret_cast<uintptr_t>(p->v_out)) & 15)
    return fail(SPLASH_INVALID_ARGUMENT, "the results must be 16-byte aligned");
  dim3 grid;
  if (int rc = cache_grid(*p, grid)) return rc;
  SPLASH_CACHE_LAUNCH(cache_read_kernel);
}
