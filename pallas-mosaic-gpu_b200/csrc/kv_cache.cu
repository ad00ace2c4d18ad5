// A paged cache of keys and values, [pages, kv_heads, page_size, head_dim]: writing new tokens into it and reading
// sequences out of it, as 16-bit numbers or as e4m3 codes with one power-of-two scale per (token, head).
//
//   e = the smallest whole number in [-64, 120] with max|x| <= 448 * 2^e,   code = e4m3(x * 2^-e),   x' = code * 2^e
// The scale is a power of two because a floating-point code loses nothing by that (its relative step is the same
// everywhere) and everything after the one rounding of 2^-4 is exact: the product with the scale, and the 16-bit number
// it gives, but at the ends of the types: f16's subnormals are rounded once more, and what was rounded up to 2^16 (f16) or 2^128
// (bf16) reads as infinity.  A row with an infinity or NaN has exponent -128 and reads back as NaN throughout.
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

// A block has ROWS * 256 / LPR consecutive tokens of one (sequence, head), LPR lanes per row of head_dim = 8 * LPR numbers and
// ROWS rows of a thread in flight together; blockIdx.y: 0 keys, 1 values.
struct CacheBlock {
  int b, h, t0;  // t0: first token of this thread
};
template <int LPR, int ROWS>
__device__ __forceinline__ CacheBlock cache_block(const SplashCacheParams& p) {
  constexpr int kTokens = ROWS * kCacheThreads / LPR;
  const int chunks = (p.len + kTokens - 1) / kTokens;
  const int bh = blockIdx.x / chunks, chunk = blockIdx.x - bh * chunks;
  const int b = bh / p.kv_heads;
  return {b, bh - b * p.kv_heads, chunk * kTokens + static_cast<int>(threadIdx.x) / LPR};
}

template <int LPR, int ROWS, bool BF16, bool QUANT>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const SplashCacheParams p) {
  constexpr int kStep = kCacheThreads / LPR;
  const CacheBlock at = cache_block<LPR, ROWS>(p);
  const int sub = threadIdx.x % LPR;
  const bool is_v = blockIdx.y != 0;
  const int count = p.counts ? min(p.counts[at.b], p.len) : p.len;
  if (at.t0 - static_cast<int>(threadIdx.x) / LPR >= count) return;  // the whole block
  const long long start = p.lengths[at.b];
  const int64_t* st = is_v ? p.v_stride : p.k_stride;
  const uint16_t* src = static_cast<const uint16_t*>(is_v ? p.v : p.k) + at.b * st[0] + at.h * st[1] + sub * 8;
  long long row[ROWS];
  uint4 x[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int t = at.t0 + i * kStep;
    x[i] = make_uint4(0, 0, 0, 0);
    row[i] = -1;
    if (t < count) {
      x[i] = *reinterpret_cast<const uint4*>(src + t * st[2]);
      row[i] = cache_row(p, at.b, start + t, at.h);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if constexpr (!QUANT) {
      if (row[i] >= 0) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + row[i] * (16 * LPR) + sub * 16) = x[i];
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[i]);
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
#pragma unroll
      for (int d = LPR / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      if (row[i] < 0) continue;  // (after the shuffles, in which every lane of the warp takes part)
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
      for (int k = 0; k < 4; ++k) {
        const float2 f = wide2<BF16>(w[k]);
        code[k] = bad ? 0x7f7fu : to_e4m3x2(f.x * scale, f.y * scale);
      }
      uint8_t* dst = static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + row[i] * (8 * LPR) + sub * 8;
      *reinterpret_cast<uint2*>(dst) = make_uint2(code[0] | (code[1] << 16), code[2] | (code[3] << 16));
      if (sub == 0) (is_v ? p.v_exponent : p.k_exponent)[row[i]] = static_cast<int8_t>(bad ? kBadExponent : e);
    }
  }
}

template <int LPR, int ROWS, bool BF16, bool QUANT>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const SplashCacheParams p) {
  constexpr int kStep = kCacheThreads / LPR;
  const CacheBlock at = cache_block<LPR, ROWS>(p);
  const int sub = threadIdx.x % LPR;
  const bool is_v = blockIdx.y != 0;
  const int count = min(p.lengths[at.b], p.len);
  const uint8_t* src = static_cast<const uint8_t*>(is_v ? p.v_cache : p.k_cache);
  const int8_t* exponents = is_v ? p.v_exponent : p.k_exponent;
  uint4 y[ROWS];  // 8 bit: the codes in the first half, their exponent in z
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int t = at.t0 + i * kStep;
    const long long row = t < count ? cache_row(p, at.b, t, at.h) : -1;
    y[i] = make_uint4(0, 0, 0, 0);
    if (row < 0) continue;
    if constexpr (!QUANT) {
      y[i] = *reinterpret_cast<const uint4*>(src + row * (16 * LPR) + sub * 16);
    } else {
      const uint2 c = *reinterpret_cast<const uint2*>(src + row * (8 * LPR) + sub * 8);
      y[i] = make_uint4(c.x, c.y, static_cast<uint32_t>(static_cast<int32_t>(exponents[row])), 0);
    }
  }
  uint16_t* dst = static_cast<uint16_t*>(is_v ? p.v_out : p.k_out) +
                  (static_cast<long long>(at.b) * p.kv_heads + at.h) * p.len * (8 * LPR) + sub * 8;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int t = at.t0 + i * kStep;
    if (t >= p.len) continue;
    if constexpr (QUANT) {
      const int e = static_cast<int32_t>(y[i].z);
      const float scale = e == kBadExponent ? __uint_as_float(0x7fc00000u) : pow2(e);
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = from_e4m3x2(((k < 2 ? y[i].x : y[i].y) >> (16 * (k & 1))) & 0xffffu);
        w[k] = pack2<BF16>(f.x * scale, f.y * scale);
      }
      y[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(dst + static_cast<long long>(t) * (8 * LPR)) = y[i];
  }
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

// Eight rows of a thread in flight where there are enough tokens (4 prompts of up to 8192 tokens, 8 bit: DRAM latency
// bounds one row a thread, 46 us), one where a call is short.
constexpr int kCacheRows = 8;

template <int LPR, int ROWS>
static int cache_blocks(const SplashCacheParams& p) {
  constexpr int kTokens = ROWS * kCacheThreads / LPR;
  return (p.len + kTokens - 1) / kTokens;
}

template <int LPR, int ROWS, bool WRITE>
static int launch_cache(const SplashCacheParams& p, cudaStream_t stream) {
  const long long blocks = static_cast<long long>(cache_blocks<LPR, ROWS>(p)) * p.batch * p.kv_heads;
  if (blocks >= (1ll << 31)) return fail(SPLASH_INVALID_ARGUMENT, "too many tokens for one call");
  const bool bf16 = p.dtype == SPLASH_DTYPE_BF16;
  auto kernel = WRITE ? (p.quantized ? (bf16 ? cache_write_kernel<LPR, ROWS, true, true> : cache_write_kernel<LPR, ROWS, false, true>)
                                     : (bf16 ? cache_write_kernel<LPR, ROWS, true, false> : cache_write_kernel<LPR, ROWS, false, false>))
                      : (p.quantized ? (bf16 ? cache_read_kernel<LPR, ROWS, true, true> : cache_read_kernel<LPR, ROWS, false, true>)
                                     : (bf16 ? cache_read_kernel<LPR, ROWS, true, false> : cache_read_kernel<LPR, ROWS, false, false>));
  kernel<<<dim3(static_cast<unsigned>(blocks), 2), kCacheThreads, 0, stream>>>(p);
  SPLASH_CUDA_CHECK(cudaGetLastError());
  return SPLASH_OK;
}

template <int LPR, bool WRITE>
static int run_cache_dim(const SplashCacheParams& p, cudaStream_t st) {
  const bool many = p.len > kCacheThreads / LPR &&
                    static_cast<long long>(cache_blocks<LPR, kCacheRows>(p)) * p.batch * p.kv_heads >= sm_count();
  return many ? launch_cache<LPR, kCacheRows, WRITE>(p, st) : launch_cache<LPR, 1, WRITE>(p, st);
}

template <bool WRITE>
static int run_cache(const SplashCacheParams& p, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p.head_dim == 64 ? run_cache_dim<8, WRITE>(p, st) : run_cache_dim<16, WRITE>(p, st);
}

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
  return run_cache<true>(*p, stream);
}

extern "C" int splash_cache_read(const SplashCacheParams* p, void* stream) {
  if (int rc = check_cache(p)) return rc;
  if (p->batch == 0 || p->len == 0) return SPLASH_OK;
  if (!p->k_out || !p->v_out) return fail(SPLASH_INVALID_ARGUMENT, "k_out and v_out must be non-null");
  if ((reinterpret_cast<uintptr_t>(p->k_out) | reinterpret_cast<uintptr_t>(p->v_out)) & 15)
    return fail(SPLASH_INVALID_ARGUMENT, "the results must be 16-byte aligned");
  return run_cache<false>(*p, stream);
}
