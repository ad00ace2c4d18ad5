// Rotary positions with several axes, forward and backward.
//
// Pair i of a row of x turns by theta_i = pos[axis(i)] * f_i:
//   (a, b) -> scale * (a cos - b sin, b cos + a sin),        backward: the same with -sin.
// The angle is kept in turns as a 64-bit fixed-point fraction: f_i / 2 pi rounded to 2^-64, times the whole position,
// modulo 2^64.  The wrap of the product is the range reduction, so an angle is off by at most |pos| 2^-65 turns (and
// 2^-25 half turns from the conversion to f32, which is more up to positions of 2^39); sin and cos are then CUDA's sincospif.
//
// Bound: HBM, each number read and written once.  A thread holds the sines of VEC pairs of one position and takes
// `chunk` heads of q and k with them, so that the ~40 instructions of a sine are shared by up to 8 heads; eight lanes
// read the 128 contiguous bytes of one half of a row.  2 x 40 heads x 8191 positions, three axes, forward and backward: 113 us, 91 % of
// the copy bandwidth.
#include "host_common.cuh"
#include "ptx.cuh"

namespace splash {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryHeads = 4;  // rows in flight per thread

struct RotaryArgs {
  SplashRotaryParams p;
  int32_t rot_items, items;  // vectors of pairs per row, and with those that pass through
  int32_t heads, chunk;      // q and k heads together; heads per thread
};

template <int VEC>
struct Raw;
template <>
struct Raw<8> { using T = uint4; };
template <>
struct Raw<4> { using T = uint2; };

template <int VEC, bool BF16>
__device__ __forceinline__ void unpack(const typename Raw<VEC>::T& r, float* x) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) {
    if constexpr (BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <int VEC, bool BF16>
__device__ __forceinline__ typename Raw<VEC>::T pack(const float* x) {
  typename Raw<VEC>::T r;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) w[i] = pack2<BF16>(x[2 * i], x[2 * i + 1]);
  return r;
}

template <int VEC, bool BF16, bool ADJACENT>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a) {
  using V = typename Raw<VEC>::T;
  const SplashRotaryParams& p = a.p;
  const long long id = static_cast<long long>(blockIdx.x) * kRotaryThreads + threadIdx.x;
  const long long token = id / a.items;
  const int item = static_cast<int>(id - token * a.items);
  if (token >= static_cast<long long>(p.batch) * p.len) return;
  const int b = static_cast<int>(token / p.len);
  const int s = static_cast<int>(token - static_cast<long long>(b) * p.len);
  const bool turning = item < a.rot_items;

  float cs[VEC], sn[VEC];
  if (turning) {
    const long long at = b * p.pos_stride[0] + s * p.pos_stride[2];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int pair = item * VEC + i;
      const long long off = at + p.axis[pair] * p.pos_stride[1];
      const long long pos = p.pos_is_64 ? static_cast<const int64_t*>(p.positions)[off]
                                        : static_cast<const int32_t*>(p.positions)[off];
      const uint64_t turns = static_cast<uint64_t>(pos) * p.turns[pair];
      sincospif(static_cast<float>(static_cast<int32_t>(turns >> 32)) * 0x1p-31f, &sn[i], &cs[i]);
      if (p.inverse) sn[i] = -sn[i];
    }
  }
  // The two vectors of a thread: the halves of its pairs, or 2 VEC neighbours; of a part that passes through one.
  const int first = !turning ? 2 * p.pairs + (item - a.rot_items) * VEC : ADJACENT ? item * 2 * VEC : item * VEC;
  const int second = first + (ADJACENT ? VEC : p.pairs);

  const int h_end = min(a.heads, (static_cast<int>(blockIdx.y) + 1) * a.chunk);
  for (int h0 = blockIdx.y * a.chunk; h0 < h_end; h0 += kRotaryHeads) {
    V lo[kRotaryHeads], hi[kRotaryHeads];
#pragma unroll
    for (int j = 0; j < kRotaryHeads; ++j) {
      const int h = h0 + j;
      if (h >= h_end) continue;
      const bool is_q = h < p.q_heads;
      const int64_t* st = is_q ? p.q_stride : p.k_stride;
      const uint16_t* src = static_cast<const uint16_t*>(is_q ? p.q : p.k) + b * st[0] +
                            (is_q ? h : h - p.q_heads) * st[1] + s * st[2];
      lo[j] = *reinterpret_cast<const V*>(src + first);
      if (turning) hi[j] = *reinterpret_cast<const V*>(src + second);
    }
#pragma unroll
    for (int j = 0; j < kRotaryHeads; ++j) {
      const int h = h0 + j;
      if (h >= h_end) continue;
      const bool is_q = h < p.q_heads;
      const long long row = is_q ? (static_cast<long long>(b) * p.q_heads + h) * p.len + s
                                 : (static_cast<long long>(b) * p.k_heads + (h - p.q_heads)) * p.len + s;
      uint16_t* dst = static_cast<uint16_t*>(is_q ? p.q_out : p.k_out) + row * p.head_dim;
      const float scale = is_q ? p.q_scale : 1.f;
      float x[2 * VEC], y[2 * VEC];
      unpack<VEC, BF16>(lo[j], x);
      if (!turning) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[i] = x[i] * scale;
        *reinterpret_cast<V*>(dst + first) = pack<VEC, BF16>(y);
        continue;
      }
      unpack<VEC, BF16>(hi[j], x + VEC);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int ia = ADJACENT ? 2 * i : i, ib = ADJACENT ? 2 * i + 1 : VEC + i;
        y[ia] = (x[ia] * cs[i] - x[ib] * sn[i]) * scale;
        y[ib] = (x[ib] * cs[i] + x[ia] * sn[i]) * scale;
      }
      *reinterpret_cast<V*>(dst + first) = pack<VEC, BF16>(y);
      *reinterpret_cast<V*>(dst + second) = pack<VEC, BF16>(y + VEC);
    }
  }
}

template <int VEC>
static int launch_rotary(const SplashRotaryParams& p, cudaStream_t stream) {
  RotaryArgs a;
  a.p = p;
  a.rot_items = p.pairs / VEC;
  a.items = a.rot_items + (p.head_dim - 2 * p.pairs) / VEC;
  a.heads = p.q_heads + (p.k ? p.k_heads : 0);
  const long long threads = static_cast<long long>(p.batch) * p.len * a.items;
  const long long blocks = (threads + kRotaryThreads - 1) / kRotaryThreads;
  if (blocks >= (1ll << 31)) return fail(SPLASH_INVALID_ARGUMENT, "batch * length too large for one rotary call");
  // Eight heads share a thread's sines where that still gives every SM a few blocks.
  a.chunk = 8;
  while (a.chunk > 1 && blocks * ((a.heads + a.chunk - 1) / a.chunk) < 4ll * sm_count()) a.chunk /= 2;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((a.heads + a.chunk - 1) / a.chunk));
  const bool bf16 = p.dtype == SPLASH_DTYPE_BF16;
  auto kernel = p.adjacent ? (bf16 ? rotary_kernel<VEC, true, true> : rotary_kernel<VEC, false, true>)
                           : (bf16 ? rotary_kernel<VEC, true, false> : rotary_kernel<VEC, false, false>);
  kernel<<<grid, kRotaryThreads, 0, stream>>>(a);
  SPLASH_CUDA_CHECK(cudaGetLastError());
  return SPLASH_OK;
}

static bool rows_aligned(const void* base, const int64_t* stride, int elems) {
  const int bytes = 2 * elems;
  return reinterpret_cast<uintptr_t>(base) % bytes == 0 && stride[0] % elems == 0 && stride[1] % elems == 0 &&
         stride[2] % elems == 0;
}

}  // namespace splash

using namespace splash;

extern "C" int splash_rotary(const SplashRotaryParams* p, void* stream) {
  if (!p) return fail(SPLASH_INVALID_ARGUMENT, "params is null");
  if (p->dtype != SPLASH_DTYPE_BF16 && p->dtype != SPLASH_DTYPE_F16) return fail(SPLASH_UNSUPPORTED, "Only bf16/f16 are supported");
  if (p->batch < 0 || p->len < 0 || p->q_heads <= 0 || (p->k && p->k_heads <= 0))
    return fail(SPLASH_INVALID_ARGUMENT, "sizes must be positive");
  if (p->head_dim <= 0 || p->pairs <= 0 || p->pairs % 4 || p->head_dim % 4 || 2 * p->pairs > p->head_dim)
    return fail(SPLASH_UNSUPPORTED, "head_dim and the number of pairs must be multiples of 4, with 2 * pairs <= head_dim");
  if (p->batch == 0 || p->len == 0) return SPLASH_OK;
  if (!p->q || !p->q_out || !p->positions || !p->turns || !p->axis || (p->k && !p->k_out))
    return fail(SPLASH_INVALID_ARGUMENT, "q, q_out, positions, turns and axis must be non-null");
  if (p->q_heads + static_cast<int64_t>(p->k ? p->k_heads : 0) > 65535) return fail(SPLASH_INVALID_ARGUMENT, "too many heads");
  const int64_t packed[3] = {0, 0, 0};
  auto fits = [&](int elems) {
    return p->pairs % elems == 0 && p->head_dim % elems == 0 && rows_aligned(p->q, p->q_stride, elems) &&
           rows_aligned(p->q_out, packed, elems) &&
           (!p->k || (rows_aligned(p->k, p->k_stride, elems) && rows_aligned(p->k_out, packed, elems)));
  };
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fits(8)) return launch_rotary<8>(*p, st);
  if (fits(4)) return launch_rotary<4>(*p, st);
  return fail(SPLASH_INVALID_ARGUMENT, "rows of q, k and the results must be 8-byte aligned");
}
