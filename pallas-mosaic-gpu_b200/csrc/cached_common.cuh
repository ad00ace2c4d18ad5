// Attention over a paged cache: what its two kernels (cached_kernel.cuh, cached_few_kernel.cuh) share -- the cutting of the
// work, the loads, drafted trees, and e4m3 operands.
#pragma once

#include <stddef.h>

#include "../../include/splash_sm100.h"
#include "ptx.cuh"

namespace splash {

constexpr int kCachedThreads = 384;
constexpr int kCachedTile = 128;        // keys per tile
constexpr int kCachedMaxSlots = 6;      // of the K ring, and of the V ring
constexpr int kCachedAuxSlots = 16;     // exponents of a tile; more than tiles can be on their way (see the producer)
// Lengths of segments on their way from the warp that loads the keys to P V, which is at most 14 tiles behind: the ring, and
// the scores that the softmax lets be ahead of P V (it writes no P before that of its previous tile was used).
constexpr int kCachedSegRing = 16;
constexpr int kCachedMaxTree = 128;     // nodes of a drafted tree
constexpr int kCachedMostUnitCost = 8;  // (see cached_plan)
constexpr float kCachedLog2e = 1.4426950408889634f;
constexpr float kCachedLn2 = 0.6931471805599453f;

struct CachedArgs {
  const void* q;
  const int8_t* k_exponent;
  const int8_t* v_exponent;
  const int32_t* page_table;
  const int32_t* lengths;
  const int32_t* counts;
  const int32_t* parents;
  void* out;
  float* lse_out;
  int32_t* status;
  int32_t* status_host;
  int4* cuts;         // [CTAs] first segment of each: entry (-1: none), kv head, first tile, tiles of the unit
  float* part_o;      // [2 * CTAs, R, D]
  float2* part_ml;    // [2 * CTAs, R]: maximum (powers of 2) and sum
  int64_t table_stride, parents_stride;
  int32_t batch, heads, kv_heads, n, rows, row_tiles, row_cap;  // rows = heads / kv_heads * n
  int32_t unit_cost;  // what a unit costs besides its tiles, in tiles: it stands that much longer in the line
  int32_t num_pages, page_shift, table_width;  // pages of 2^page_shift tokens
  int32_t window, sinks;  // window < 0: none
  float mask_value, soft_cap;
};

// What the rows of one (sequence, row tile) can see, the same for every kv head.
struct CachedGeom {
  int count, before;   // new tokens; tokens in front of them
  int i0, i1;          // new tokens among the rows of the tile: [i0, i1)
  int lo, hi, sink_hi; // keys that some row sees lie in [lo, hi) or [0, sink_hi)
  int first, sink_tiles, tiles;  // first tile of the window, tiles of sinks in front of it, all tiles
};

__device__ __forceinline__ CachedGeom cached_geom(const CachedArgs& a, int entry) {
  CachedGeom g;
  const int b = entry / a.row_tiles, rt = entry - b * a.row_tiles;
  const int capacity = a.table_width << a.page_shift;  // (checked on the host to fit)
  const int len = min(max(a.lengths[b], 0), capacity);
  g.count = min(a.counts ? min(max(a.counts[b], 0), a.n) : a.n, len);
  g.before = len - g.count;
  const int r0 = rt * a.row_cap, r1 = min(a.rows, r0 + a.row_cap);
  g.i0 = 0;
  g.i1 = g.count;
  if (r1 - r0 < a.n && r0 % a.n <= (r1 - 1) % a.n) {  // rows of one head
    g.i0 = r0 % a.n;
    g.i1 = min(g.count, (r1 - 1) % a.n + 1);
  }
  g.hi = g.before + g.i1;
  const bool tree = a.parents != nullptr;
  g.lo = a.window < 0 ? 0 : max(0, g.before + (tree ? 0 : g.i0) - a.window);
  g.sink_hi = a.window < 0 ? 0 : min(a.sinks, g.lo);
  g.first = g.lo / kCachedTile;
  g.sink_tiles = min((g.sink_hi + kCachedTile - 1) / kCachedTile, g.first);
  g.tiles = g.i0 < g.i1 ? g.sink_tiles + (g.hi + kCachedTile - 1) / kCachedTile - g.first : 0;
  return g;
}

// Where CTA c's share of a line of this length begins, cut for `ctas` CTAs.
__device__ __forceinline__ int cached_share(int c, int length, int ctas) {
  return static_cast<int>(static_cast<long long>(c) * length / ctas);
}

// A CTA's way along its share: one segment (a unit or the part of it that falls into the share) after the other.
struct CachedCursor {
  int entry, head, offset, left;  // the next unit, where in it the share goes on, what is left of the share
  CachedGeom g;
  int seg_tile, seg_n, seg_entry, seg_head;  // the current segment: its unit's tiles seg_tile .. seg_tile + seg_n - 1
  bool whole;                                // it is all of its unit

  __device__ __forceinline__ void start(const CachedArgs& a, int e, int h, int o, int n) {
    entry = e; head = h; offset = o; left = n;
    if (left > 0) g = cached_geom(a, entry);
  }
  __device__ __forceinline__ bool next(const CachedArgs& a) {
    while (left > 0) {
      if (head == a.kv_heads) {
        head = 0;
        const int entries = a.batch * a.row_tiles;
        do {
          if (++entry >= entries) return false;
          g = cached_geom(a, entry);
        } while (g.tiles == 0);
      }
      const int from = max(offset - a.unit_cost, 0), to = min(offset + left - a.unit_cost, g.tiles);
      seg_entry = entry;
      seg_head = head;
      left -= g.tiles + a.unit_cost - offset;
      offset = 0;
      ++head;
      if (to > from) {
        seg_tile = from;
        seg_n = to - from;
        whole = seg_n == g.tiles;
        return true;
      }
    }
    return false;
  }
  // First key of the segment's i-th tile.
  __device__ __forceinline__ int key0(int i) const {
    const int t = seg_tile + i;
    return (t < g.sink_tiles ? t : g.first + t - g.sink_tiles) * kCachedTile;
  }
};

enum CachedSite : int {
  kCSiteLoadEmpty = 301, kCSiteLoadQ, kCSiteMmaQ, kCSiteMmaFull, kCSiteMmaP, kCSiteMmaO, kCSiteSmxS, kCSiteSmxV,
  kCSiteSmxSync, kCSiteSmxDone, kCSiteConvQ, kCSiteTree, kCSiteSmxTree, kCSiteMmaS, kCSiteSmxM, kCSiteSmxP, kCSiteSmxO,
};

struct CachedBarriers {
  // The keys' ring and the values' are apart: a parity tells a slot's phase only from the one before, so whoever waits for
  // a slot must have waited for its previous use, and scores and P V go through their tiles at paces of their own.
  uint64_t k_full[kCachedMaxSlots], k_empty[kCachedMaxSlots], v_full[kCachedMaxSlots], v_empty[kCachedMaxSlots];
  uint64_t s_ready[4], pv_done[2];
  uint64_t s_free[4], p_ready[2];
  uint64_t q_full[2], q_free[2], o_free, sync;  // (one of either in use where Q has one buffer)
  uint64_t tree_full[2], tree_free[2];
  uint32_t tmem_base, abort_flag, dead;
  int32_t first_entry, first_head, first_offset, share;
  int32_t seg_n[kCachedSegRing];
};
static_assert(sizeof(CachedBarriers) <= 512, "");

// ---- 8-bit operands -------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float exponent_scale(int e) {  // -128 marks a row that was not finite
  return e == -128 ? __uint_as_float(0x7fc00000u) : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Warp-collective forms as in ptx.cuh, for 8-bit operands (kind::f8f6f4, e4m3 by e4m3).
__device__ __forceinline__ void umma8_ss2_w(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      ".reg .b64 da, db;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t"
      "}\n"
      ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma8_ts2_w(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      ".reg .b64 db;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], db, %4, p;\n\t"
      "}\n"
      ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Probabilities as operands of 8 bits.  A number of f16 is a sum of numbers of e5m2: its upper byte is one (sign, exponent, the
// first 2 of 10 bits, subnormals alike), what that leaves is a number of f16 again and needs no rounding, and so on, 3 bits each.
// Four hold all of it, three round it to 9 bits; every one is a float of its own, so what is small loses nothing beside what is
// large, down to e5m2's lowest step, 2^-16.  Two pairs of f16 to TERMS words of four codes.
template <int TERMS>
__device__ __forceinline__ void e5m2_terms(uint32_t a, uint32_t b, uint32_t* codes) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    if (t == TERMS - 1) {  // to nearest (numbers that are left over are far from the carry into the sign, but for NaN)
      a += 0x00800080u;
      b += 0x00800080u;
    }
    codes[t] = __byte_perm(a, b, 0x7531);
    if (t < TERMS - 1) {
      asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a) : "r"(a & 0xff00ff00u));
      asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(b) : "r"(b & 0xff00ff00u));
    }
  }
}
// Probabilities are scaled so that a row's largest 2^ev p stands at 2^12, or up to 2^kCachedLag8 above while the maximum lags behind
// (f16 and e5m2 end below 2^16): what is lost of a small one is half of 2^-16, 2^-29 of the row's largest or less.
// The exponentials, and with them the sums, carry 2^5 of that and the values' scales the rest: 2^ev goes up to 2^120.
constexpr float kCachedLag8 = 3.f;
constexpr float kCachedExpBits8 = 5.f;
constexpr float kCachedVScale8 = 128.f;

// Upper half of a shared-memory descriptor of tiles with 128- or 64-byte rows, swizzled over their rows.
template <int BOX_BYTES>
__host__ __device__ constexpr uint32_t cached_desc_hi() {
  return (((8u * BOX_BYTES) >> 4) & 0x3fff) | (1u << 14) | ((BOX_BYTES == 128 ? 2u : 4u) << 29);
}
// Byte offset of 16-byte chunk `chunk` of row `row` in such a tile.
template <int BOX_BYTES>
__device__ __forceinline__ uint32_t cached_swz(uint32_t row, uint32_t chunk) {
  if constexpr (BOX_BYTES == 128) return row * 128u + ((chunk ^ (row & 7u)) << 4);
  else return row * 64u + ((chunk ^ ((row >> 1) & 3u)) << 4);
}

// Programmatic dependent launch: the second pass may be set up while this one runs; it waits for its end itself.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Whole 64-bit words: tile (low half) and maximum of a row arrive together.
__device__ __forceinline__ uint64_t lds64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.volatile.shared.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts64(uint32_t addr, uint64_t v) {
  asm volatile("st.volatile.shared.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
// Whether a barrier's phase is over, without waiting.
__device__ __forceinline__ bool mbar_probe(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred P;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// N = 2 or 4 bytes.
template <int N>
__device__ __forceinline__ void sts_bytes(uint32_t addr, uint32_t v) {
  if constexpr (N == 4) sts32(addr, v);
  else asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(static_cast<uint16_t>(v)) : "memory");
}
__device__ __forceinline__ int lds_s8(uint32_t addr) {
  int v;
  asm volatile("ld.shared.s8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

#define SPLASH_KBAR(field, idx) \
  (bars_u32 + static_cast<uint32_t>(offsetof(CachedBarriers, field)) + 8u * static_cast<uint32_t>(idx))
#define SPLASH_KWORD(field) (bars_u32 + static_cast<uint32_t>(offsetof(CachedBarriers, field)))

// A walk of the warp that issues the products, over the CTA's tiles; there are two, the scores' and P V's.  `step`: tiles so far,
// which give buffers, ring slots and parities.  The segments' lengths come from the warp that loads the keys, which is ahead (a
// cursor of its own would cost registers that this warp does not have).
struct CachedWalk {
  int seg = 0, i = 0, step = 0, n = 0;
  __device__ __forceinline__ void at_tile(uint32_t bars_u32) {  // once the tile's keys have come
    if (i == 0) n = static_cast<int>(lds32(SPLASH_KWORD(seg_n) + (seg % kCachedSegRing) * 4));
  }
  __device__ __forceinline__ void advance() {
    ++step;
    if (++i == n) {
      i = 0;
      ++seg;
    }
  }
};
__device__ __forceinline__ int cached_share_tiles(const CachedArgs& a, CachedCursor cur) {
  int tiles = 0;
  while (cur.next(a)) tiles += cur.seg_n;
  return tiles;
}

// ---- what the warps of both kernels have in common ------------------------------------------------------------------
// One warp: barriers.  The softmax warps arrive once each: 32 arrivals of a warp would be taken one after the other.
__device__ __forceinline__ void cached_init_barriers(uint32_t bars_u32, int lane) {
  constexpr uint32_t kNumBarriers = offsetof(CachedBarriers, tmem_base) / 8;
  for (uint32_t i = lane; i < kNumBarriers; i += 32) {
    const uint32_t off = 8u * i;
    uint32_t count = 1;
    if (off >= offsetof(CachedBarriers, s_free) && off < offsetof(CachedBarriers, q_full)) count = 4;
    if (off == offsetof(CachedBarriers, o_free) || off == offsetof(CachedBarriers, sync)) count = 8;
    if (off >= offsetof(CachedBarriers, tree_free) && off < offsetof(CachedBarriers, tmem_base)) count = 8;
    mbar_init(bars_u32 + off, count);
  }
}

// One warp: this CTA's share of the line.
__device__ __forceinline__ void cached_find_share(const CachedArgs& a, uint32_t bars_u32, int lane) {
  const int entries = a.batch * a.row_tiles;
  auto line = [&](int e) -> int {  // what (sequence, row tile) e takes of the line, all kv heads
    if (e >= entries) return 0;
    const int tiles = cached_geom(a, e).tiles;
    return tiles > 0 ? (tiles + a.unit_cost) * a.kv_heads : 0;
  };
  int total = 0;
  for (int e0 = 0; e0 < entries; e0 += 32) total += __reduce_add_sync(0xffffffffu, line(e0 + lane));
  const int ctas = min(static_cast<int>(gridDim.x), total);
  const int c = blockIdx.x;
  const int begin = c < ctas ? cached_share(c, total, ctas) : 0, end = c < ctas ? cached_share(c + 1, total, ctas) : 0;
  if (begin < end) {
    int passed = 0;
    for (int e0 = 0; e0 < entries; e0 += 32) {
      const int mine = line(e0 + lane);
      const int sum = __reduce_add_sync(0xffffffffu, mine);
      if (begin < passed + sum) {
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const int x = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += x;
        }
        const int from = passed + upto - mine;
        if (begin >= from && begin < from + mine) {
          const int unit = mine / a.kv_heads;
          sts32(SPLASH_KWORD(first_entry), e0 + lane);
          sts32(SPLASH_KWORD(first_head), (begin - from) / unit);
          sts32(SPLASH_KWORD(first_offset), (begin - from) % unit);
        }
        break;
      }
      passed += sum;
    }
  }
  if (lane == 0) sts32(SPLASH_KWORD(share), end - begin);
}

// 256 threads: zeros for the CTA's share of the units whose rows see no key.
template <int D>
__device__ __forceinline__ void cached_fill_unseen(const CachedArgs& a, int thread) {
  for (int e = blockIdx.x; e < a.batch * a.row_tiles; e += gridDim.x) {
    if (cached_geom(a, e).tiles > 0) continue;
    const int b = e / a.row_tiles, rt = e - b * a.row_tiles;
    const int rows = min(a.row_cap, a.rows - rt * a.row_cap);
    for (int h = 0; h < a.kv_heads; ++h) {
      const long long row0 = static_cast<long long>(b * a.kv_heads + h) * a.rows + rt * a.row_cap;
      for (int x = thread; x < rows * (D / 8); x += 256)
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row0 * D)[x] = make_uint4(0, 0, 0, 0);
      if (a.lse_out)
        for (int x = thread; x < rows; x += 256) a.lse_out[row0 + x] = a.mask_value;
    }
  }
}

// The K or the V producer.  L: layout of a tile in the ring; `load_q` brings the rows of a segment.
template <class L, bool QUANT, typename LoadQ>
__device__ __forceinline__ void cached_load(const CachedArgs& a, CachedCursor cur, uint32_t bars_u32, uint32_t ring, uint32_t aux_u32,
                                            const CUtensorMap* tm, bool is_v, int lane, const WaitCtx& ctx, LoadQ load_q) {
  const uint32_t full = is_v ? SPLASH_KBAR(v_full, 0) : SPLASH_KBAR(k_full, 0);
  const uint32_t empty = is_v ? SPLASH_KBAR(v_empty, 0) : SPLASH_KBAR(k_empty, 0);
  const int piece_shift = min(a.page_shift, 7), piece = 1 << piece_shift;  // keys per TMA box; a lane has one box of a tile
  const int pieces = kCachedTile >> piece_shift;
  int slot = 0;
  uint32_t phase = 0;
  int step = 0;
  for (int seg = 0; cur.next(a); ++seg) {
    const CachedGeom& g = cur.g;
    const int b = cur.seg_entry / a.row_tiles, rt = cur.seg_entry - b * a.row_tiles;
    if (!QUANT && !is_v) {  // (an 8-bit call splits its rows in another warp)
      if (seg > 0 && !warp_wait(SPLASH_KBAR(q_free, 0), (seg - 1) & 1, ctx, kCSiteLoadQ, seg)) return;
      load_q(b, rt, cur.seg_head);
    }
    if (!is_v && lane == 0) sts32(SPLASH_KWORD(seg_n) + (seg % kCachedSegRing) * 4, static_cast<uint32_t>(cur.seg_n));
    const int32_t* table = a.page_table + b * a.table_stride;
    // This lane's piece of tile i: its page id, -1 where nobody sees it; asked for two tiles ahead of its use, so that
    // the load never waits for it.
    auto page_of = [&](int i) -> int {
      int id = -1;
      if (i < cur.seg_n && lane < pieces) {
        const int key = cur.key0(i) + lane * piece;
        if (key < g.hi && (key + piece > g.lo || key < g.sink_hi))
          asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(id) : "l"(table + (key >> a.page_shift)));
      }
      return id;
    };
    int page = page_of(0), page_1 = page_of(1);  // of tiles i, i + 1
    for (int i = 0; i < cur.seg_n; ++i, ++step) {
      const int page_2 = page_of(i + 2);
      if (step >= L::kSlots && !warp_wait(empty + 8 * slot, phase ^ 1, ctx, kCSiteLoadEmpty, step)) return;
      asm volatile("" : "+r"(page));
      const bool some = page >= 0 && page < a.num_pages;
      const uint32_t count = __popc(__ballot_sync(0xffffffffu, some));
      if (lane == 0) mbar_arrive_expect_tx(full + 8 * slot, count * piece * (L::kRowBytes + (QUANT && !is_v ? 2 : 0)));
      __syncwarp();
      if (some) {
        const int row = ((page * a.kv_heads + cur.seg_head) << a.page_shift) + ((cur.key0(i) + lane * piece) & ((1 << a.page_shift) - 1));
        const uint32_t dst = ring + slot * L::kSlotBytes + lane * piece * L::kBoxBytes;
#pragma unroll
        for (int c = 0; c < L::kBoxes; ++c)
          tma_load_2d(dst + c * (kCachedTile * L::kBoxBytes), tm, c * L::kBoxElems, row, full + 8 * slot);
        if (QUANT && !is_v) {
          // Exponents of the tile's keys and values.  Their slot is used again 16 tiles on; this warp is ahead of the
          // scores by the ring (at most 6 tiles), and those of the softmax by two.
          const uint32_t x = aux_u32 + (step % kCachedAuxSlots) * (2 * kCachedTile) + lane * piece;
          bulk_load_1d(x, a.k_exponent + row, piece, full + 8 * slot);
          bulk_load_1d(x + kCachedTile, a.v_exponent + row, piece, full + 8 * slot);
        }
      }
      if (++slot == L::kSlots) { slot = 0; phase ^= 1; }
      page = page_1;
      page_1 = page_2;
    }
  }
}

// One warp: the drafted tree of sequence b into one of two buffers, the `trees`-th of the CTA.  A tree is [128 nodes][8
// words]: 0, four words of the nodes a node sees, 0, unused, depth.
// Which nodes each node sees -- itself and its ancestors -- by doubling: what a node sees is what it and the node
// `up` steps above it see, for up = 1, 2, 4, ...
__device__ __forceinline__ bool cached_make_tree(const CachedArgs& a, int b, int before, int trees, uint32_t bars_u32, uint32_t parents_u32,
                                                 int lane, const WaitCtx& ctx) {
  const uint32_t ups_u32 = parents_u32 + kCachedMaxTree * 4, trees_u32 = ups_u32 + kCachedMaxTree * 4;
  const int buf = trees & 1;
  if (trees >= 2 && !warp_wait(SPLASH_KBAR(tree_free, buf), ((trees >> 1) & 1) ^ 1, ctx, kCSiteTree, trees)) return false;
  const uint32_t tree = trees_u32 + buf * (kCachedMaxTree * 32);
  constexpr int kPer = kCachedMaxTree / 32;
  static_assert(kPer == 4, "");
  uint32_t bits[kPer][4];
  int up[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = j * 32 + lane;
    up[j] = i < a.n ? a.parents[b * a.parents_stride + i] : -1;
    if (up[j] >= i || up[j] < 0) up[j] = -1;  // a parent stands before its child; anything else is the context
#pragma unroll
    for (int w = 0; w < 4; ++w) bits[j][w] = w == j ? 1u << lane : 0u;
    sts32(parents_u32 + i * 4, static_cast<uint32_t>(up[j]));
    sts32(ups_u32 + i * 4, static_cast<uint32_t>(up[j]));
#pragma unroll
    for (int w = 0; w < 8; ++w) sts32(tree + (i * 8 + w) * 4, w >= 1 && w <= 4 ? bits[j][w - 1] : 0u);
  }
  __syncwarp();
  while (__any_sync(0xffffffffu, (up[0] & up[1] & up[2] & up[3]) >= 0)) {  // (-1 in all: every chain is at its end)
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (up[j] < 0) continue;
#pragma unroll
      for (int w = 0; w < 4; ++w) bits[j][w] |= lds32(tree + (up[j] * 8 + 1 + w) * 4);
      up[j] = static_cast<int>(lds32(ups_u32 + up[j] * 4));
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = j * 32 + lane;
#pragma unroll
      for (int w = 0; w < 4; ++w) sts32(tree + (i * 8 + 1 + w) * 4, bits[j][w]);
      sts32(ups_u32 + i * 4, static_cast<uint32_t>(up[j]));
    }
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = j * 32 + lane;
    const int depth = __popc(bits[j][0]) + __popc(bits[j][1]) + __popc(bits[j][2]) + __popc(bits[j][3]) - 1;
    sts32(tree + (i * 8 + 7) * 4, static_cast<uint32_t>(depth));
    if (a.window >= 0 && depth > a.window) {
      // Ancestors in front of the window: only as sinks.
#pragma unroll
      for (int w = 0; w < 4; ++w) bits[j][w] = 0;
      int x = i;
      for (int d = depth; d >= 0; --d) {
        if (d >= depth - a.window || before + d < a.sinks) {
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (w == (x >> 5)) bits[j][w] |= 1u << (x & 31);
        }
        x = static_cast<int>(lds32(parents_u32 + x * 4));
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < kPer; ++j)
#pragma unroll
    for (int w = 0; w < 4; ++w) sts32(tree + ((j * 32 + lane) * 8 + 1 + w) * 4, bits[j][w]);
  __syncwarp();
  if (lane == 0) mbar_arrive(SPLASH_KBAR(tree_full, buf));
  return true;
}

// One warp: the rows of a segment as TERMS e4m3 terms each, handed to `store`, into one of BUFFERS in turn, and their scales into
// one of SLOTS.  Scales stay longer than the rows: the scores of a segment's last tile free its rows, and the softmax may be that
// tile and as many more behind as there are buffers of scores, each of another segment.
template <int D, bool BF16, int TERMS, int R, int BUFFERS, int SLOTS, typename Store>
__device__ __forceinline__ bool cached_split_q(const CachedArgs& a, int seg, int b, int rt, int head, uint32_t bars_u32, uint32_t qscale_u32,
                                               int lane, const WaitCtx& ctx, Store store) {
  constexpr int kPer = D / 32;  // neighbouring numbers per lane
  const int buffer = seg % BUFFERS, use = seg / BUFFERS;
  if (use > 0 && !warp_wait(SPLASH_KBAR(q_free, buffer), (use - 1) & 1, ctx, kCSiteConvQ, seg)) return false;
  const long long row0 = static_cast<long long>(b * a.kv_heads + head) * a.rows + rt * R;
  const int rows = min(R, a.rows - rt * R);
  constexpr int kBatch = 8;  // rows whose loads are in flight together
  for (int r0 = 0; r0 < R; r0 += kBatch) {
    if (seg >= SLOTS && a.row_tiles == 1 && r0 >= rows) break;  // zeros, as the first segments have left them
    uint32_t w[kBatch][kPer / 2];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int r = r0 + j;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) + (row0 + r) * D) + lane * (kPer / 2);
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) w[j][i] = r < rows ? __ldg(src + i) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int r = r0 + j;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) top = max(top, max(w[j][i] & 0x7fffu, (w[j][i] >> 16) & 0x7fffu));
      top = __reduce_max_sync(0xffffffffu, top);
      const bool bad = top >= (BF16 ? 0x7f80u : 0x7c00u);
      float amax;
      if constexpr (BF16) amax = __uint_as_float(top << 16);
      else amax = __half2float(__ushort_as_half(static_cast<unsigned short>(top)));
      // 2^-eq takes the largest number of the row into [128, 256).
      const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 7, -100), 120);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      float x[kPer];
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) {
        float2 f;
        if constexpr (BF16) f = make_float2(__uint_as_float(w[j][i] << 16), __uint_as_float(w[j][i] & 0xffff0000u));
        else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j][i]));
        x[2 * i] = f.x * down;
        x[2 * i + 1] = f.y * down;
      }
      if (lane == 0)
        sts32(qscale_u32 + (seg % SLOTS * R + r) * 4, bad ? 0x7fc00000u : static_cast<uint32_t>(e + 127) << 23);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        uint32_t code[kPer / 2];
#pragma unroll
        for (int i = 0; i < kPer / 2; ++i) {
          code[i] = e4m3x2(x[2 * i], x[2 * i + 1]);
          const float2 f = e4m3x2_to_f32(code[i]);
          x[2 * i] -= f.x;
          x[2 * i + 1] -= f.y;
        }
        // Term t of row r, this lane's kPer bytes from lane * kPer on.
        store(t, r, static_cast<uint32_t>(lane * kPer), kPer == 4 ? code[0] | (code[kPer / 2 - 1] << 16) : code[0]);
      }
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(SPLASH_KBAR(q_full, buffer));
  return true;
}

}  // namespace splash
