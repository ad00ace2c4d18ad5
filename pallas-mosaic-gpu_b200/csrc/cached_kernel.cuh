// Attention of a few new tokens per sequence over a paged cache: one token, a run of tokens, or a tree of drafted ones.
//
// Mathematics.  A unit of work is (sequence, row tile, kv head): up to R rows -- the new tokens of the heads that share
// the kv head -- against the keys its rows can see, in tiles of 128 keys:  S = Q K^T, online softmax, O += P V.
//
// What bounds it: HBM with up to 64 rows over a 16-bit cache (16 sequences of 4000 to 32768 keys, 32 / 8 heads: 188 us, 98 % of
// the copy bandwidth); the products over an 8-bit one, whose tiles take 1390 cycles to arrive and 1280 (f16: 1792) or more to
// multiply (64 rows, 32 sequences of 8192 keys, 8 kv heads: 211 us, f16 246; the bytes are 83); with more rows the start and end of
// a unit, and the exponentials.  2 * 128 * head_dim
// numbers a tile are read once for all rows, so everything is arranged to keep a ring of loads full:
//   * The tiles of all units stand in one line that is cut into equal shares, one per CTA (one CTA per SM), whatever the
//     lengths of the sequences are.  A unit that several CTAs share leaves partial results (unnormalised O, maximum and
//     sum per row, f32) for cached_finish_kernel, which adds them in the order of the keys: the same bits every time.
//   * Two producer warps, for keys and values, walk the line ahead of the others, across units: page ids two tiles ahead, one
//     TMA box per page.
//   * Rows are few, so the 128 rows of an MMA are used otherwise: Q is laid into shared memory 128 / R times, and each
//     copy's warps take the exponentials of their own part of the tile's keys (P is zero elsewhere); the copies' results
//     are added like partial ones.  A softmax warp of a one-token call thus works on 32 of 128 keys.
//   * Two softmax warpgroups take the tiles in turn.  They hand the (lagging) maxima to one another through shared memory,
//     a tile's right after its comparison and long before its exponentials, and keep partial sums; P has columns of its
//     own, so the scores of tile t + 2 are computed as soon as those of tile t are in registers: the warp that issues the
//     products looks at what either kind waits for and takes what is ready.  Tensor memory: S0 S1 P0 P1 O = 128 + 128 + 64 + 64
//     + head_dim columns.
//
// 8-bit caches are not widened on the way: e4m3 keys and values are operands of the MMA as they lie in the cache, and
// the 16-bit Q and the probabilities are split into e4m3 terms instead, which are few:
//   * q * 2^-eq = q1 + q2 (+ q3 for f16), each term what the ones before leave; S sums their products.  bf16 has 8 bits,
//     a term 4: nothing is lost but below 2^-18 of the row's largest number.
//   * 2^ek of a key scales its column of S; 2^ev of a value scales its column of P, and the running maximum is one of
//     s + ev and lags behind by a factor of 8 at most, so that a row's largest scaled probability stands at 2^12 to 2^15.
//   * P is rounded to f16 and cut into e5m2 terms (e5m2_terms), three for bf16 (9 bits, where a bf16 P has 8) and four for f16 (all
//     of it).  Every probability down to 2^-18 of the row's largest keeps these bits and every one down to 2^-29 some: many
//     small ones beside a large one add up to what they should.  Two terms of e4m3 would be one product less, but their steps
//     end at 2^-14 of the largest, and with the tail of a softmax goes its mass (one key of 32768 with weight 0.4: results off by a
//     third).  Tensor memory has columns for two terms; the others lie where the tile's scores did, and the scores of tile t + 2
//     wait for P V of tile t.
#pragma once

#include "cached_common.cuh"

namespace splash {

template <int D, bool BF16, bool QUANT, int KG>
struct CachedLayout {
  static constexpr int kRows = 128 / KG;                   // R: KG copies of the rows are the 128 of an MMA
  static constexpr int kKeys = kCachedTile / KG;           // keys whose probabilities a row's thread computes
  static constexpr int kItem = QUANT ? 1 : 2;
  static constexpr int kRowBytes = D * kItem;              // of a key
  static constexpr int kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;  // swizzle span = inner extent of a TMA box
  static constexpr int kBoxes = kRowBytes / kBoxBytes;
  static constexpr int kBoxElems = kBoxBytes / kItem;
  static constexpr int kSlotBytes = kCachedTile * kRowBytes;
  static constexpr int kTerms = QUANT ? (BF16 ? 2 : 3) : 1;   // of Q
  static constexpr int kPTerms = QUANT ? (BF16 ? 3 : 4) : 1;  // of P
  static constexpr int kQTerm = 128 * kRowBytes;
  static constexpr int kQBytes = kTerms * kQTerm;
  static constexpr int kStageStride = 36;                  // words per row of the staging area (32 used)
  static constexpr int kStageBytes = 256 * kStageStride * 4;
  // Behind the staging area: maxima and sums, barriers, then (8 bit) exponents, scales, row scales, and the tree.
  static constexpr int kMlBytes = 128 * 8 + 2 * 256 * 4;
  static constexpr int kBarBytes = 512;
  static constexpr int kAuxBytes = QUANT ? kCachedAuxSlots * 2 * kCachedTile : 0;
  static constexpr int kScaleBytes = QUANT ? 8 * kKeys * 12 : 0;  // per warp: three numbers for each of its keys
  static constexpr int kQScaleSlots = 4;                   // (two buffers of scores: see cached_split_q)
  static constexpr int kQScaleBytes = QUANT ? kQScaleSlots * kRows * 4 : 0;
  static constexpr int kTreeBytes = kCachedMaxTree * 8 + 2 * kCachedMaxTree * 8 * 4;  // parents, pointers | two trees
  static constexpr int kFixed = 1024 + kQBytes + kStageBytes + kMlBytes + kBarBytes + kAuxBytes + kScaleBytes + kQScaleBytes + kTreeBytes;
  static constexpr int kSlotsFit = (227 * 1024 - kFixed) / (2 * kSlotBytes);
  static constexpr int kSlots = kSlotsFit < kCachedMaxSlots ? kSlotsFit : kCachedMaxSlots;  // tiles of either ring
  static_assert(kSlots >= 2, "two tiles have to fit");
  static constexpr int kSmem = kFixed + 2 * kSlots * kSlotBytes;
  static constexpr int kPCol = 256, kOCol = 384;  // S of the two warpgroups | P of the two | O
  // Scores that a thread has in registers at a time.  With all 128 of a row without copies it has registers for little else, and
  // what is spilled comes back from L2, as shared memory leaves the L1 cache next to nothing: halves are read from tensor memory
  // for the maximum, and the second once more for the exponentials (64 sequences of 100 to 3000 keys, 8 kv heads, 192 rows: 191 ->
  // 172 us; 8 bit, where a half is also scaled twice, 343 -> 326 with a P of two terms).
  static constexpr int kPart = kKeys < 64 ? kKeys : 64, kParts = kKeys / kPart;
  static constexpr int kSoftmaxRegs = 184, kLoadRegs = 136;  // 384 * 168 at launch = 256 * 184 + 128 * 136
};

template <int D, bool BF16, bool QUANT, int KG>
__global__ void __launch_bounds__(kCachedThreads, 1)
cached_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const CachedArgs a) {
  using L = CachedLayout<D, BF16, QUANT, KG>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t q_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t k_u32 = q_u32 + L::kQBytes;
  const uint32_t v_u32 = k_u32 + L::kSlots * L::kSlotBytes;
  const uint32_t stage_u32 = v_u32 + L::kSlots * L::kSlotBytes;
  const uint32_t ml_u32 = stage_u32 + L::kStageBytes;
  const uint32_t bars_u32 = ml_u32 + L::kMlBytes;
  const uint32_t aux_u32 = bars_u32 + L::kBarBytes;
  const uint32_t scale_u32 = aux_u32 + L::kAuxBytes;
  const uint32_t qscale_u32 = scale_u32 + L::kScaleBytes;
  const uint32_t parents_u32 = qscale_u32 + L::kQScaleBytes;
  const uint32_t trees_u32 = parents_u32 + 2 * kCachedMaxTree * 4;

  const int warp = uniform_warp_index();
  const int lane = threadIdx.x & 31;
  const WaitCtx ctx{SPLASH_KWORD(abort_flag)};

  // ---- set-up: barriers, tensor memory, this CTA's share of the line ------------------------------------------------
  if (warp == 8) {
    cached_init_barriers(bars_u32, lane);
    if (lane == 0) {
      launch_dependents();
      sts32(SPLASH_KWORD(abort_flag), 0);
      sts32(SPLASH_KWORD(dead), a.status[0] != 0);
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
      if (!QUANT) prefetch_tensormap(&tm_q);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
  } else if (warp == 9) {
    tmem_alloc(SPLASH_KWORD(tmem_base), 512);
    tmem_relinquish();
  } else if (warp >= 4 && warp < 8) {
    sts64(ml_u32 + (threadIdx.x - 128) * 8, 0xffffffffull);  // no tile yet
  } else if (warp == 0) {
    cached_find_share(a, bars_u32, lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = lds32(SPLASH_KWORD(tmem_base));
  if (lds32(SPLASH_KWORD(dead))) {
    if (blockIdx.x == 0 && threadIdx.x == 0) repeat_abort(a.status, a.status_host);
    if (warp == 9) {
      __syncwarp();
      tmem_dealloc(tmem, 512);
    }
    return;
  }
  CachedCursor cur;
  cur.start(a, lds32(SPLASH_KWORD(first_entry)), lds32(SPLASH_KWORD(first_head)), lds32(SPLASH_KWORD(first_offset)),
            lds32(SPLASH_KWORD(share)));

  if (warp >= 8) {
    setmaxnreg_dec<L::kLoadRegs>();
    if (warp == 8 || warp == 11) {
      // ------------------------------------------ loads: keys (and Q, and exponents), values ----------------------------
      const bool is_v = warp == 11;
      cached_load<L, QUANT>(a, cur, bars_u32, is_v ? v_u32 : k_u32, aux_u32, is_v ? &tm_v : &tm_k, is_v, lane, ctx, [&](int b, int rt, int head) {
        if (elect_one()) {
          const int row = (b * a.kv_heads + head) * a.rows + rt * L::kRows;
          mbar_arrive_expect_tx(SPLASH_KBAR(q_full, 0), L::kQBytes);
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int copy = 0; copy < KG; ++copy)
              tma_load_2d(q_u32 + c * (128 * 128) + copy * (L::kRows * 128), &tm_q, c * 64, row, SPLASH_KBAR(q_full, 0));
        }
      });
    } else if (warp == 9) {
      // ------------------------------------------ products -----------------------------------------------------------
      constexpr uint32_t kHi = cached_desc_hi<L::kBoxBytes>();
      constexpr uint32_t kIdescQK = make_idesc(BF16 && !QUANT, 128, kCachedTile, false, false);
      constexpr uint32_t kIdescPV = make_idesc(BF16 && !QUANT, 128, D, false, true) | (QUANT ? 1u << 7 : 0u);  // P: e5m2
      constexpr int kStepsPerBox = L::kBoxBytes / 32;  // an MMA takes 32 bytes of K per row
      const int tiles = cached_share_tiles(a, cur);
      CachedWalk qk, pv;
      uint32_t spins = 0;
      uint64_t t0 = 0;
      while (pv.step < tiles) {
        bool issued = false;
        if (qk.step < tiles) {
          const int buf = qk.step & 1, slot = qk.step % L::kSlots;
          const bool ready = mbar_probe(SPLASH_KBAR(k_full, slot), (qk.step / L::kSlots) & 1) &&
                             (qk.step < 2 || mbar_probe(SPLASH_KBAR(s_free, buf), ((qk.step - 2) >> 1) & 1)) &&
                             (!QUANT || qk.step < 2 || mbar_probe(SPLASH_KBAR(pv_done, buf), ((qk.step - 2) >> 1) & 1)) &&
                             (qk.i > 0 || mbar_probe(SPLASH_KBAR(q_full, 0), qk.seg & 1));
          if (__all_sync(0xffffffffu, ready)) {
            tc_fence_after();
            qk.at_tile(bars_u32);
            const uint32_t b_lo = desc_lo(k_u32 + slot * L::kSlotBytes, 16);
#pragma unroll
            for (int t = 0; t < L::kTerms; ++t) {
              const uint32_t a_lo = desc_lo(q_u32 + t * L::kQTerm, 16);
#pragma unroll
              for (int kk = 0; kk < L::kRowBytes / 32; ++kk) {
                const uint32_t off = ((kk / kStepsPerBox) * (128 * L::kBoxBytes) + (kk % kStepsPerBox) * 32) >> 4;
                if constexpr (QUANT) umma8_ss2_w(tmem + buf * 128, a_lo + off, kHi, b_lo + off, kHi, kIdescQK, t > 0 || kk > 0);
                else umma_ss2_w(tmem + buf * 128, a_lo + off, kHi, b_lo + off, kHi, kIdescQK, kk > 0);
              }
            }
            umma_commit_w(SPLASH_KBAR(s_ready, buf));
            umma_commit_w(SPLASH_KBAR(k_empty, slot));
            if (qk.i + 1 == qk.n) umma_commit_w(SPLASH_KBAR(q_free, 0));
            qk.advance();
            issued = true;
          }
        }
        {
          const int buf = pv.step & 1, slot = pv.step % L::kSlots;
          const bool ready = mbar_probe(SPLASH_KBAR(p_ready, buf), (pv.step >> 1) & 1) &&
                             mbar_probe(SPLASH_KBAR(v_full, slot), (pv.step / L::kSlots) & 1) &&
                             // O may be written again once the previous segment's has been read.
                             (pv.i > 0 || pv.seg == 0 || mbar_probe(SPLASH_KBAR(o_free, 0), (pv.seg - 1) & 1));
          if (__all_sync(0xffffffffu, ready)) {
            tc_fence_after();
            pv.at_tile(bars_u32);
            const uint32_t b_lo = desc_lo(v_u32 + slot * L::kSlotBytes, kCachedTile * L::kBoxBytes);
            const uint32_t p_tmem = tmem + L::kPCol + buf * 64;
            constexpr int kKeysPerMma = QUANT ? 32 : 16;
            // P is 8 columns an MMA; 8 bit: its second term follows in columns 32 .. 63, the others where the scores were, on the
            // same values.
#pragma unroll
            for (int kk = 0; kk < L::kPTerms * kCachedTile / kKeysPerMma; ++kk) {
              const uint32_t off = ((kk * kKeysPerMma) % kCachedTile * L::kBoxBytes) >> 4;
              const uint32_t p_at = kk < 8 ? p_tmem + kk * 8 : tmem + buf * 128 + (kk - 8) * 8;
              if constexpr (QUANT) umma8_ts2_w(tmem + L::kOCol, p_at, b_lo + off, kHi, kIdescPV, pv.i > 0 || kk > 0);
              else umma_ts2_w(tmem + L::kOCol, p_at, b_lo + off, kHi, kIdescPV, pv.i > 0 || kk > 0);
            }
            umma_commit_w(SPLASH_KBAR(v_empty, slot));
            umma_commit_w(SPLASH_KBAR(pv_done, buf));
            pv.advance();
            issued = true;
          }
        }
        // Bounded, as every wait: about a second without anything to issue.
        if (issued) {
          spins = 0;
        } else if ((++spins & 0xff) == 0) {
          const uint64_t now = global_timer_ns();
          if (spins == 0x100) t0 = now;
          bool give_up = lds32(SPLASH_KWORD(abort_flag)) != 0;
          if (!give_up && now - t0 > kWaitLimitNs) {
            sts32(SPLASH_KWORD(abort_flag), 0x80000000u | (static_cast<uint32_t>(kCSiteMmaFull) << 20) | (static_cast<uint32_t>(pv.step) & 0xfffffu));
            give_up = true;
          }
          if (__any_sync(0xffffffffu, give_up)) break;
        }
      }
    } else if (warp == 10 && (QUANT || a.parents != nullptr)) {
      // ------------------------------ drafted trees, and Q as e4m3 terms, ahead of their use ------------------------------
      int trees = 0, last = -1;
      for (int seg = 0; cur.next(a); ++seg) {
        const int b = cur.seg_entry / a.row_tiles, rt = cur.seg_entry - b * a.row_tiles;
        if (a.parents != nullptr && b != last) {
          last = b;
          if (!cached_make_tree(a, b, cur.g.before, trees++, bars_u32, parents_u32, lane, ctx)) break;
        }
        if constexpr (QUANT) {
          auto store = [&](int t, int r, uint32_t byte, uint32_t codes) {
#pragma unroll
            for (int copy = 0; copy < KG; ++copy)
              sts_bytes<D / 32>(q_u32 + t * L::kQTerm + cached_swz<L::kBoxBytes>(copy * L::kRows + r, byte >> 4) + (byte & 15u), codes);
          };
          if (!cached_split_q<D, BF16, L::kTerms, L::kRows, 1, L::kQScaleSlots>(a, seg, b, rt, cur.seg_head, bars_u32, qscale_u32, lane, ctx, store)) break;
        }
      }
    }
  } else {
    // ============================================ softmax ==============================================================
    setmaxnreg_inc<L::kSoftmaxRegs>();
    if (threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);  // (its first segment overwrites it)
    const int grp = warp >> 2;
    const int row_lane = (warp & 3) * 32 + lane;
    const int part = row_lane / L::kRows;                   // which copy of the rows, and which part of a tile's keys
    const int r = row_lane % L::kRows;
    const int col0 = part * L::kKeys;
    const uint32_t tmem_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t o_tmem = tmem_lane + L::kOCol;
    const uint32_t m_sh = ml_u32 + row_lane * 8;  // the latest tile of this row and copy, and the maximum after it
    // A lane's maximum after tile `step`, which its counterpart in the other warpgroup has left or will leave there.
    float m_got = 0.f;
    auto wait_m = [&](int step) -> bool {
      uint64_t got = lds64(m_sh);
      if (!__all_sync(0xffffffffu, static_cast<uint32_t>(got) == static_cast<uint32_t>(step))) {
        const uint64_t t0 = global_timer_ns();
        for (uint32_t spins = 1; ; ++spins) {
          got = lds64(m_sh);
          if (__all_sync(0xffffffffu, static_cast<uint32_t>(got) == static_cast<uint32_t>(step))) break;
          if ((spins & 0xff) == 0) {
            bool give_up = lds32(SPLASH_KWORD(abort_flag)) != 0;
            if (!give_up && global_timer_ns() - t0 > kWaitLimitNs) {
              sts32(SPLASH_KWORD(abort_flag), 0x80000000u | (static_cast<uint32_t>(kCSiteSmxM) << 20) | (static_cast<uint32_t>(step) & 0xfffffu));
              give_up = true;
            }
            if (__any_sync(0xffffffffu, give_up)) return false;
          }
        }
      }
      m_got = __uint_as_float(static_cast<uint32_t>(got >> 32));
      return true;
    };
    const uint32_t my_scales = scale_u32 + warp * (L::kKeys * 12);
    const int piece_shift = min(a.page_shift, 7);
    const bool tree = a.parents != nullptr;
    const float unit = a.soft_cap > 0.f ? a.soft_cap : 1.f;
    const float unit2 = unit * kCachedLog2e;
    const float inv_cap = a.soft_cap > 0.f ? 1.f / a.soft_cap : 1.f;
    // Powers of 2 by which the maximum may lag behind before O is rescaled, which takes about a tile's time.  8 bit: with a
    // lag of 2^1 every third tile rescales (32 x 64 heads, 2000 to 32768 keys: 272 us), with 2^3 hardly one.
    constexpr float kThreshold = QUANT ? kCachedLag8 : 8.f;
    // Powers of 2 that the exponentials, and with them the sums and O, are scaled by.  8 bit: see kCachedLag8.  An f16 P has steps of
    // 2^-24 at the least: with a row's largest at 2^7 or above, and below 2^16, that is 2^-31 of it (131072 keys of weight 2^-20
    // beside a large one: results off by 3 % without).
    constexpr float kVScale = QUANT ? kCachedVScale8 : 1.f, kExpBits = QUANT ? kCachedExpBits8 : BF16 ? 0.f : 7.f;
    uint32_t sync_par = 0;
    int step0 = 0;   // tiles of the CTA in front of the segment
    bool ok = true;
    if constexpr (KG > 1) {
      // The probabilities of the other copies' keys are zero, once and for all: buffer `grp` is written by this warpgroup.
      uint32_t zero16[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) zero16[j] = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_st16(tmem_lane + L::kPCol + grp * 64 + c * 16, zero16);
      tmem_wait_st();
    }
    int trees = 0, last_b = -1;
    bool tree_seen = false;
    auto see_tree = [&](int seg) -> bool {  // of the trees so far, the last
      const bool fine = tree_seen || warp_wait(SPLASH_KBAR(tree_full, (trees - 1) & 1), ((trees - 1) >> 1) & 1, ctx, kCSiteSmxTree, seg);
      tree_seen = true;
      return fine;
    };
    auto arrive = [&](uint32_t bar) {  // of a warp, for what all its lanes have done
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto group_sync = [&]() -> bool {
      arrive(SPLASH_KBAR(sync, 0));
      const bool fine = warp_wait(SPLASH_KBAR(sync, 0), sync_par, ctx, kCSiteSmxSync, 0);
      sync_par ^= 1;
      return fine;
    };

    for (int seg = 0; ok && cur.next(a); ++seg) {
      const CachedGeom& g = cur.g;
      const int n = cur.seg_n;
      const int b = cur.seg_entry / a.row_tiles, rt = cur.seg_entry - b * a.row_tiles;
      const int row_all = rt * L::kRows + r;       // among the rows of this (sequence, kv head)
      const int node = row_all % a.n;
      const bool live = row_all < a.rows && node < g.count;
      int depth = node;
      uint32_t above = 0;  // the words of this row's node
      if (tree) {
        if (b != last_b) {
          // (Also waited for if nobody looked at it: the barrier's parity tells a tree only from the one before.)
          if (last_b >= 0) {
            if (!see_tree(seg)) { ok = false; break; }
            arrive(SPLASH_KBAR(tree_free, (trees - 1) & 1));
          }
          last_b = b;
          ++trees;
          tree_seen = false;
        }
        above = trees_u32 + (((trees - 1) & 1) * kCachedMaxTree + node) * 32;
        // Positions are only looked at for a window; without one the tree is, once its tiles come.
        if (a.window >= 0) {
          if (!see_tree(seg)) { ok = false; break; }
          depth = static_cast<int>(lds32(above + 28));
        }
      }
      // Keys of the context (tree) or of context and run that this row sees: [v_lo, v_hi) and [0, v_sink).
      const int position = g.before + depth;
      const int v_hi = !live ? 0 : (tree ? g.before : position + 1);
      const int v_lo = a.window < 0 ? 0 : max(0, position - a.window);
      const int v_sink = a.window < 0 ? 0 : min(a.sinks, v_hi);
      const int seen_by_all = g.before + (tree ? 0 : g.i0 + 1);  // keys in front of this are behind no row
      const int all_from = a.window < 0 ? 0 : g.before + g.i1 - 1 - a.window;
      const int32_t* table = a.page_table + b * a.table_stride;
      float q_mul = inv_cap;  // what takes a score to the argument of the soft-cap
      float mul = unit2;      // ... and what it holds then to powers of 2
      float m_run = -INFINITY, l_run = 0.f;  // powers of 2; 8 bit: the maximum of s + ev
      const int pages = kCachedTile >> piece_shift;
      auto page_of = [&](int i) -> int {  // lane p: page id of piece p of tile i (anything for pieces nobody sees)
        if (i >= n || lane >= pages) return 0;
        const int key = cur.key0(i) + (lane << piece_shift);
        int id = 0;  // (asked for here, whatever the compiler thinks of its use a tile later)
        if (key < g.hi) asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(id) : "l"(table + (key >> a.page_shift)));
        return id;
      };
      const int i0 = (grp ^ step0) & 1;  // the CTA's tiles alternate between the warpgroups, whatever segment they are of
      int page = page_of(i0);

      for (int i = i0; i < n; i += 2) {
        const int step = step0 + i, buf = grp;
        const uint32_t par = (step >> 1) & 1;
        const uint32_t s_tmem = tmem_lane + buf * 128, p_tmem = tmem_lane + L::kPCol + buf * 64;
        const int key0 = cur.key0(i);
        asm volatile("" : "+r"(page));  // looked at here and not where it was asked for, a tile ago
        const uint32_t good = __ballot_sync(0xffffffffu, page >= 0 && page < a.num_pages);  // pieces that have a page
        page = page_of(i + 2);
        const bool plain = key0 + kCachedTile <= seen_by_all && (key0 >= all_from || key0 + kCachedTile <= g.sink_hi) &&
                           good == 0xffffffffu;
        // Whether key `at` of the tile is there for some row; the others may hold anything, and nothing was loaded for some.
        auto there = [&](int at) {
          const int key = key0 + at;
          return key < g.hi && (key >= g.lo || key < g.sink_hi) && ((good >> (at >> piece_shift)) & 1u);
        };
        if (!warp_wait(SPLASH_KBAR(s_ready, buf), par, ctx, kCSiteSmxS, step)) { ok = false; break; }
        tc_fence_after();
        float sv[L::kPart];  // scores of part h of this thread's keys
        auto fetch = [&](int h) {
          uint32_t* raw = reinterpret_cast<uint32_t*>(sv);
#pragma unroll
          for (int c = 0; c < L::kPart / 32; ++c) tmem_ld32(s_tmem + col0 + h * L::kPart + c * 32, raw + c * 32);
        };
        auto fetched = [&](bool last) {
          tmem_wait_ld();
          if (!last) return;
          tc_fence_before();
          arrive(SPLASH_KBAR(s_free, buf));  // the scores of tile step + 2 may come
        };
        fetch(L::kParts - 1);
        if constexpr (QUANT) {
          // Scales of this warp's keys in shared memory of its own: 2^ek | ev | 2^ev * 32, while the scores arrive.
          // (The exponents came with the keys, for which the scores waited.)
          if (i == i0) {
            const float q_scale = __uint_as_float(lds32(qscale_u32 + (seg % L::kQScaleSlots * L::kRows + r) * 4));
            q_mul = q_scale * inv_cap;
            mul = a.soft_cap > 0.f ? unit2 : unit2 * q_scale;
          }
          const uint32_t x = aux_u32 + (step % kCachedAuxSlots) * (2 * kCachedTile) + col0;
          __syncwarp();
#pragma unroll
          for (int c = 0; c < L::kKeys / 32; ++c) {
            const int at = c * 32 + lane;
            int ek = 0, ev = 0;
            if (plain || there(col0 + at)) {
              ek = lds_s8(x + at);
              ev = lds_s8(x + kCachedTile + at);
            }
            sts32(my_scales + at * 4, __float_as_uint(exponent_scale(ek)));
            sts32(my_scales + (L::kKeys + at) * 4, __float_as_uint(static_cast<float>(ev)));
            sts32(my_scales + (2 * L::kKeys + at) * 4, __float_as_uint(exponent_scale(ev) * kVScale));
          }
          __syncwarp();
        }
        if (__builtin_expect(!plain, 0) && tree && !see_tree(seg)) { ok = false; break; }
        auto prepare = [&](int h) {
          if constexpr (QUANT) {
#pragma unroll
            for (int j = 0; j < L::kPart; j += 4) {
              const uint4 k4 = lds128(my_scales + (h * L::kPart + j) * 4);
              const float2 x = mul2(make_float2(sv[j], sv[j + 1]), make_float2(__uint_as_float(k4.x), __uint_as_float(k4.y)));
              const float2 y = mul2(make_float2(sv[j + 2], sv[j + 3]), make_float2(__uint_as_float(k4.z), __uint_as_float(k4.w)));
              sv[j] = x.x; sv[j + 1] = x.y; sv[j + 2] = y.x; sv[j + 3] = y.y;
            }
          }
          if (__builtin_expect(a.soft_cap > 0.f, 0)) {
#pragma unroll
            for (int j = 0; j < L::kPart; ++j) sv[j] = tanh_approx(sv[j] * q_mul);
          }
          if (__builtin_expect(!plain, 0)) {
#pragma unroll
            for (int c = 0; c < L::kPart / 32; ++c) {
              const int at = col0 + h * L::kPart + c * 32, kb = key0 + at;
              uint32_t vis = bit_run(v_lo - kb, v_hi - kb) | bit_run(-kb, v_sink - kb);
              const int d0 = kb - g.before;
              if (tree && d0 > -32 && d0 < kCachedMaxTree) {
                const uint32_t w = above + (1 + (d0 >> 5)) * 4;
                if (live) vis |= __funnelshift_r(lds32(w), lds32(w + 4), d0 & 31);
              }
              if (piece_shift >= 5) {
                if (!((good >> (at >> piece_shift)) & 1u)) vis = 0;
              } else {
                if (!((good >> (at / 16)) & 1u)) vis &= 0xffff0000u;
                if (!((good >> (at / 16 + 1)) & 1u)) vis &= 0x0000ffffu;
              }
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((vis >> j) & 1u)) sv[c * 32 + j] = -INFINITY;
            }
          }
        };
        const float2 mul_2 = make_float2(mul, mul);
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int h = L::kParts - 1; h >= 0; --h) {
          if (h < L::kParts - 1) fetch(h);
          fetched(L::kParts == 1);
          prepare(h);
#pragma unroll
          for (int j = 0; j < L::kPart; j += 4) {
            if constexpr (QUANT) {
              const uint4 e4 = lds128(my_scales + (L::kKeys + h * L::kPart + j) * 4);
              const float2 x = fma2(make_float2(sv[j], sv[j + 1]), mul_2, make_float2(__uint_as_float(e4.x), __uint_as_float(e4.y)));
              const float2 y = fma2(make_float2(sv[j + 2], sv[j + 3]), mul_2, make_float2(__uint_as_float(e4.z), __uint_as_float(e4.w)));
              mx0 = max3(mx0, x.x, x.y);
              mx1 = max3(mx1, y.x, y.y);
            } else {
              mx0 = max3(mx0, sv[j], sv[j + 1]);
              mx1 = max3(mx1, sv[j + 2], sv[j + 3]);
            }
          }
        }
        if (__builtin_expect(!plain, 0)) {
          // Values that no row sees are cleared: their probability is 0, and 0 times what lies there may be NaN.
          const uint32_t clear = __ballot_sync(0xffffffffu, !there(row_lane));
          if (clear) {
            // (P V of tile step - 2 is over: so is the previous use of the slot, without which its parity says nothing.)
            const int slot = step % L::kSlots;
            if ((step >= 2 && !warp_wait(SPLASH_KBAR(pv_done, buf), ((step - 2) >> 1) & 1, ctx, kCSiteSmxP, step)) ||
                !warp_wait(SPLASH_KBAR(v_full, slot), (step / L::kSlots) & 1, ctx, kCSiteSmxV, step)) { ok = false; break; }
            // The warp's 32 rows of the tile, 32 pieces of 16 bytes at a time.
            constexpr int kChunks = L::kBoxBytes / 16, kAtOnce = 32 / kChunks;
            const uint32_t dst = v_u32 + slot * L::kSlotBytes + (warp & 3) * 32 * L::kBoxBytes + (lane % kChunks) * 16;
#pragma unroll 1
            for (int k = lane / kChunks; k < 32; k += kAtOnce)
              if ((clear >> k) & 1u)
#pragma unroll
                for (int c = 0; c < L::kBoxes; ++c)
                  sts128(dst + c * (kCachedTile * L::kBoxBytes) + k * L::kBoxBytes, make_uint4(0, 0, 0, 0));
            fence_proxy_async_smem();
          }
        }

        // ---- online softmax with a maximum that may lag behind ----
        float top = fmaxf(mx0, mx1);
        if constexpr (!QUANT) top *= mul;
        if (i > 0) {
          // The maximum that the previous tile settled on; this warpgroup's sum moves there first.
          if (!wait_m(step - 1)) { ok = false; break; }
          const float m_prev = m_got;
          if (m_prev != m_run) {
            l_run = m_run == -INFINITY ? (l_run == l_run ? 0.f : l_run) : l_run * ex2_approx(m_run - m_prev);
            m_run = m_prev;
          }
        }
        const float m_new = fmaxf(m_run, top);
        const bool moved = m_new - m_run > kThreshold;  // false for NaN (-inf - -inf)
        float alpha = 1.f;
        if (moved) {
          alpha = ex2_approx(m_run - m_new);  // 0 when m_run was -inf
          m_run = m_new;
          l_run *= alpha;
        }
        sts64(m_sh, static_cast<uint64_t>(__float_as_uint(m_run)) << 32 | static_cast<uint32_t>(step));
        // P's columns are free once P.V of this warpgroup's previous tile is done.
        if (step >= 2 && !warp_wait(SPLASH_KBAR(pv_done, buf), ((step - 2) >> 1) & 1, ctx, kCSiteSmxP, step)) { ok = false; break; }
        const float shift = m_run == -INFINITY ? 0.f : kExpBits - m_run;
        const float2 shift_2 = make_float2(shift, shift);
        float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
        // P is written 32 keys at a time: 16 columns of 16-bit numbers, or 8 columns of every e5m2 term, each 32 columns behind
        // the one before.
#pragma unroll
        for (int c = 0; c < L::kKeys / 32; ++c) {
          constexpr int kChunks = L::kPart / 32;
          const int in_part = c % kChunks * 32;  // (the loop is unrolled)
          if (c >= kChunks && c % kChunks == 0) {
            fetch(c / kChunks);
            fetched(c / kChunks == L::kParts - 1);
            prepare(c / kChunks);
          }
          if constexpr (QUANT) {
            uint32_t codes[8][L::kPTerms];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at = c * 32 + j * 4;
              const uint4 v4 = lds128(my_scales + (2 * L::kKeys + at) * 4);
              const int in = in_part + j * 4;
              const float2 x = fma2(make_float2(sv[in], sv[in + 1]), mul_2, shift_2);
              const float2 y = fma2(make_float2(sv[in + 2], sv[in + 3]), mul_2, shift_2);
              const float2 ex = make_float2(ex2_approx(x.x), ex2_approx(x.y)), ey = make_float2(ex2_approx(y.x), ex2_approx(y.y));
              sum_a = add2(sum_a, ex);
              sum_b = add2(sum_b, ey);
              const float2 px = mul2(ex, make_float2(__uint_as_float(v4.x), __uint_as_float(v4.y)));
              const float2 py = mul2(ey, make_float2(__uint_as_float(v4.z), __uint_as_float(v4.w)));
              e5m2_terms<L::kPTerms>(pack2<false>(px.x, px.y), pack2<false>(py.x, py.y), codes[j]);
            }
#pragma unroll
            for (int t = 0; t < L::kPTerms; ++t) {
              uint32_t x[8];
              if (t < 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = codes[j][t];
                tmem_st8(p_tmem + t * 32 + col0 / 4 + c * 8, x);
                continue;
              }
              // (The other copies' keys are scores here, and not zeros from the start.  Rows without copies have read the scores of
              // columns 0 .. 63 when they write the first of these; the others they read from behind them.)
#pragma unroll
              for (int other = 0; other < KG; ++other) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = other == part ? codes[j][t] : 0u;
                tmem_st8(s_tmem + (t - 2) * 32 + other * (L::kKeys / 4) + c * 8, x);
              }
            }
          } else {
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 x = fma2(make_float2(sv[in_part + 2 * j], sv[in_part + 2 * j + 1]), mul_2, shift_2);
              const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              if (j & 1) sum_b = add2(sum_b, e); else sum_a = add2(sum_a, e);
              pk[j] = pack2<BF16>(e.x, e.y);
            }
            tmem_st16(p_tmem + col0 / 2 + c * 16, pk);
          }
        }
        l_run += (sum_a.x + sum_a.y) + (sum_b.x + sum_b.y);
        if (__builtin_expect(i > 0 && __any_sync(0xffffffffu, moved), 0)) {
          // O may be touched once P.V of the previous tile is done.
          if (!warp_wait(SPLASH_KBAR(pv_done, (step - 1) & 1), ((step - 1) >> 1) & 1, ctx, kCSiteSmxO, step)) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(o_tmem + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st32(o_tmem + c * 32, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        arrive(SPLASH_KBAR(p_ready, buf));
      }
      if (!ok) break;

      // ---- the parts of a row, added up: the sums of the warpgroups, and the copies of the rows ----
      const int last = step0 + n - 1;
      if (!wait_m(last)) { ok = false; break; }
      {
        const float m_fin = m_got;
        if (m_fin != m_run) {
          l_run = m_run == -INFINITY ? (l_run == l_run ? 0.f : l_run) : l_run * ex2_approx(m_run - m_fin);
          m_run = m_fin;
        }
      }
      // Sums of the warpgroups, by parity of the segment: a warp that still reads them has not freed O, without which the next
      // but one cannot end.
      const uint32_t l_u32 = ml_u32 + 128 * 8 + (seg & 1) * (256 * 4);
      sts32(l_u32 + threadIdx.x * 4, __float_as_uint(l_run));
      if (!group_sync()) { ok = false; break; }
      // (Maxima of other copies in shared memory: their next tile comes after the barriers of this epilogue.)
      float m_tot = m_run, l_tot = 0.f;
      if constexpr (KG > 1) {
#pragma unroll
        for (int src = 0; src < KG; ++src) m_tot = fmaxf(m_tot, __uint_as_float(lds32(ml_u32 + (src * L::kRows + r) * 8 + 4)));
      }
#pragma unroll
      for (int src = 0; src < KG; ++src) {
        const uint32_t at = (src * L::kRows + r) * 4;
        const float m = KG > 1 ? __uint_as_float(lds32(ml_u32 + 2 * at + 4)) : m_run;
        const float l = __uint_as_float(lds32(l_u32 + at)) + __uint_as_float(lds32(l_u32 + 512 + at));
        if (l != 0.f) l_tot += m == -INFINITY ? l : l * ex2_approx(m - m_tot);
      }
      const float l_mine = __uint_as_float(lds32(l_u32 + row_lane * 4)) + __uint_as_float(lds32(l_u32 + 512 + row_lane * 4));
      if (!warp_wait(SPLASH_KBAR(pv_done, last & 1), (last >> 1) & 1, ctx, kCSiteSmxDone, last)) { ok = false; break; }
      tc_fence_after();
      const bool whole = cur.whole;
      float w = m_run == -INFINITY ? 0.f : ex2_approx(m_run - m_tot);
      w *= 1.f / kVScale;
      if (l_mine != l_mine) w = l_mine;  // NaN: no maximum may have been met
      if (whole) w *= l_tot > 0.f || l_tot != l_tot ? 1.f / l_tot : 0.f;
      const long long out_row0 = static_cast<long long>(b * a.kv_heads + cur.seg_head) * a.rows + rt * L::kRows;
      const long long part0 = static_cast<long long>(2 * blockIdx.x + (seg > 0)) * L::kRows;
      if (seg == 0 && threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(cur.seg_entry, cur.seg_head, cur.seg_tile, g.tiles);
      if (grp == 0 && part == 0) {
        if (!whole) a.part_ml[part0 + r] = make_float2(m_tot - kExpBits, l_tot);
        else if (a.lse_out && row_all < a.rows)
          a.lse_out[out_row0 + r] = live && l_tot != 0.f ? (m_tot - kExpBits + lg2_approx(l_tot)) * kCachedLn2 : a.mask_value;
      }
      // Each warpgroup has one half of O's columns, 32 at a time: every copy's lanes leave theirs, eight threads add up the 128
      // bytes of a row.  Rows without copies stay within their warp, which waits for no other.
      const int col = (threadIdx.x % 8) * 4;
      const uint32_t my_stage = stage_u32 + grp * (128 * L::kStageStride * 4);
#pragma unroll 1
      for (int c = grp * (D / 64); c < (grp + 1) * (D / 64); ++c) {
        uint32_t o[32];
        tmem_ld32(o_tmem + c * 32, o);
        tmem_wait_ld();
        if (c == (grp + 1) * (D / 64) - 1) {
          tc_fence_before();
          arrive(SPLASH_KBAR(o_free, 0));
        }
        const uint32_t dst = my_stage + row_lane * (L::kStageStride * 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (live) {
            x.x = __float_as_uint(__uint_as_float(o[k * 4]) * w);
            x.y = __float_as_uint(__uint_as_float(o[k * 4 + 1]) * w);
            x.z = __float_as_uint(__uint_as_float(o[k * 4 + 2]) * w);
            x.w = __float_as_uint(__uint_as_float(o[k * 4 + 3]) * w);
          }
          sts128(dst + k * 16, x);
        }
        if constexpr (KG > 1) {
          if (!group_sync()) { ok = false; break; }
        } else {
          __syncwarp();
        }
#pragma unroll
        for (int k = 0; k < 8 / KG; ++k) {
          const int row = KG > 1 ? k * 16 + (threadIdx.x & 127) / 8 : (warp & 3) * 32 + k * 4 + lane / 8;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int src = 0; src < KG; ++src) {
            const uint4 x = lds128(my_stage + ((src * L::kRows + row) * L::kStageStride + col) * 4);
            acc.x += __uint_as_float(x.x);
            acc.y += __uint_as_float(x.y);
            acc.z += __uint_as_float(x.z);
            acc.w += __uint_as_float(x.w);
          }
          if (rt * L::kRows + row >= a.rows) continue;
          if (!whole) {
            *reinterpret_cast<float4*>(a.part_o + (part0 + row) * D + c * 32 + col) = acc;
          } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (out_row0 + row) * D + c * 32 + col) =
                make_uint2(pack2<BF16>(acc.x, acc.y), pack2<BF16>(acc.z, acc.w));
          }
        }
        if constexpr (KG > 1) {
          if (!group_sync()) { ok = false; break; }
        } else {
          __syncwarp();
        }
      }
      step0 += n;
    }
    // Units whose rows see no key stand nowhere in the line: zeros.
    if (ok) cached_fill_unseen<D>(a, static_cast<int>(threadIdx.x));
  }

  // ---- teardown: every thread of every role ends up here ----
  tc_fence_before();
  __syncthreads();
  if (const uint32_t gave_up = lds32(SPLASH_KWORD(abort_flag))) {
    if (threadIdx.x == 0) report_abort(a.status, gave_up, a.status_host);
    // Copies still in flight land before the shared memory goes to another CTA.
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000) {}
  }
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace splash
