// Attention over an 8-bit paged cache for few rows: up to 16 new tokens x heads of a kv head, as in token-by-token decoding.
//
// cached_kernel.cuh spends an MMA's 128 rows on copies of the few rows there are, and its products then take about as long as
// an 8-bit tile's transfer (32 sequences of 2000 to 32768 keys, 64 / 8 heads: 278 us; here 196).  Here the keys are the 128
// rows instead:
//   S^T = K Q^T       [128 keys x rows]        A = K as it lies in the cache, B = Q, 16 to 48 columns
//   O^T += V^T P^T    [head_dim x rows]        A = V^T (V read M-major), B = P^T, which a key's thread writes as 32 to 64 bytes
// An MMA costs its 4 KB of A, 32 cycles: 256 a tile, where the copies cost 1280.  A thread has one key and all rows: the
// scales of the key and its value are two numbers of its own, and no exponential is computed twice.
//
// The rows' maxima lie across the threads now.  They are not looked for: a thread compares its scores with the lagging maxima
// (the same in every warp of a warpgroup), and only if one of the warpgroup's threads is above by 2^lag do the
// four warps reduce, agree on new maxima and rescale their warpgroup's O.  The two warpgroups take the tiles in turn, each
// with maxima, sums and O of its own, joined at the end of a segment.
//
// Q is 2 (bf16) or 3 (f16) e4m3 terms side by side in B, whose columns of S are added; P is 3 (bf16) or 4 (f16) terms of e5m2 (see
// e5m2_terms), side by side as well, whose columns of O are added.
//
// Maxima and factors of the rows are in shared memory between the tiles: with them in registers 16 rows need more than a thread
// has, and what is spilled comes back from L2, as shared memory leaves the L1 cache next to nothing (173 us instead of 105).
//
// Not here: 16-bit caches, whose tiles take twice as long to arrive while the copies' products take no longer than here (192
// us there, 203 here for 16 sequences of 4000 to 32768 keys, 32 / 8 heads).
#pragma once

#include "cached_common.cuh"

namespace splash {

template <int D, bool BF16, int R>
struct CachedFewLayout {
  static constexpr int kTerms = BF16 ? 2 : 3;
  static constexpr int kSCols = (kTerms * R + 15) / 16 * 16;  // N of the scores: a multiple of 16
  static constexpr int kPTerms = BF16 ? 3 : 4;
  static constexpr int kOCols = (kPTerms * R + 15) / 16 * 16;  // N of P V
  static constexpr int kItem = 1, kRowBytes = D, kBoxBytes = D, kBoxes = 1, kBoxElems = D;  // a key: one box of 64 or 128 bytes
  static constexpr int kSlotBytes = kCachedTile * kRowBytes;
  static constexpr int kQBytes = (kSCols * D + 1023) / 1024 * 1024;  // of one of two buffers
  // P^T: core matrices of 8 keys x 16 bytes one after the other, and 2 KB on the next 16 columns.
  static constexpr int kPBlock = kCachedTile * 16;
  static constexpr int kPBytes = kCachedTile * kOCols;
  static constexpr int kBarBytes = 512;
  static constexpr int kAuxBytes = kCachedAuxSlots * 2 * kCachedTile;
  static constexpr int kQScaleSlots = 8;                      // (four buffers of scores: see cached_split_q)
  static constexpr int kQScaleBytes = kQScaleSlots * R * 4;
  static constexpr int kVoteBytes = 2 * 2 * 16;               // by warpgroup and parity of its tiles: a word per warp
  static constexpr int kMaxBytes = 8 * R * 4;                 // per warp: maxima of its keys
  static constexpr int kStateBytes = 8 * R * 8;                // per warp: maxima, and the rows' factors
  static constexpr int kSumBytes = 2 * (8 + 2) * R * 4;       // by parity of the segment: sums per warp, maxima per warpgroup
  static constexpr int kRowInfoBytes = 8 * R * 16;            // per warp: what each row sees
  static constexpr int kTreeBytes = kCachedMaxTree * 8 + 2 * kCachedMaxTree * 8 * 4;
  static constexpr int kFixed = 1024 + 2 * kQBytes + 2 * kPBytes + kBarBytes + kAuxBytes + kQScaleBytes + kVoteBytes +
                                kMaxBytes + kStateBytes + kSumBytes + kRowInfoBytes + kTreeBytes;
  static constexpr int kSlotsFit = (227 * 1024 - kFixed) / (2 * kSlotBytes);
  static constexpr int kSlots = kSlotsFit < kCachedMaxSlots ? kSlotsFit : kCachedMaxSlots;
  static constexpr int kSmem = kFixed + 2 * kSlots * kSlotBytes;
  // Tensor memory: four buffers of scores, O of the two warpgroups.
  static constexpr int kOCol = 4 * kSCols;
  static constexpr int kTmemCols = kOCol + 2 * kOCols > 256 ? 512 : 256;
  static_assert(kOCol + 2 * kOCols <= kTmemCols, "");
  static constexpr int kSoftmaxRegs = 184, kLoadRegs = 136;   // 384 * 168 = 256 * 184 + 128 * 136
};

template <int D, bool BF16, int R>
__global__ void __launch_bounds__(kCachedThreads, 1)
cached_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const CachedArgs a) {
  using L = CachedFewLayout<D, BF16, R>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t q_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t k_u32 = q_u32 + 2 * L::kQBytes;
  const uint32_t v_u32 = k_u32 + L::kSlots * L::kSlotBytes;
  const uint32_t p_u32 = v_u32 + L::kSlots * L::kSlotBytes;
  const uint32_t bars_u32 = p_u32 + 2 * L::kPBytes;
  const uint32_t aux_u32 = bars_u32 + L::kBarBytes;
  const uint32_t vote_u32 = aux_u32 + L::kAuxBytes;
  const uint32_t qscale_u32 = vote_u32 + L::kVoteBytes;
  const uint32_t max_u32 = qscale_u32 + L::kQScaleBytes;
  const uint32_t state_u32 = max_u32 + L::kMaxBytes;
  const uint32_t sum_u32 = state_u32 + L::kStateBytes;
  const uint32_t info_u32 = sum_u32 + L::kSumBytes;
  const uint32_t parents_u32 = info_u32 + L::kRowInfoBytes;
  const uint32_t trees_u32 = parents_u32 + 2 * kCachedMaxTree * 4;

  const int warp = uniform_warp_index();
  const int lane = threadIdx.x & 31;
  const WaitCtx ctx{SPLASH_KWORD(abort_flag)};

  if (warp == 8) {
    cached_init_barriers(bars_u32, lane);
    if (lane == 0) {
      launch_dependents();
      sts32(SPLASH_KWORD(abort_flag), 0);
      sts32(SPLASH_KWORD(dead), a.status[0] != 0);
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
  } else if (warp == 9) {
    tmem_alloc(SPLASH_KWORD(tmem_base), L::kTmemCols);
    tmem_relinquish();
  } else if (warp == 10) {
    // No votes yet; and zeros in rows of Q that no term fills (the scores' columns are a multiple of 16).
    if (lane < L::kVoteBytes / 4) sts32(vote_u32 + lane * 4, 0xffffffffu);
    for (int i = lane; i < 2 * L::kQBytes / 16; i += 32) sts128(q_u32 + i * 16, make_uint4(0, 0, 0, 0));
    fence_proxy_async_smem();
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
      tmem_dealloc(tmem, L::kTmemCols);
    }
    return;
  }
  CachedCursor cur;
  cur.start(a, lds32(SPLASH_KWORD(first_entry)), lds32(SPLASH_KWORD(first_head)), lds32(SPLASH_KWORD(first_offset)),
            lds32(SPLASH_KWORD(share)));

  if (warp >= 8) {
    setmaxnreg_dec<L::kLoadRegs>();
    if (warp == 8 || warp == 11) {
      // ------------------------------------------ loads: keys (and exponents), values -----------------------------------
      const bool is_v = warp == 11;
      cached_load<L, true>(a, cur, bars_u32, is_v ? v_u32 : k_u32, aux_u32, is_v ? &tm_v : &tm_k, is_v, lane, ctx, [](int, int, int) {});
    } else if (warp == 9) {
      // ------------------------------------------ products -----------------------------------------------------------
      constexpr uint32_t kHi = cached_desc_hi<L::kBoxBytes>();
      constexpr uint32_t kPHi = desc_hi_plain(L::kPBlock);  // N-major without swizzle
      constexpr uint32_t kIdescS = make_idesc(false, 128, L::kSCols, false, false);
      constexpr uint32_t kIdescO = make_idesc(false, 128, L::kOCols, true, true) | (1u << 10);  // B is e5m2
      // An MMA takes 32 of a key's numbers, or 32 keys.  V^T has 128 rows; at head_dim 64 they are the 64 of its box twice, whose
      // second half is not read (distance 0 from one box to the next).
      const int tiles = cached_share_tiles(a, cur);
      CachedWalk qk, pv;
      uint32_t spins = 0;
      uint64_t t0 = 0;
      while (pv.step < tiles) {
        bool issued = false;
        {
          const int grp = pv.step & 1, slot = pv.step % L::kSlots;
          const bool ready = mbar_probe(SPLASH_KBAR(p_ready, grp), (pv.step >> 1) & 1) &&
                             mbar_probe(SPLASH_KBAR(v_full, slot), (pv.step / L::kSlots) & 1) &&
                             // O may be written again once the previous segment's has been read.
                             (pv.i > 0 || pv.seg == 0 || mbar_probe(SPLASH_KBAR(o_free, 0), (pv.seg - 1) & 1));
          if (__all_sync(0xffffffffu, ready)) {
            tc_fence_after();
            pv.at_tile(bars_u32);
            const uint32_t a_lo = desc_lo(v_u32 + slot * L::kSlotBytes, 0);
            const uint32_t b_lo = desc_lo_plain(p_u32 + grp * L::kPBytes, 128);
            const uint32_t o_tmem = tmem + L::kOCol + grp * L::kOCols;
#pragma unroll
            for (int kk = 0; kk < kCachedTile / 32; ++kk)
              umma8_ss2_w(o_tmem, a_lo + ((kk * 32 * D) >> 4), kHi, b_lo + ((kk * 32 * 16) >> 4), kPHi, kIdescO, pv.i > 1 || kk > 0);
            umma_commit_w(SPLASH_KBAR(v_empty, slot));
            umma_commit_w(SPLASH_KBAR(pv_done, grp));
            pv.advance();
            issued = true;
          }
        }
        if (qk.step < tiles) {
          const int buf = qk.step & 3, slot = qk.step % L::kSlots;
          const bool ready = mbar_probe(SPLASH_KBAR(k_full, slot), (qk.step / L::kSlots) & 1) &&
                             (qk.step < 4 || mbar_probe(SPLASH_KBAR(s_free, buf), ((qk.step - 4) >> 2) & 1)) &&
                             (qk.i > 0 || mbar_probe(SPLASH_KBAR(q_full, qk.seg & 1), (qk.seg >> 1) & 1));
          if (__all_sync(0xffffffffu, ready)) {
            tc_fence_after();
            qk.at_tile(bars_u32);
            const uint32_t a_lo = desc_lo(k_u32 + slot * L::kSlotBytes, 16), b_lo = desc_lo(q_u32 + (qk.seg & 1) * L::kQBytes, 16);
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
              umma8_ss2_w(tmem + buf * L::kSCols, a_lo + kk * 2, kHi, b_lo + kk * 2, kHi, kIdescS, kk > 0);
            umma_commit_w(SPLASH_KBAR(s_ready, buf));
            umma_commit_w(SPLASH_KBAR(k_empty, slot));
            if (qk.i + 1 == qk.n) umma_commit_w(SPLASH_KBAR(q_free, qk.seg & 1));
            qk.advance();
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
    } else if (warp == 10) {
      // ------------------------------ drafted trees, and Q as e4m3 terms, ahead of their use ------------------------------
      int trees = 0, last = -1;
      for (int seg = 0; cur.next(a); ++seg) {
        const int b = cur.seg_entry / a.row_tiles, rt = cur.seg_entry - b * a.row_tiles;
        if (a.parents != nullptr && b != last) {
          last = b;
          if (!cached_make_tree(a, b, cur.g.before, trees++, bars_u32, parents_u32, lane, ctx)) break;
        }
        auto store = [&](int t, int r, uint32_t byte, uint32_t codes) {
          sts_bytes<D / 32>(q_u32 + (seg & 1) * L::kQBytes + cached_swz<L::kBoxBytes>(t * R + r, byte >> 4) + (byte & 15u), codes);
        };
        if (!cached_split_q<D, BF16, L::kTerms, R, 2, L::kQScaleSlots>(a, seg, b, rt, cur.seg_head, bars_u32, qscale_u32, lane, ctx, store)) break;
      }
    }
  } else {
    // ============================================ softmax ==============================================================
    setmaxnreg_inc<L::kSoftmaxRegs>();
    if (threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);  // (its first segment overwrites it)
    const int grp = warp >> 2, quarter = warp & 3;
    const int key_lane = quarter * 32 + lane;   // key of a tile; row of O^T
    const uint32_t tmem_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t o_tmem = tmem_lane + L::kOCol;
    const uint32_t p_row = p_u32 + grp * L::kPBytes + key_lane * 16;
    const uint32_t my_info = info_u32 + warp * (R * 16);
    const uint32_t my_state = state_u32 + warp * (R * 8);
    auto load4 = [&](uint32_t at, float* x) {
      const uint4 w = lds128(at);
      x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
    };
    const int piece_shift = min(a.page_shift, 7);
    const bool tree = a.parents != nullptr;
    const bool capped = a.soft_cap > 0.f;
    // What takes a score to powers of 2, or to the argument of the soft-cap and from there to powers of 2.
    const float pre = capped ? 1.f / a.soft_cap : kCachedLog2e, post = a.soft_cap * kCachedLog2e;
    constexpr float kThreshold = kCachedLag8;  // powers of 2 by which the maxima may lag behind
    constexpr float kVScale = kCachedVScale8, kExpBits = kCachedExpBits8;
    uint32_t sync_par = 0;
    int step0 = 0;           // tiles of the CTA in front of the segment
    int trees = 0, last_b = -1;
    bool ok = true;
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
    // The four warps of a warpgroup on one question, asked once a tile and once more where the answer was yes: a word
    // (ballot number, answer) per warp, of two sets in turn -- a warp is at most one ballot ahead of the slowest.
    uint32_t ballots = 0;
    auto vote = [&](bool yes, bool& any) -> bool {
      const uint32_t set = vote_u32 + (grp * 2 + (ballots & 1)) * 16;
      const uint32_t want = ballots & 0x7fffffffu;
      ++ballots;
      __syncwarp();
      if (lane == 0) sts32(set + quarter * 4, want << 1 | (yes ? 1u : 0u));
      uint64_t t0 = 0;
      for (uint32_t spins = 0;; ++spins) {
        uint64_t lo = lds64(set), hi = lds64(set + 8);
        const uint32_t w0 = static_cast<uint32_t>(lo), w1 = static_cast<uint32_t>(lo >> 32), w2 = static_cast<uint32_t>(hi), w3 = static_cast<uint32_t>(hi >> 32);
        const bool all = (w0 >> 1) == want && (w1 >> 1) == want && (w2 >> 1) == want && (w3 >> 1) == want;
        if (__all_sync(0xffffffffu, all)) {
          any = (w0 | w1 | w2 | w3) & 1u;
          return true;
        }
        if ((spins & 0xff) == 0xff) {
          const uint64_t now = global_timer_ns();
          if (t0 == 0) t0 = now;
          bool give_up = lds32(SPLASH_KWORD(abort_flag)) != 0;
          if (!give_up && now - t0 > kWaitLimitNs) {
            sts32(SPLASH_KWORD(abort_flag), 0x80000000u | (static_cast<uint32_t>(kCSiteSmxM) << 20));
            give_up = true;
          }
          if (__any_sync(0xffffffffu, give_up)) return false;
        }
      }
    };

    for (int seg = 0; ok && cur.next(a); ++seg) {
      const CachedGeom& g = cur.g;
      const int n = cur.seg_n;
      const int b = cur.seg_entry / a.row_tiles, rt = cur.seg_entry - b * a.row_tiles;
      if (tree && b != last_b) {
        if (last_b >= 0) arrive(SPLASH_KBAR(tree_free, (trees - 1) & 1));
        last_b = b;
        if (!warp_wait(SPLASH_KBAR(tree_full, trees & 1), (trees >> 1) & 1, ctx, kCSiteSmxTree, seg)) { ok = false; break; }
        ++trees;
      }
      // What each row sees, a lane per row: keys [lo, hi) and [0, sink), and the words of its node in a tree.
      __syncwarp();
      uint32_t live = 0;  // bit r: row r is a new token's
      {
        const int row_all = rt * R + lane;
        const int node = row_all % a.n;
        const bool alive = lane < R && row_all < a.rows && node < g.count;
        uint32_t above = 0;
        int depth = node;
        if (tree) {
          above = trees_u32 + (((trees - 1) & 1) * kCachedMaxTree + node) * 32;
          depth = static_cast<int>(lds32(above + 28));
        }
        const int position = g.before + depth;
        const int v_hi = !alive ? 0 : (tree ? g.before : position + 1);
        const int v_lo = a.window < 0 ? 0 : max(0, position - a.window);
        const int v_sink = a.window < 0 ? 0 : min(a.sinks, v_hi);
        if (lane < R)
          sts128(my_info + lane * 16, make_uint4(v_lo, v_hi, v_sink, alive ? above : 0u));
        live = __ballot_sync(0xffffffffu, alive);
      }
      __syncwarp();
      const int seen_by_all = g.before + (tree ? 0 : g.i0 + 1);  // keys in front of this are behind no row
      const int all_from = a.window < 0 ? 0 : g.before + g.i1 - 1 - a.window;
      const int32_t* table = a.page_table + b * a.table_stride;
      const int pages = kCachedTile >> piece_shift;
      auto page_of = [&](int i) -> int {  // lane p: page id of piece p of tile i (anything for pieces nobody sees)
        if (i >= n || lane >= pages) return 0;
        const int key = cur.key0(i) + (lane << piece_shift);
        int id = 0;  // (asked for here, whatever the compiler thinks of its use a tile later)
        if (key < g.hi) asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(id) : "l"(table + (key >> a.page_shift)));
        return id;
      };
      float l[R];  // this key's sums
#pragma unroll
      for (int r = 0; r < R; ++r) l[r] = 0.f;
      // Maxima of s + ev (powers of 2; the same in every warp of the warpgroup) and the factors of the rows' scores: in shared
      // memory and not in registers between the tiles.  Rows that are none have factor 0 and never call for new maxima.
      if (lane < R) sts32(my_state + lane * 4, __float_as_uint(-INFINITY));
      __syncwarp();
      const int i0 = (grp ^ step0) & 1;  // the CTA's tiles alternate between the warpgroups, whatever segment they are of
      int page = page_of(i0);

      for (int i = i0; i < n; i += 2) {
        const int step = step0 + i, buf = step & 3;
        const int key0 = cur.key0(i), key = key0 + key_lane;
        asm volatile("" : "+r"(page));  // looked at here and not where it was asked for, a tile ago
        const uint32_t good = __ballot_sync(0xffffffffu, page >= 0 && page < a.num_pages);  // pieces that have a page
        page = page_of(i + 2);
        const bool plain = key0 + kCachedTile <= seen_by_all && (key0 >= all_from || key0 + kCachedTile <= g.sink_hi) &&
                           good == 0xffffffffu;
        // Whether this thread's key is there for some row; others may hold anything, and nothing was loaded for some.
        const bool there = key < g.hi && (key >= g.lo || key < g.sink_hi) && ((good >> (key_lane >> piece_shift)) & 1u);
        if (!warp_wait(SPLASH_KBAR(s_ready, buf), (step >> 2) & 1, ctx, kCSiteSmxS, step)) { ok = false; break; }
        tc_fence_after();
        uint32_t raw[L::kSCols];
#pragma unroll
        for (int c = 0; c < L::kSCols; c += 16) tmem_ld16(tmem_lane + buf * L::kSCols + c, raw + c);
        float k_scale = 1.f, v_exp = 0.f, v_scale = kVScale;
        // The key's own scales, and once the rows'.  (The exponents came with the keys, for which the scores waited.)
        if (i == i0) {
          if (lane < R)
            sts32(my_state + (R + lane) * 4,
                  (live >> lane) & 1u ? __float_as_uint(pre * __uint_as_float(lds32(qscale_u32 + (seg % L::kQScaleSlots * R + lane) * 4))) : 0u);
          __syncwarp();
        }
        if (there) {
          const uint32_t at = aux_u32 + (step % kCachedAuxSlots) * (2 * kCachedTile) + key_lane;
          const int ek = lds_s8(at), ev = lds_s8(at + kCachedTile);
          k_scale = exponent_scale(ek);
          v_exp = static_cast<float>(ev);
          v_scale = exponent_scale(ev) * kVScale;
        }
        tmem_wait_ld();
        tc_fence_before();
        arrive(SPLASH_KBAR(s_free, buf));  // the scores of tile step + 4 may come
        float x[R];  // scores in powers of 2
#pragma unroll
        for (int r4 = 0; r4 < R; r4 += 4) {
          float mul[4];
          load4(my_state + (R + r4) * 4, mul);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = r4 + k;
            x[r] = __uint_as_float(raw[r]);
#pragma unroll
            for (int t = 1; t < L::kTerms; ++t) x[r] += __uint_as_float(raw[t * R + r]);
            x[r] *= k_scale * mul[k];
          }
        }
        if (__builtin_expect(capped, 0)) {
#pragma unroll
          for (int r = 0; r < R; ++r) x[r] = tanh_approx(x[r]) * post;
        }
        if (__builtin_expect(!plain, 0)) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const uint4 info = lds128(my_info + r * 16);
            bool seen = (key >= static_cast<int>(info.x) && key < static_cast<int>(info.y)) || key < static_cast<int>(info.z);
            const int d = key - g.before;
            if (info.w != 0 && d >= 0 && d < kCachedMaxTree) seen = seen || ((lds32(info.w + (1 + (d >> 5)) * 4) >> (d & 31)) & 1u);
            if (!seen || !there) x[r] = -INFINITY;
          }
          // Values that no row sees are cleared: their probability is 0, and 0 times what lies there may be NaN.
          const uint32_t clear = __ballot_sync(0xffffffffu, !there);
          if (clear) {
            // (P V of tile step - 2 is over: so is the previous use of the slot, without which its parity says nothing.)
            const int slot = step % L::kSlots;
            if ((step >= 2 && !warp_wait(SPLASH_KBAR(pv_done, grp), ((step - 2) >> 1) & 1, ctx, kCSiteSmxP, step)) ||
                !warp_wait(SPLASH_KBAR(v_full, slot), (step / L::kSlots) & 1, ctx, kCSiteSmxV, step)) { ok = false; break; }
            // The warp's 32 rows of the tile, 32 pieces of 16 bytes at a time.
            constexpr int kChunks = L::kBoxBytes / 16, kAtOnce = 32 / kChunks;
            const uint32_t dst = v_u32 + slot * L::kSlotBytes + quarter * 32 * L::kBoxBytes + (lane % kChunks) * 16;
#pragma unroll 1
            for (int k = lane / kChunks; k < 32; k += kAtOnce)
              if ((clear >> k) & 1u)
#pragma unroll
                for (int c = 0; c < L::kBoxes; ++c)
                  sts128(dst + c * (kCachedTile * L::kBoxBytes) + k * L::kBoxBytes, make_uint4(0, 0, 0, 0));
          }
        }
        // ---- does a score stand above the maxima by more than they may lag? ----
        bool above = false;
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          float m[4];
          load4(my_state + r * 4, m);
#pragma unroll
          for (int k = 0; k < 4; ++k) above = above || x[r + k] + v_exp > m[k] + kThreshold;  // (-inf + lag is -inf)
        }
        bool move;
        if (!vote(__any_sync(0xffffffffu, above), move)) { ok = false; break; }
        if (__builtin_expect(move, 0)) {
          // New maxima where they are above by that much: of the warp by exchange, of the warpgroup through shared memory.
          const uint32_t mine = max_u32 + warp * (R * 4);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            // Floats that order like integers, for the one instruction that takes a maximum over a warp.
            const int bits = __float_as_int(x[r] + v_exp);
            const int top = __reduce_max_sync(0xffffffffu, bits ^ ((bits >> 31) & 0x7fffffff));
            if (lane == 0) sts32(mine + r * 4, static_cast<uint32_t>(top ^ ((top >> 31) & 0x7fffffff)));
          }
          bool unused;
          __threadfence_block();
          if (!vote(false, unused)) { ok = false; break; }
          __threadfence_block();
          // O may be touched once P V of this warpgroup's previous tile is done.
          if (i >= 2 && !warp_wait(SPLASH_KBAR(pv_done, grp), ((step - 2) >> 1) & 1, ctx, kCSiteSmxO, step)) { ok = false; break; }
          tc_fence_after();
          float alpha[R], m[R];
#pragma unroll
          for (int r = 0; r < R; r += 4) load4(my_state + r * 4, m + r);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float t = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) t = fmaxf(t, __uint_as_float(lds32(max_u32 + ((grp * 4 + w) * R + r) * 4)));
            alpha[r] = 1.f;
            if (t > m[r] + kThreshold) {
              alpha[r] = ex2_approx(m[r] - t);  // 0 when m was -inf
              m[r] = t;
              l[r] *= alpha[r];
            }
          }
          __syncwarp();  // (all have read the old ones)
          if (lane == 0) {
#pragma unroll
            for (int r = 0; r < R; r += 4)
              sts128(my_state + r * 4, make_uint4(__float_as_uint(m[r]), __float_as_uint(m[r + 1]), __float_as_uint(m[r + 2]), __float_as_uint(m[r + 3])));
          }
          __syncwarp();
          if (i >= 2) {
#pragma unroll
            for (int c = 0; c < L::kOCols; c += 16) {
              uint32_t o[16];
              tmem_ld16(o_tmem + grp * L::kOCols + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha[(c + k) % R]);
              tmem_st16(o_tmem + grp * L::kOCols + c, o);
            }
            tmem_wait_st();
          }
        }
        // ---- P ----
        uint32_t pk[L::kOCols / 4] = {};
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          float p[4], m[4];
          load4(my_state + r * 4, m);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float shift = m[k] == -INFINITY ? 0.f : kExpBits - m[k];
            const float e = ex2_approx(x[r + k] + shift);
            l[r + k] += e;
            p[k] = e * v_scale;
          }
          uint32_t codes[L::kPTerms];
          e5m2_terms<L::kPTerms>(pack2<false>(p[0], p[1]), pack2<false>(p[2], p[3]), codes);
#pragma unroll
          for (int t = 0; t < L::kPTerms; ++t) pk[t * (R / 4) + r / 4] = codes[t];
        }
        // P's room is free once P V of this warpgroup's previous tile is done.
        if (step >= 2 && !warp_wait(SPLASH_KBAR(pv_done, grp), ((step - 2) >> 1) & 1, ctx, kCSiteSmxP, step)) { ok = false; break; }
#pragma unroll
        for (int c = 0; c < L::kOCols / 16; ++c)
          sts128(p_row + c * L::kPBlock, make_uint4(pk[c * 4], pk[c * 4 + 1], pk[c * 4 + 2], pk[c * 4 + 3]));
        fence_proxy_async_smem();
        tc_fence_before();
        arrive(SPLASH_KBAR(p_ready, grp));
      }
      if (!ok) break;

      // ---- the parts of a row, added up: the sums of the keys, the two warpgroups ----
      const uint32_t sums = sum_u32 + (seg & 1) * (10 * R * 4), maxima = sums + 8 * R * 4;
      {
        // Sums over the warp's keys: the lanes halve the rows between them until each has one, lane / (32 / R).
#pragma unroll
        for (int s = 1; s < R; s *= 2) {
          const bool upper = lane & (16 / s);
#pragma unroll
          for (int k = 0; k < R / 2 / s; ++k) {
            const float low = l[k], high = l[k + R / 2 / s];
            l[k] = (upper ? high : low) + __shfl_xor_sync(0xffffffffu, upper ? low : high, 16 / s);
          }
        }
#pragma unroll
        for (int d = 16 / R; d > 0; d /= 2) l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
        if ((lane & (32 / R - 1)) == 0) sts32(sums + (warp * R + lane / (32 / R)) * 4, __float_as_uint(l[0]));
      }
      if (quarter == 0 && lane < R) sts32(maxima + (grp * R + lane) * 4, lds32(my_state + lane * 4));
      if (!group_sync()) { ok = false; break; }
      // (Both warpgroups are past their tiles, so the barrier's phase before the last tile's is over.)
      const int last = step0 + n - 1;
      if (!warp_wait(SPLASH_KBAR(pv_done, last & 1), (last >> 1) & 1, ctx, kCSiteSmxDone, last)) { ok = false; break; }
      tc_fence_after();
      const bool whole = cur.whole;
      const bool has[2] = {n > 1 || !(step0 & 1), n > 1 || (step0 & 1)};  // which warpgroups had a tile
      // Warpgroup g writes its half of the rows, a thread one number of each: of 8 rows' columns of every term, from row `r0` on.
      const int r0 = R > 8 ? grp * 8 : 0;
      uint32_t o0[L::kPTerms * 8], o1[L::kPTerms * 8];
#pragma unroll
      for (int t = 0; t < L::kPTerms; ++t) {
        if (has[0]) tmem_ld8(o_tmem + t * R + r0, o0 + t * 8);
        if (has[1]) tmem_ld8(o_tmem + L::kOCols + t * R + r0, o1 + t * 8);
      }
      tmem_wait_ld();
      tc_fence_before();
      arrive(SPLASH_KBAR(o_free, 0));
      const long long out_row0 = static_cast<long long>(b * a.kv_heads + cur.seg_head) * a.rows + rt * R;
      const long long part0 = static_cast<long long>(2 * blockIdx.x + (seg > 0)) * R;
      if (seg == 0 && threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(cur.seg_entry, cur.seg_head, cur.seg_tile, g.tiles);
      // Lane r: what the warpgroups' numbers of row r count for.
      float m_tot, l_tot, w0, w1;
      {
        const int r = lane % R;
        const float m0 = __uint_as_float(lds32(maxima + r * 4)), m1 = __uint_as_float(lds32(maxima + (R + r) * 4));
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          l0 += __uint_as_float(lds32(sums + (w * R + r) * 4));
          l1 += __uint_as_float(lds32(sums + ((4 + w) * R + r) * 4));
        }
        m_tot = fmaxf(m0, m1);
        // A warpgroup that met no key has nothing to add, but its sum if that is NaN.
        w0 = m0 == -INFINITY ? 0.f : ex2_approx(m0 - m_tot);
        w1 = m1 == -INFINITY ? 0.f : ex2_approx(m1 - m_tot);
        l_tot = (l0 != 0.f ? (m0 == -INFINITY ? l0 : l0 * w0) : 0.f) + (l1 != 0.f ? (m1 == -INFINITY ? l1 : l1 * w1) : 0.f);
        const float scale = l_tot != l_tot ? l_tot : (whole ? (l_tot > 0.f ? 1.f / l_tot : 0.f) : 1.f) / kVScale;
        w0 *= scale;
        w1 *= scale;
        if (l_tot != l_tot) w0 = w1 = l_tot;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = r0 + k;
        const float w0_r = __shfl_sync(0xffffffffu, w0, r), w1_r = __shfl_sync(0xffffffffu, w1, r);
        if ((R == 8 && (k >= 4) != (grp == 1)) || rt * R + r >= a.rows) continue;
        float value = 0.f;
        if ((live >> r) & 1u) {
          auto all_terms = [&](const uint32_t* o) {
            float x = __uint_as_float(o[(L::kPTerms - 1) * 8 + k]);
#pragma unroll
            for (int t = L::kPTerms - 2; t >= 0; --t) x += __uint_as_float(o[t * 8 + k]);
            return x;
          };
          if (has[0]) value = all_terms(o0) * w0_r;
          if (has[1]) value = fmaf(all_terms(o1), w1_r, value);
        }
        if (key_lane >= D) continue;
        if (!whole) a.part_o[(part0 + r) * D + key_lane] = value;
        else static_cast<uint16_t*>(a.out)[(out_row0 + r) * D + key_lane] = static_cast<uint16_t>(pack2<BF16>(value, 0.f));
      }
      if (warp == 0 && lane < R && rt * R + lane < a.rows) {
        if (!whole) a.part_ml[part0 + lane] = make_float2(m_tot - kExpBits, l_tot);
        else if (a.lse_out)
          a.lse_out[out_row0 + lane] = ((live >> lane) & 1u) && l_tot != 0.f ? (m_tot - kExpBits + lg2_approx(l_tot)) * kCachedLn2 : a.mask_value;
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
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

}  // namespace splash
