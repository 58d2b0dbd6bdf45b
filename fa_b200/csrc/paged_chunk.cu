// paged_chunk.cu -- attention over a paged cache for many rows: chunks of
// prompts.  Bound by the tensor cores (4 * 128 * rows flops per key), so the
// products run as the dense attention kernel's do (fa_kernel.cuh; what the two
// share is in fa_pipeline.cuh): pairs of CTAs, tcgen05 cta_group::2, M = 256, S and PV issued by a thread
// each, two softmax warpgroups on alternate key blocks, TMA rings for K and V.
//
// What differs:
//   * a work item is a tile of new tokens times the heads that share their
//     keys (rank r of the pair holds the tile's r-th half), cut out of a
//     worker's stretch of the line of key blocks (paged.h); the worker is the
//     pair.  A Q tile is one box of the [tokens][heads_kv][group][128] view,
//     so its rows land in the order token * group + head.
//   * K and V come page by page, a box (K: one per 64 columns) for each page
//     of a block, K and V by a warp each, which read the block table 32
//     entries ahead.
//   * in a block that holds keys that no row of the item sees -- an item's
//     last, the last of the sinks', the first of the window's -- V is loaded in
//     smaller boxes, with zeros in those keys' places (load_seen_v).
//   * scores are masked in tensor memory before the softmax loads them.
//   * 4096 + 1024 tokens over 32768 + 20480 keys, 12 heads on 1: 829 us in short
//     bursts, 917 under the power cap, 979 TFLOP/s of visible products.
//   * an item that lies in the stretch is normalised and stored; one that a
//     stretch's end cuts leaves FP32 partial results, joined by
//     b200_paged_combine_kernel.
#include "b200fa.h"
#include "fa_pipeline.cuh"
#include "paged.h"
#include "paged_common.cuh"

namespace b200fa {
namespace chunk {

constexpr int kSmBar = kSmemV + kRing * kStageBytes;    // the dense kernel's barriers
constexpr int kSmXchg = kSmBar + kNumBars * 8;            // float [2][128]
constexpr int kSmTmem = kSmXchg + 2 * kBlockM * 4;      // TMEM base, abort flag
constexpr int kSmStart = kSmTmem + 16;                  // PagedStart
constexpr int kSmScan = kSmStart + 64;                  // int64 [12]
constexpr int kSmPages = kSmScan + (kThreads / 32) * 8;  // 32 page numbers for each producer
constexpr int kSmUsed = kSmPages + 256;
constexpr int kBytes = kSmUsed + 1024;
static_assert(kBytes <= 232448, "shared memory budget exceeded");
static_assert(kSmBar % 8 == 0 && kSmStart % 8 == 0 && kSmScan % 8 == 0 && sizeof(PagedStart) <= 64, "layout");

struct Sm {
  uint32_t base;
  __device__ __forceinline__ uint32_t bar(int i) const { return base + kSmBar + 8 * i; }
  __device__ __forceinline__ uint32_t q(int t) const { return base + kSmemQ + t * kQTileBytes; }
  __device__ __forceinline__ uint32_t k(uint32_t e) const { return base + kSmemK + e * kStageBytes; }
  __device__ __forceinline__ uint32_t v(uint32_t e) const { return base + kSmemV + e * kStageBytes; }
  __device__ __forceinline__ uint32_t xchg(uint32_t slot, int row) const { return base + kSmXchg + (slot * kBlockM + uint32_t(row)) * 4u; }
  __device__ __forceinline__ uint32_t tmem_slot() const { return base + kSmTmem; }
  __device__ __forceinline__ uint32_t abort_slot() const { return base + kSmTmem + 4; }
  __device__ __forceinline__ uint32_t pages(bool v) const { return base + kSmPages + (v ? 128 : 0); }
};

__device__ __forceinline__ Sm sm_of(uint8_t* raw) { return Sm{(smem_addr(raw) + 1023u) & ~1023u}; }
__device__ __forceinline__ const PagedStart* start_of(uint8_t* raw) {
  return reinterpret_cast<const PagedStart*>(raw + (sm_of(raw).base - smem_addr(raw)) + kSmStart);
}

// What a wait does every thousand probes: the time of the first such look (`t0`,
// 0 before it); a wait that runs out raises both CTAs' abort flags with its site,
// which it then finds.  Out of line: these few instructions at every wait of the
// hot loops cost 13 to 18 % of a chunk's time (4096 + 1024 tokens over 32768 +
// 20480 keys: 987 against 836 us; called like this: within 2 % of a count alone).
__device__ __noinline__ uint64_t wait_look(uint64_t t0, uint32_t abort_slot, uint64_t limit_ns, uint32_t site) {
  const uint64_t now = global_timer_ns();
  if (t0 == 0u) return now;
  if (now - t0 <= limit_ns) return t0;
  st_volatile_shared(abort_slot, site | 0x80000000u);
  st_cluster_u32(map_shared(abort_slot, cluster_rank() ^ 1u), site | 0x80000000u);
  return t0;
}

// Bounded waits.  A probe may suspend the thread, for about a microsecond, so a
// wait ends within its bound and some milliseconds; the other roles of the pair
// end with the one that gave up, and the teardown reports its site.
struct Wait {
  uint32_t abort_slot;
  const PagedParams* p;
  template <bool kCluster = false>
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity, uint32_t site) const {
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t n = 0;; ++n) {
      if (kCluster ? mbar_test_cluster(bar, parity) : mbar_test(bar, parity)) return true;
      if (ld_volatile_shared(abort_slot) != 0u) return false;
      if ((n & 1023u) == 1023u) t0 = wait_look(t0, abort_slot, p->timeout_ns, site);
    }
  }
  // Exit-path wait for copies and products under way; it ignores the abort slot
  // and gives up 100 ms after `t0`.
  __device__ __forceinline__ void drain(uint32_t bar, uint32_t parity, uint64_t t0) const {
    while (!mbar_test_cluster(bar, parity) && global_timer_ns() - t0 < 100000000ull) {}
  }
};

template <bool kBf16>
constexpr uint32_t kIdescS = kIdescQK | (kBf16 ? (1u << 7) | (1u << 10) : 0u);
template <bool kBf16>
constexpr uint32_t kIdescO = kIdescPV | (kBf16 ? (1u << 7) | (1u << 10) : 0u);

// Rank 0, one thread: S = Q K^T of every block.
template <bool kBf16>
__device__ __forceinline__ void s_issuer(const PagedParams& p, const PagedStart& start, const Sm& sm, uint32_t tmem, const Wait& wait) {
  const uint32_t site = uint32_t(kSIssuerWarp) << 8;
  uint32_t g = 0;
  bool ok = true;
  int it = 0;
  for (PagedWalk w(p, start); ok && w.more(); w.next(p), ++it) {
    const int qt = it & 1;
    const uint64_t q_desc = smem_desc(sm.q(qt));
    if (!wait(sm.bar(kBarQFull + qt), uint32_t(it >> 1) & 1u, site | uint32_t(kBarQFull + qt))) break;
    for (int j = 0; j < w.take; ++j, ++g) {
      const uint32_t b = buf(g), e = ring_entry(g);
      if ((g >= 2 && !wait(sm.bar(kBarSFree + int(b)), buf_parity(g - 2u), site | uint32_t(kBarSFree + int(b)))) ||
          !wait(sm.bar(kBarKFull + int(e)), ring_parity(g), site | uint32_t(kBarKFull + int(e)))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t k_desc = smem_desc(sm.k(e));
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        mma_pair_ss(tmem + kTmemS + 128u * b, q_desc + uint64_t((kk >> 2) * (kQHalfBytes >> 4) + (kk & 3) * 2),
                    k_desc + uint64_t((kk >> 2) * (kKBoxBytes >> 4) + (kk & 3) * 2), kIdescS<kBf16>, kk > 0 ? 1u : 0u);
      mma_commit_pair_both(sm.bar(kBarSFull + int(b)));
      mma_commit_pair_both(sm.bar(kBarKEmpty + int(e)));
    }
  }
  mma_commit_pair(sm.bar(kBarDrain + 0));
  wait.drain(sm.bar(kBarDrain + 0), 0u, global_timer_ns());
}

// Rank 0, one thread: O += P V of every block, in order.
template <bool kBf16>
__device__ __forceinline__ void pv_issuer(const PagedParams& p, const PagedStart& start, const Sm& sm, uint32_t tmem, const Wait& wait) {
  const uint32_t site = uint32_t(kPVIssuerWarp) << 8;
  uint32_t g = 0;
  bool ok = true;
  for (PagedWalk w(p, start); ok && w.more(); w.next(p)) {
    for (int j = 0; j < w.take; ++j, ++g) {
      const uint32_t b = buf(g), e = ring_entry(g);
      if (!wait(sm.bar(kBarVFull + int(e)), ring_parity(g), site | uint32_t(kBarVFull + int(e))) ||
          !wait(sm.bar(kBarPFull + int(b)), buf_parity(g), site | uint32_t(kBarPFull + int(b)))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t v_desc = smem_desc(sm.v(e));
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        mma_pair_ts(tmem + kTmemO, tmem + kTmemP + 64u * b + 8u * uint32_t(kk), v_desc + uint64_t(kk * 128), kIdescO<kBf16>,
                    kk > 0 || j > 0 ? 1u : 0u);
      mma_commit_pair_both(sm.bar(kBarPVDone + int(b)));
      mma_commit_pair_both(sm.bar(kBarVEmpty + int(e)));
    }
  }
  mma_commit_pair(sm.bar(kBarDrain + 1));
  wait.drain(sm.bar(kBarDrain + 1), 0u, global_timer_ns());
}

// Rank 1, one thread: passes its Q, K and V stages on to rank 0's barriers.
__device__ __forceinline__ void forward(const PagedParams& p, const PagedStart& start, const Sm& sm, const Wait& wait) {
  const uint32_t site = (1u << 16) | (uint32_t(kForwardWarp) << 8);
  uint32_t g = 0;
  int it = 0;
  auto pass = [&](int bar, uint32_t parity) -> bool {
    if (!wait(sm.bar(bar), parity, site | uint32_t(bar))) return false;
    mbar_arrive_cluster_relaxed(map_shared(sm.bar(bar), 0));
    return true;
  };
  for (PagedWalk w(p, start); w.more(); w.next(p), ++it) {
    if (!pass(kBarQFull + (it & 1), uint32_t(it >> 1) & 1u)) return;
    for (int j = 0; j < w.take; ++j, ++g) {
      const int e = int(ring_entry(g));
      if (!pass(kBarKFull + e, ring_parity(g)) || !pass(kBarVFull + e, ring_parity(g))) return;
    }
  }
}

// V of a block that holds keys that no row of the item sees: 0 times what may be
// an infinity or NaN is no 0, so zeros take their place.  Boxes of 8 keys, of
// single ones where a group of 8 is seen in part (a row's place in the swizzle
// goes by its address); the unseen ones name the page behind the cache, for
// which a copy delivers zeros.  At most 48 boxes, once to three times an item,
// and nothing else in the kernel has to know.  (Cleared after the copy instead,
// by warps between it and the products, chunks took up to 28 % longer: the loops
// of the issuing warps grew.)
// `pages`: shared memory, the block's page numbers; the keys before `end_key` and
// not between the sinks and `first_key` are seen.
__device__ __noinline__ void load_seen_v(const PagedParams& p, uint32_t pages, int end_key, int first_key, int key0, int h, int col,
                                         uint32_t dst, uint32_t bar) {
  const int size_mask = (1 << p.page_shift) - 1, shift = p.page_shift < 7 ? p.page_shift : 7;
#pragma unroll 1
  for (int c = 0; c < kPagedBlock; c += 8, dst += 1024u) {
    const int page = int(ld_volatile_shared(pages + 4u * uint32_t(c >> shift))), key = key0 + c;
    const uint32_t seen = bits_below(end_key - key) & (bits_below(p.sinks - key) | ~bits_below(first_key - key)) & 255u;
    if (seen == 0u || seen == 255u) {
      tma_load_4d(dst, &p.tm_v8, bar, col, key & size_mask, h, seen ? page : p.num_pages);
    } else {
#pragma unroll 1
      for (int i = 0; i < 8; ++i)
        tma_load_4d(dst + uint32_t(i) * 128u, &p.tm_v1, bar, col, (key + i) & size_mask, h, (seen >> i) & 1u ? page : p.num_pages);
    }
  }
}

// Both ranks, a warp each for Q and K and for V: this CTA's Q tiles and its
// halves of every block.  Two warps because a block of small pages is many
// copies (16-token pages: 8 of K, 8 of V), which one thread issued in more time
// than the products take (1.36 us a block of 16-token pages against 1.07 of
// 64-token ones).
template <bool kV>
__device__ __forceinline__ void load(const PagedParams& p, const PagedStart& start, const Sm& sm, const Wait& wait,
                                     uint32_t rank, uint32_t warp, uint32_t lane) {
  const uint32_t site = (rank << 16) | (warp << 8);
  const int half_tok = p.tokens_per_tile / 2;
  const uint32_t q_bytes = uint32_t(half_tok * p.group) * 256u;
  const int size_mask = (1 << p.page_shift) - 1;
  const int k_rows = p.page_shift < 6 ? 1 << p.page_shift : kPairKeys;  // of a K box: this rank's keys of a page
  if (kV && (p.flags & B200FA_PAGED_TEST_WITHHOLD_V)) return;
  uint32_t g0 = 0, issued = 0, q_issued = 0;  // issued, q_issued: in the issuing lane
  bool ok = true;
  int it = 0;
  // Bounded wait for a free stage, then the announcement of its bytes.
  auto claim = [&](int empty, uint32_t parity, int full, uint32_t bytes) -> bool {
    if (!wait(sm.bar(empty), parity, site | uint32_t(empty))) return false;
    mbar_arrive_expect_tx(sm.bar(full), bytes);
    return true;
  };
  PageFeed feed(p, sm.pages(kV));
  const int k_first = feed.per > 1 ? int(rank) * (feed.per / 2) : 0, k_pages = kPairKeys / k_rows;
  for (PagedWalk w(p, start); ok && w.more(); w.next(p), ++it) {
    feed.begin(w, lane);
    if (!kV && elect_one()) {
      const int qt = it & 1;
      if ((ok = claim(kBarQEmpty + qt, (uint32_t(it >> 1) & 1u) ^ 1u, kBarQFull + qt, q_bytes))) {
        const int tok = w.req.q0 + w.tile * p.tokens_per_tile + int(rank) * half_tok;
        tma_load_4d(sm.q(qt), &p.tm_q, sm.bar(kBarQFull + qt), 0, 0, w.h, tok);
        tma_load_4d(sm.q(qt) + kQHalfBytes, &p.tm_q, sm.bar(kBarQFull + qt), 64, 0, w.h, tok);
        ++q_issued;
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    for (int j0 = 0; ok && j0 < w.take; j0 += feed.blocks_per_batch()) {
      feed.batch(w, j0, lane);
      const int n = min(feed.blocks_per_batch(), w.take - j0);
      if (elect_one()) {
        for (int j = 0; j < n; ++j) {
          const uint32_t g = g0 + uint32_t(j), e = ring_entry(g);
          int key = w.blocks.key_block(w.off + j0 + j) * kPagedBlock;
          if constexpr (!kV) {
            if (!(ok = claim(kBarKEmpty + int(e), ring_parity(g) ^ 1u, kBarKFull + int(e), kStageBytes))) break;
            uint32_t dst = sm.k(e);
            key += int(rank) * kPairKeys;
            for (int i = 0; i < k_pages; ++i, dst += uint32_t(k_rows) * 128u, key += k_rows) {
              const int page = feed(j, k_first + i);
              tma_load_4d(dst, &p.tm_k, sm.bar(kBarKFull + int(e)), 0, key & size_mask, w.h, page);
              tma_load_4d(dst + kKBoxBytes, &p.tm_k, sm.bar(kBarKFull + int(e)), 64, key & size_mask, w.h, page);
            }
          } else {
            const int bar = kBarVFull + int(e);
            if (!(ok = claim(kBarVEmpty + int(e), ring_parity(g) ^ 1u, bar, kStageBytes))) break;
            uint32_t dst = sm.v(e);
            if (w.blocks.unseen(p, key)) {
              load_seen_v(p, feed.slots + 4u * uint32_t(j * feed.per), w.blocks.end_key, w.blocks.first_key, key, w.h,
                          int(rank) * kPairDims, dst, sm.bar(bar));
            } else {
              for (int i = 0; i < feed.per; ++i, dst += uint32_t(feed.rows) * 128u, key += feed.rows)
                tma_load_4d(dst, &p.tm_v, sm.bar(bar), int(rank) * kPairDims, key & size_mask, w.h, feed(j, i));
            }
          }
          ++issued;
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      g0 += uint32_t(n);
    }
  }
  // The last copies land before the CTA exits, also when a role gave up.
  if (elect_one()) {
    const uint64_t t0 = global_timer_ns();
    const int full = kV ? kBarVFull : kBarKFull;
    for (uint32_t i = issued > kRing ? issued - kRing : 0; i < issued; ++i) wait.drain(sm.bar(full + int(ring_entry(i))), ring_parity(i), t0);
    for (uint32_t i = q_issued > 2 ? q_issued - 2 : 0; i < q_issued; ++i) wait.drain(sm.bar(kBarQFull + int(i & 1u)), (i >> 1) & 1u, t0);
  }
  __syncwarp();
}

// Exponentials of 64 keys of one row: P rounded to the cache's type, as the
// tensor cores take it (errors against 64 bits are 2.3e-3 beside 1.7e-3 with P in
// 32 bits in BF16, 3.0e-4 beside 2.1e-4 in FP16), and four chains of FP32 sums of
// the unrounded values.  All through MUFU: with one pair of eight on the FMA pipe, as in
// the dense kernel, chunks took 4 to 10 % longer here (4 x 512 tokens over 32768
// keys, 12 heads on 1: 248 against 225 us) -- the pipe's turn comes while the
// other group loads and reduces, and the loop is shorter without it.
template <bool kBf16>
__device__ __forceinline__ void exp64(const uint32_t* r, uint64_t sl2x2, uint64_t nmx2, uint32_t* pk, uint64_t* acc) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float a, b;
    f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), sl2x2, nmx2), a, b);
    a = ex2_approx(a);
    b = ex2_approx(b);
    pk[i] = pack2<kBf16>(a, b);
    acc[i & 3] = f2_add(acc[i & 3], f2_pack(a, b));
  }
}

// Masks this thread's row of a block's scores in tensor memory, before the
// softmax loads it (mask_window of fa_kernel.cuh, in place).  A masked block
// takes some 2000 cycles longer than with selects on the loaded registers, but
// the loop that most blocks of a long context run is shorter by those selects:
// 866 against 922 us for 4096 + 1024 tokens over 32768 + 20480 keys, the same
// within 2 % for short chunks and windows.
__device__ __forceinline__ void mask_scores(uint32_t tS, int valid, int lo, int sink) {
#pragma unroll 1
  for (int c0 = 0; c0 < kBlockN; c0 += 32) {
    const uint32_t keep = bits_below(valid - c0) & (~bits_below(lo - c0) | bits_below(sink - c0));
    if (__all_sync(0xffffffffu, keep == 0xffffffffu)) continue;
    uint32_t s[32];
    tmem_ld32(tS + uint32_t(c0), s);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if ((keep & (1u << i)) == 0u) s[i] = __float_as_uint(-INFINITY);
    tmem_st32(tS + uint32_t(c0), s);
  }
  tmem_wait_st();
}

// The softmax of the CTA's half tile: group grp takes the item's blocks j with
// j % 2 == grp, one thread per row; fa_kernel.cuh's softmax_role on the walk.
template <bool kBf16>
__device__ __forceinline__ void softmax(const PagedParams& p, const PagedStart& start, const Sm& sm, uint32_t tmem,
                                        const Wait& wait, uint32_t warp, uint32_t lane, uint32_t rank) {
  const int grp = int(warp >> 2);
  const int row = int(warp & 3) * 32 + int(lane);
  const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
  const uint32_t tO = tmem + lane_off + kTmemO;
  const uint32_t site = (rank << 16) | (warp << 8);
  const float sl2 = p.scale_log2;
  const uint64_t sl2x2 = f2_pack(sl2, sl2);
  const int half_tok = p.tokens_per_tile / 2;
  const int row_tok = row / p.group + int(rank) * half_tok;  // this row's token in the tile
  constexpr float kFirstRef = -1e30f;  // finite: a row may see nothing of its first blocks
  auto arrive_rank0 = [&](int bar) {
    __syncwarp();
    if (lane == 0) {
      if (rank == 0) mbar_arrive(sm.bar(bar));
      else mbar_arrive_cluster_relaxed(map_shared(sm.bar(bar), 0));
    }
  };
  auto arrive_local = [&](int bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(sm.bar(bar));
  };
  auto wait_warp = [&](int bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, wait(sm.bar(bar), parity, site | uint32_t(bar)));
  };
  auto wait_pv = [&](uint32_t gp) -> bool { return wait_warp(kBarPVDone + int(buf(gp)), buf_parity(gp)); };
  bool ok = true;
  uint32_t g0 = 0;
  int it = 0;
  for (PagedWalk w(p, start); ok && w.more(); w.next(p), ++it) {
    const int n = w.take;
    const int pos = w.blocks.pos0 + row_tok;
    // Key blocks that some row of this CTA does not see in full: from its first
    // row's position on, and up to the end of its last row's window.
    const int first_pos = w.blocks.pos0 + int(rank) * half_tok, behind = first_pos + half_tok - 1 - p.window;
    const int kb_hi = first_pos > 0 ? (first_pos + 1) / kPagedBlock : 0;
    const int kb_lo = p.window > 0 && behind >= 0 ? behind / kPagedBlock : -1;
    float m_cur = kFirstRef, l_g = 0.f;
    for (int j = grp; j < n; j += 2) {
      const uint32_t gb = g0 + uint32_t(j);
      const uint32_t b = buf(gb);
      const uint32_t tS = tmem + lane_off + kTmemS + 128u * b;
      const uint32_t tP = tmem + lane_off + kTmemP + 64u * b;
      float m_prev = kFirstRef;
      if (!wait_warp(kBarSFull + int(b), buf_parity(gb))) {
        ok = false;
        break;
      }
      tc_fence_after();
      {
        const int kb = w.blocks.key_block(w.off + j);
        if (kb >= kb_hi || kb <= kb_lo) {
          const int valid = pos + 1 - kb * kPagedBlock;
          mask_scores(tS, valid, p.window > 0 ? valid - p.window : 0, p.sinks - kb * kPagedBlock);
        }
      }
      uint32_t r[kBlockN];
      tmem_ld128(tS, r);
      if (gb > 0) {
        if (!wait_warp(kBarRef + int((gb - 1u) & 1u), ((gb - 1u) >> 1) & 1u)) {
          tmem_wait_ld();
          ok = false;
          break;
        }
        if (j > 0) m_prev = ld_shared_f32(sm.xchg((gb - 1u) & 1u, row));
      }
      tmem_wait_ld();
      arrive_rank0(kBarSFree + int(b));
      const float mx = fmaxf(row_max64(r), row_max64(r + 64)) * sl2;
      if (j >= 2 && m_prev != m_cur) l_g *= ex2_approx(m_cur - m_prev);
      float m_new = m_prev, alpha = 1.f;
      bool moved = false;
      if (mx > m_prev + kRescaleLog2) {
        m_new = mx;
        moved = j > 0;
        alpha = ex2_approx(m_prev - mx);
      }
      st_shared_f32(sm.xchg(gb & 1u, row), m_new);
      arrive_local(kBarRef + int(gb & 1u));
      if (moved) l_g *= alpha;
      m_cur = m_new;
      uint32_t pk[kBlockN / 2];
      uint64_t acc[4] = {0ull, 0ull, 0ull, 0ull};
      const uint64_t nm = f2_pack(-m_new, -m_new);
      exp64<kBf16>(r, sl2x2, nm, pk, acc);
      exp64<kBf16>(r + 64, sl2x2, nm, pk + 32, acc);
      if (__any_sync(0xffffffffu, moved)) {
        if (!wait_pv(gb - 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        scale_o_row(tO, moved ? alpha : 1.f);
      }
      float a0, b0, a1, b1;
      f2_unpack(f2_add(acc[0], acc[2]), a0, b0);
      f2_unpack(f2_add(acc[1], acc[3]), a1, b1);
      l_g += (a0 + b0) + (a1 + b1);
      if (gb >= 2 && !wait_pv(gb - 2u)) {
        ok = false;
        break;
      }
      tc_fence_after();
      tmem_st32(tP, pk);
      tmem_st32(tP + 32u, pk + 32);
      tmem_wait_st();
      tc_fence_before();
      // The item's first product overwrites O: both groups have read the last
      // item's by then.
      if (j == 0 && it > 0 && warp == 0 && !wait_warp(kBarOStaged, uint32_t(it - 1) & 1u)) {
        ok = false;
        break;
      }
      arrive_rank0(kBarPFull + int(b));
    }
    if (!ok) break;

    // ---- the item's end: the row's sum, then O
    const uint32_t g_last = g0 + uint32_t(n) - 1u;
    g0 += uint32_t(n);
    float m_final = m_cur;
    if ((n - 1) % 2 != grp) {
      if (!wait_warp(kBarRef + int(g_last & 1u), (g_last >> 1) & 1u)) {
        ok = false;
        break;
      }
      m_final = ld_shared_f32(sm.xchg(g_last & 1u, row));
    }
    if (l_g != 0.f && m_final != m_cur) l_g *= ex2_approx(m_cur - m_final);
    // The groups' sums meet in the item's Q tile, which nothing reads any more
    // (a group here has seen, or waited for the reference after, the scores of
    // the last block), while the last product of P and V is under way.
    const uint32_t sums = sm.q(it & 1) + uint32_t(row) * 4u;
    st_shared_f32(sums + uint32_t(grp) * 512u, l_g);
    arrive_local(kBarXchg);
    if (!wait_warp(kBarXchg, uint32_t(it) & 1u)) {
      ok = false;
      break;
    }
    const float l = l_g + ld_shared_f32(sums + uint32_t(grp ^ 1) * 512u);  // 0: the row saw no key
    fence_proxy_async_smem();
    arrive_local(kBarQEmpty + (it & 1));
    if (!wait_pv(g_last)) {
      ok = false;
      break;
    }
    tc_fence_after();
    const int t0 = w.tile * p.tokens_per_tile;
    const int toks = w.req.len - t0 < p.tokens_per_tile ? w.req.len - t0 : p.tokens_per_tile;
    const bool real = row < half_tok * p.group && row_tok < toks;
    if (w.begins() && w.ends()) {
      const float inv_l = l > 0.f ? 1.f / l : 0.f;
      uint16_t* dst = static_cast<uint16_t*>(p.o) + int64_t(w.req.q0 + t0 + row_tok) * p.o_tok +
                      int64_t(w.h * p.group + row % p.group) * p.o_head + 64 * grp;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + 64u * uint32_t(grp) + 32u * uint32_t(c), o);
        tmem_wait_ld();
        if (real) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              h[i] = pack2<kBf16>(__uint_as_float(o[8 * u + 2 * i]) * inv_l, __uint_as_float(o[8 * u + 2 * i + 1]) * inv_l);
            *reinterpret_cast<uint4*>(dst + 32 * c + 8 * u) = make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
      }
    } else {
      const int worker = int(cluster_id_x());
      float* part = paged_partial(p, 2 * worker + (w.begins() ? 1 : 0));
      const int prow = row + int(rank) * half_tok * p.group;  // token * group + head in the tile
      float* dst = part + prow * 128 + 64 * grp;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + 64u * uint32_t(grp) + 32u * uint32_t(c), o);
        tmem_wait_ld();
        if (real) {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4*>(dst + 32 * c + 4 * u) =
                make_float4(__uint_as_float(o[4 * u]), __uint_as_float(o[4 * u + 1]), __uint_as_float(o[4 * u + 2]),
                            __uint_as_float(o[4 * u + 3]));
        }
      }
      if (real && grp == 0) {
        part[p.part_rows * 128 + prow] = m_final;
        part[p.part_rows * 129 + prow] = l;
      }
    }
    tc_fence_before();
    arrive_local(kBarOStaged);
  }
}

__device__ __forceinline__ void setup(const PagedParams& p, uint8_t* raw) {
  const Sm sm = sm_of(raw);
  uint8_t* smem = raw + (sm.base - smem_addr(raw));
  const uint32_t tid = tid_x();
  const uint32_t rank = cluster_rank();
  if (tid == 0) {
    const uint32_t fed = rank == 0 ? 2u : 1u;  // rank 0's full barriers also count rank 1's forward
    for (int t = 0; t < 2; ++t) {
      mbar_init(sm.bar(kBarQFull + t), fed);
      mbar_init(sm.bar(kBarQEmpty + t), 8);
      mbar_init(sm.bar(kBarSFull + t), 1);
      mbar_init(sm.bar(kBarSFree + t), kGroupWarps);
      mbar_init(sm.bar(kBarPFull + t), kGroupWarps);
      mbar_init(sm.bar(kBarPVDone + t), 1);
      mbar_init(sm.bar(kBarRef + t), 4);
      mbar_init(sm.bar(kBarDrain + t), 1);
    }
    mbar_init(sm.bar(kBarXchg), 8);
    mbar_init(sm.bar(kBarOStaged), 8);
    for (int e = 0; e < kRing; ++e) {
      mbar_init(sm.bar(kBarKFull + e), fed);
      mbar_init(sm.bar(kBarKEmpty + e), 1);
      mbar_init(sm.bar(kBarVFull + e), fed);
      mbar_init(sm.bar(kBarVEmpty + e), 1);
    }
    st_volatile_shared(sm.abort_slot(), 0u);
    fence_mbarrier_init();
    tma_prefetch_map(&p.tm_q);
    tma_prefetch_map(&p.tm_k);
    tma_prefetch_map(&p.tm_v);
  }
  // Rows of a Q tile that no box covers stay zeros.
  for (uint32_t i = tid; i < 2 * kQTileBytes / 16; i += kThreads) st_shared_v4(sm.base + kSmemQ + i * 16u, 0, 0, 0, 0);
  fence_proxy_async_smem();
  grid_wait();
  grid_release();
  find_start(p, int(cluster_id_x()), reinterpret_cast<int64_t*>(smem + kSmScan), reinterpret_cast<PagedStart*>(smem + kSmStart));
  if ((tid >> 5) == 0) {
    __syncwarp();
    tmem_alloc_pair(sm.tmem_slot(), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
}

template <bool kBf16>
__device__ __forceinline__ void roles(const PagedParams& p, uint8_t* raw) {
  const Sm sm = sm_of(raw);
  const uint32_t tid = tid_x();
  const uint32_t warp = tid >> 5, lane = tid & 31u;
  if (warp < 8) {
    regs_increase<kSoftmaxRegs>();
    softmax<kBf16>(p, *start_of(raw), sm, ld_volatile_shared(sm.tmem_slot()), Wait{sm.abort_slot(), &p}, warp, lane, cluster_rank());
  } else {
    regs_decrease<kControlRegs>();
    const uint32_t rank = cluster_rank();
    const Wait wait{sm.abort_slot(), &p};
    const PagedStart& start = *start_of(raw);
    if (warp == kLoadWarp) {
      load<false>(p, start, sm, wait, rank, warp, lane);
    } else if (warp == (rank == 0 ? kForwardWarp : kPVIssuerWarp)) {
      load<true>(p, start, sm, wait, rank, warp, lane);
    } else if (warp == kForwardWarp) {
      if (elect_one()) forward(p, start, sm, wait);
    } else if (rank == 1) {
      if (lane == 0) write_record(p, start, int(cluster_id_x()));
    } else {
      const uint32_t tmem = ld_volatile_shared(sm.tmem_slot());
      if (elect_one()) {
        if (warp == kPVIssuerWarp) pv_issuer<kBf16>(p, start, sm, tmem, wait);
        else s_issuer<kBf16>(p, start, sm, tmem, wait);
      }
    }
  }
  __syncwarp();
}

__device__ __forceinline__ void teardown(const PagedParams& p, uint8_t* raw) {
  const Sm sm = sm_of(raw);
  tc_fence_before();
  cluster_sync();
  if (tid_x() == 0) {
    const uint32_t site = ld_volatile_shared(sm.abort_slot());
    if (site != 0u) paged_status(p, kDevTimeout, site & 0x7fffffffu);
  }
  if ((tid_x() >> 5) == 0) {
    tc_fence_after();
    tmem_dealloc_pair(ld_volatile_shared(sm.tmem_slot()), kTmemCols);
  }
}

}  // namespace chunk
}  // namespace b200fa

using namespace b200fa;

#define B200FA_PAGED_CHUNK_KERNEL(name, bf16)                                                                  \
  __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) name(const __grid_constant__ PagedParams p) { \
    extern __shared__ uint8_t smem_raw[];                                                                      \
    chunk::setup(p, smem_raw);                                                                                 \
    chunk::roles<bf16>(p, smem_raw);                                                                           \
    chunk::teardown(p, smem_raw);                                                                                \
  }
B200FA_PAGED_CHUNK_KERNEL(b200_paged_chunk_fp16_kernel, false)
B200FA_PAGED_CHUNK_KERNEL(b200_paged_chunk_bf16_kernel, true)

namespace b200fa {

PagedChunkKernel paged_chunk_kernel(bool bf16) { return bf16 ? b200_paged_chunk_bf16_kernel : b200_paged_chunk_fp16_kernel; }

int paged_chunk_setup(int* pairs) {
  cudaError_t e = cudaSuccess;
  for (bool bf16 : {false, true})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_chunk_kernel(bf16), cudaFuncAttributeMaxDynamicSharedMemorySize, chunk::kBytes);
  if (e != cudaSuccess) return int(e);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(2, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = chunk::kBytes;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(pairs, b200_paged_chunk_fp16_kernel, &cfg);
  if (e == cudaSuccess && *pairs < 1) e = cudaErrorInvalidConfiguration;
  return int(e);
}

int paged_chunk_launch(const PagedParams& p, bool bf16, cudaStream_t stream) {
  return int(launch_early(paged_chunk_kernel(bf16), dim3(unsigned(2 * p.workers)), dim3(kThreads), chunk::kBytes, stream, p));
}

}  // namespace b200fa
