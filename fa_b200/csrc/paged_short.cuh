// paged_short.cuh -- attention over a paged cache for few rows: single tokens
// and short chunks (a tile of 16, 32 or 64 rows).
//
// Bound by reading the cache (2 bytes of K and V each per 4 * rows flops a
// key), so the layout serves the loads: one block per SM, one warp that does
// nothing but keep five 32 KiB entries of K and V in flight (a page per
// TMA box, in two halves of 64 columns, 128-byte swizzle), and eight warps that multiply with
// mma.sync -- 16 rows are an eighth of a tcgen05 tile, and the products are far
// from the limit (tensor pipe 15 % busy).  32 tokens over 4096..16384 keys, 32
// heads on 8: 222 us, 6.2 TB/s of the cache's bytes (212 us, 6.5 TB/s in short
// bursts); one token over 2048 keys, 12 heads on 1: 11 us with the join, a chain
// of latencies.  A warp owns 16 rows and a share of
// each block's keys (all eight share the keys of a 16-row tile) with its own
// running maximum, sum and output in registers; the shares are joined once,
// at the item's end, through shared memory.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "b200fa.h"
#include "paged.h"
#include "paged_common.cuh"
#include "ptx.cuh"

namespace b200fa {

constexpr int kShortWarps = 8;                       // consumers
// Three warpgroups, the last one for the producer: registers are handed out
// per four warps, and 384 x 168 = 256 x 208 + 128 x 88 leaves the consumers 208.
constexpr int kShortThreads = 384;
constexpr uint32_t kShortRegs = 208, kShortLoadRegs = 88;
constexpr int kShortRing = 5;
constexpr int kTileBytes = kPagedBlock * 256;        // K or V of a block
constexpr int kShortMergeBytes = 4 * 16 * 128 * 4;   // outputs of four warps
constexpr int kShortQBytes = 64 * 256;
constexpr int kSmRing = 0;
constexpr int kSmMerge = kShortRing * kTileBytes;
constexpr int kSmQ = kSmMerge + kShortMergeBytes;
constexpr int kSmMl = kSmQ + kShortQBytes;           // float2 [8 warps][16 rows]
constexpr int kSmBars = kSmMl + 8 * 16 * 8;
constexpr int kSmScan = kSmBars + 2 * kShortRing * 8;
constexpr int kSmStart = kSmScan + (kShortThreads / 32) * 8;
constexpr int kSmAbort = kSmStart + 64;
constexpr int kSmPages = kSmAbort + 16;              // 32 page numbers
constexpr int kShortSmemBytes = kSmPages + 128 + 1024;
static_assert(sizeof(PagedStart) <= 64 && kShortSmemBytes <= 232448, "shared memory budget");

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Bounded wait of one thread; false when the block gave up.
__device__ __forceinline__ bool paged_wait(const PagedParams& p, uint32_t bar, uint32_t parity, uint32_t abort_slot,
                                           uint32_t site) {
  if (mbar_test(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 16; ++i)
      if (mbar_test(bar, parity)) return true;
    if (ld_volatile_shared(abort_slot) != 0u) return false;
    if (global_timer_ns() - t0 > p.timeout_ns) {
      st_volatile_shared(abort_slot, 1u);
      paged_status(p, B200FA_DEV_TIMEOUT, site);
      return false;
    }
  }
}

// The producer warp: K and V of every block of the worker's stretch, a box per
// page with both 64-column halves.  One lane issues them all: copies issued by
// many lanes are taken one lane after another anyway, with more to do for each.
__device__ __forceinline__ void short_load(const PagedParams& p, const PagedStart& s, uint32_t sm, uint32_t lane) {
  const uint32_t abort_slot = sm + kSmAbort;
  const int size_mask = (1 << p.page_shift) - 1;
  uint32_t g = 0;     // ring uses: K, V of block 0, K, V of block 1, ...
  uint32_t last = 0;  // uses begun, in the issuing lane
  bool ok = true;
  PageFeed feed(p, sm + kSmPages);
  for (PagedWalk w(p, s); ok && w.more(); w.next(p)) {
    feed.begin(w, lane);
    for (int j0 = 0; ok && j0 < w.take; j0 += feed.blocks_per_batch()) {
      feed.batch(w, j0, lane);
      const int n = min(feed.blocks_per_batch(), w.take - j0);
      if (elect_one()) {
        for (int j = 0; ok && j < n; ++j) {
          const int key0 = w.blocks.key_block(w.off + j0 + j) * kPagedBlock;
          for (int kv = 0; kv < 2; ++kv) {
            if (kv && (p.flags & B200FA_PAGED_TEST_WITHHOLD_V)) {
              ok = false;
              break;
            }
            const uint32_t use = g + 2u * uint32_t(j) + uint32_t(kv), e = use % kShortRing;
            const uint32_t full = sm + kSmBars + 8 * e, empty = full + 8 * kShortRing;
            if (!(ok = paged_wait(p, empty, ((use / kShortRing) & 1u) ^ 1u, abort_slot, 0x800u | e))) break;
            mbar_arrive_expect_tx(full, kTileBytes);
            uint32_t dst = sm + kSmRing + e * kTileBytes;
            for (int i = 0; i < feed.per; ++i, dst += uint32_t(feed.rows) * 256u)
              tma_load_5d(dst, kv ? &p.tm_v : &p.tm_k, full, 0, (key0 + i * feed.rows) & size_mask, 0, w.h, feed(j, i));
            last = use + 1;
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      g += 2u * uint32_t(n);
    }
  }
  // The last copies land before the block exits, also when a warp gave up.
  if (elect_one()) {
    const uint64_t t0 = global_timer_ns();
    for (uint32_t i = last > kShortRing ? last - kShortRing : 0; i < last; ++i)
      while (!mbar_test(sm + kSmBars + 8 * (i % kShortRing), (i / kShortRing) & 1u) && global_timer_ns() - t0 < 100000000ull) {}
  }
  __syncwarp();
}

// Rows kM * 16 of a tile; kN = 8 / kM warps share a block's keys.
template <bool kBf16, int kM>
__device__ __forceinline__ void short_rows(const PagedParams& p, const PagedStart& s, uint32_t sm, uint8_t* smem,
                                           int worker, uint32_t warp, uint32_t lane) {
  constexpr int kN = kShortWarps / kM;
  constexpr int kKeys = kPagedBlock / kN;  // of a block, per warp
  constexpr int kTiles = kKeys / 8;        // score tiles of 8 keys
  const int wm = int(warp) % kM, wn = int(warp) / kM;
  const uint32_t abort_slot = sm + kSmAbort;
  const int quad = int(lane & 3), rq = int(lane >> 2);
  float2* ml = reinterpret_cast<float2*>(smem + kSmMl);
  float* merge = reinterpret_cast<float*>(smem + kSmMerge);
  // Byte offset of a key's row in a tile, [page][half][row][128 B], and the
  // distance of its halves.
  const int row_shift = p.page_shift < 7 ? p.page_shift : 7;
  const uint32_t half_bytes = 128u << row_shift;
  auto row_of = [&](int key) { return (uint32_t(key >> row_shift) * 2u << row_shift) * 128u + (uint32_t(key) & ((1u << row_shift) - 1u)) * 128u; };
  // This lane's rows for ldmatrix: of K (8 keys by 8 dims: keys, then dims) ...
  const int mi = int(lane >> 3), l8 = int(lane & 7);
  uint32_t k_off[kTiles / 2], v_off[kKeys / 16];
#pragma unroll
  for (int i = 0; i < kTiles / 2; ++i) k_off[i] = row_of(wn * kKeys + i * 16 + (mi >> 1) * 8 + l8);
  // ... and of V (keys and dims swapped).
#pragma unroll
  for (int i = 0; i < kKeys / 16; ++i) v_off[i] = row_of(wn * kKeys + i * 16 + (mi & 1) * 8 + l8);
  auto bar_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(kShortWarps * 32) : "memory"); };
  uint32_t g = 0;
  bool ok = true;

  for (PagedWalk w(p, s); w.more(); w.next(p)) {
    const int t0 = w.tile * p.tokens_per_tile;
    const int tok = min(p.tokens_per_tile, w.req.len - t0);
    const int rows = tok * p.group;
    // Q: rows beyond the tile's are zeros.
    {
      const uint16_t* q = static_cast<const uint16_t*>(p.q);
      for (int i = int(warp * 32 + lane); i < kM * 16 * 16; i += kShortWarps * 32) {
        const int row = i >> 4, c = i & 15;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < rows) {
          const int t = row / p.group, hd = row - t * p.group;
          v = *reinterpret_cast<const uint4*>(q + int64_t(w.req.q0 + t0 + t) * p.q_tok +
                                              int64_t(w.h * p.group + hd) * p.q_head + c * 8);
        }
        st_shared_v4(sm + kSmQ + uint32_t(row * 256 + ((c ^ (row & 7)) << 4)), v.x, v.y, v.z, v.w);
      }
    }
    bar_sync();
    uint32_t qf[8][4];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const int row = wm * 16 + int(lane & 15), c = kk * 2 + int(lane >> 4);
      ldsm4(sm + kSmQ + uint32_t(row * 256 + ((c ^ (row & 7)) << 4)), qf[kk]);
    }
    // Positions of this thread's two rows.
    const int ra = wm * 16 + rq, rb = ra + 8;
    const int pa = w.blocks.pos0 + ra / p.group, pb = w.blocks.pos0 + rb / p.group;
    const int la = p.window > 0 ? pa - p.window : -1, lb = p.window > 0 ? pb - p.window : -1;  // last key behind the window
    float o[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float ma = -1e30f, mb = -1e30f, suma = 0.f, sumb = 0.f;  // finite floor: a masked score stays -inf under it

    for (int j = w.off; j < w.off + w.take; ++j) {
      const int key0 = w.blocks.key_block(j) * kPagedBlock;
      const int wk0 = wn * kKeys;
      // ---- scores
      uint32_t e = g % kShortRing;
      ok = ok && paged_wait(p, sm + kSmBars + 8 * e, (g / kShortRing) & 1u, abort_slot, (warp << 8) | e);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint32_t tile = sm + kSmRing + e * kTileBytes;
      float sc[kTiles][4];
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) sc[i][u] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
#pragma unroll
        for (int i = 0; i < kTiles; i += 2) {
          const int c = (kk & 3) * 2 + (mi & 1);
          uint32_t b[4];
          ldsm4(tile + k_off[i / 2] + (kk >> 2) * half_bytes + uint32_t((c ^ l8) << 4), b);
          mma16816<kBf16>(sc[i], qf[kk], b[0], b[1]);
          mma16816<kBf16>(sc[i + 1], qf[kk], b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(sm + kSmBars + 8 * (kShortRing + e));
      ++g;
      // ---- mask, running maximum
      const bool edge = key0 + kPagedBlock > w.blocks.pos0 + 1 || (p.window > 0 && key0 <= w.blocks.pos0 + tok - 1 - p.window);
      if (edge) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int key = key0 + wk0 + i * 8 + quad * 2 + (u & 1);
            const int pos = u < 2 ? pa : pb, out = u < 2 ? la : lb;
            if (key > pos || (key <= out && key >= p.sinks)) sc[i][u] = -INFINITY;
          }
      }
      float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        xa = max3(xa, sc[i][0], sc[i][1]);
        xb = max3(xb, sc[i][2], sc[i][3]);
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, d));
        xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, d));
      }
      const float na = fmaxf(ma, xa * p.scale_log2), nb = fmaxf(mb, xb * p.scale_log2);
      const float fa = ex2_approx(ma - na), fb = ex2_approx(mb - nb);
      ma = na;
      mb = nb;
      suma *= fa;
      sumb *= fb;
      if (__any_sync(0xffffffffu, fa != 1.f || fb != 1.f)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i][0] *= fa, o[i][1] *= fa, o[i][2] *= fb, o[i][3] *= fb;
      }
      // P is rounded to the cache's type, as the tensor cores take it: errors
      // against 64 bits are 2.2e-3 beside 1.7e-3 with P in 32 bits (BF16), 2.5e-4
      // beside 2.2e-4 (FP16).  Its sum is that of the unrounded values.
      uint32_t pf[kTiles][2];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const float e0 = ex2_approx(fmaf(sc[i][0], p.scale_log2, -na)), e1 = ex2_approx(fmaf(sc[i][1], p.scale_log2, -na));
        const float e2 = ex2_approx(fmaf(sc[i][2], p.scale_log2, -nb)), e3 = ex2_approx(fmaf(sc[i][3], p.scale_log2, -nb));
        suma += e0 + e1;
        sumb += e2 + e3;
        pf[i][0] = pack2<kBf16>(e0, e1);
        pf[i][1] = pack2<kBf16>(e2, e3);
      }
      // ---- output
      e = g % kShortRing;
      ok = paged_wait(p, sm + kSmBars + 8 * e, (g / kShortRing) & 1u, abort_slot, (warp << 8) | 0x80u | e);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tile = sm + kSmRing + e * kTileBytes;
      if (w.blocks.unseen(p, key0)) {
        // Values at keys that no row of the item sees may be anything, and
        // 0 * NaN is no 0: this warp's rows of them are cleared.
        for (int part = 0; part < 2; ++part) {
          const int2 keys = w.blocks.unseen_keys(p, key0, part);
          const int from = max(wk0, keys.x), to = min(wk0 + kKeys, keys.y);
          for (int i = int(lane); i < (to - from) * 16; i += 32)
            st_shared_v4(tile + row_of(from + (i >> 4)) + (i & 1) * half_bytes + uint32_t((i >> 1) & 7) * 16u, 0, 0, 0, 0);
        }
        fence_proxy_async_smem();  // the next copy into this entry follows these writes
        __syncwarp();
      }
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk) {
        const uint32_t a[4] = {pf[2 * kk][0], pf[2 * kk][1], pf[2 * kk + 1][0], pf[2 * kk + 1][1]};
#pragma unroll
        for (int d = 0; d < 8; ++d) {  // 16 columns at a time
          const int c = (d & 3) * 2 + (mi >> 1);
          uint32_t b[4];
          ldsm4_trans(tile + v_off[kk] + (d >> 2) * half_bytes + uint32_t((c ^ l8) << 4), b);
          mma16816<kBf16>(o[2 * d], a, b[0], b[1]);
          mma16816<kBf16>(o[2 * d + 1], a, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(sm + kSmBars + 8 * (kShortRing + e));
      ++g;
    }
    // After an abort every warp still takes part in the barriers below, so
    // that none waits for one that left; what is written is then meaningless
    // and the status says so.
    // ---- join the warps' shares
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      suma += __shfl_xor_sync(0xffffffffu, suma, d);
      sumb += __shfl_xor_sync(0xffffffffu, sumb, d);
    }
    if (quad == 0) {
      ml[warp * 16 + rq] = make_float2(ma, suma);
      ml[warp * 16 + rq + 8] = make_float2(mb, sumb);
    }
    bar_sync();
    float top_a = -1e30f, top_b = -1e30f, la_sum = 0.f, lb_sum = 0.f;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      top_a = fmaxf(top_a, ml[(n * kM + wm) * 16 + rq].x);
      top_b = fmaxf(top_b, ml[(n * kM + wm) * 16 + rq + 8].x);
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const float2 a = ml[(n * kM + wm) * 16 + rq], b = ml[(n * kM + wm) * 16 + rq + 8];
      la_sum += a.y * ex2_approx(a.x - top_a);
      lb_sum += b.y * ex2_approx(b.x - top_b);
    }
    const float ga = ex2_approx(ma - top_a), gb = ex2_approx(mb - top_b);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i][0] *= ga, o[i][1] *= ga, o[i][2] *= gb, o[i][3] *= gb;
#pragma unroll
    for (int half = kN / 2; half >= 1; half >>= 1) {  // shares [half, 2 half) are added to [0, half)
      float* mine = merge + ((wn - half) * kM + wm) * 2048;
      if (wn >= half && wn < 2 * half) {
#pragma unroll
        for (int i = 0; i < 16; ++i) *reinterpret_cast<float4*>(mine + (i * 32 + int(lane)) * 4) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
      }
      bar_sync();
      if (wn < half) {
        const float* theirs = merge + (wn * kM + wm) * 2048;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float4 v = *reinterpret_cast<const float4*>(theirs + (i * 32 + int(lane)) * 4);
          o[i][0] += v.x, o[i][1] += v.y, o[i][2] += v.z, o[i][3] += v.w;
        }
      }
      bar_sync();
    }
    // ---- write: the whole item's result, or this stretch's part of it
    if (wn == 0) {
      if (w.begins() && w.ends()) {
        const float ia = la_sum > 0.f ? 1.f / la_sum : 0.f, ib = lb_sum > 0.f ? 1.f / lb_sum : 0.f;
        uint16_t* out = static_cast<uint16_t*>(p.o);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = half ? rb : ra;
          if (row < rows) {
            const int t = row / p.group, hd = row - t * p.group;
            uint16_t* dst = out + int64_t(w.req.q0 + t0 + t) * p.o_tok + int64_t(w.h * p.group + hd) * p.o_head;
            const float f = half ? ib : ia;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              *reinterpret_cast<uint32_t*>(dst + i * 8 + quad * 2) = pack2<kBf16>(o[i][2 * half] * f, o[i][2 * half + 1] * f);
          }
        }
      } else {
        float* part = paged_partial(p, 2 * worker + (w.begins() ? 1 : 0));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          *reinterpret_cast<float2*>(part + ra * 128 + i * 8 + quad * 2) = make_float2(o[i][0], o[i][1]);
          *reinterpret_cast<float2*>(part + rb * 128 + i * 8 + quad * 2) = make_float2(o[i][2], o[i][3]);
        }
        float* tail = part + p.part_rows * 128;
        if (quad == 0) {
          tail[ra] = top_a;
          tail[rb] = top_b;
          tail[p.part_rows + ra] = la_sum;
          tail[p.part_rows + rb] = lb_sum;
        }
      }
    }
    // One decision for all eight warps: a warp that went on alone would wait
    // at the next item's barrier for the ones that left.
    uint32_t failed;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(failed)
        : "r"(ok ? 0u : 1u), "n"(kShortWarps * 32)
        : "memory");
    if (failed) break;
  }
}

template <bool kBf16, int kM>
__device__ __forceinline__ void paged_short_body(const PagedParams& p) {
  extern __shared__ uint8_t raw[];
  const uint32_t sm = (smem_addr(raw) + 1023u) & ~1023u;
  uint8_t* smem = raw + (sm - smem_addr(raw));
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int e = 0; e < kShortRing; ++e) {
      mbar_init(sm + kSmBars + 8 * e, 1);
      mbar_init(sm + kSmBars + 8 * (kShortRing + e), kShortWarps);
    }
    st_volatile_shared(sm + kSmAbort, 0u);
    fence_mbarrier_init();
    tma_prefetch_map(&p.tm_k);
    tma_prefetch_map(&p.tm_v);
  }
  grid_wait();
  grid_release();
  PagedStart* start = reinterpret_cast<PagedStart*>(smem + kSmStart);
  find_start(p, int(blockIdx.x), reinterpret_cast<int64_t*>(smem + kSmScan), start);
  if (warp < kShortWarps) {
    regs_increase<kShortRegs>();
    short_rows<kBf16, kM>(p, *start, sm, smem, int(blockIdx.x), warp, lane);
  } else {
    regs_decrease<kShortLoadRegs>();
    if (warp == kShortWarps) short_load(p, *start, sm, lane);
    else if (threadIdx.x == kShortThreads - 1) write_record(p, *start, int(blockIdx.x));
  }
}

}  // namespace b200fa
