// paged_common.cuh -- device helpers of both paged attention kernels.
#pragma once
#include "b200fa.h"
#include "paged.h"
#include "ptx.cuh"

namespace b200fa {

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y,
                                            int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y,
                                            int32_t z, int32_t u, int32_t v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v)
      : "memory");
}

// Two floats rounded to the cache's type (lo in bits 0..15).
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  } else {
    return pack_h2(lo, hi);
  }
}

// The pages of a worker's blocks for the producer warp.  The lanes read 32
// table entries at once, a batch ahead of their use, and leave the pages in
// shared memory; one lane then issues the copies of the batch's blocks alone.
// (Read block by block the entries' latency paced the producer; told lane by
// lane with shuffles, the steps between two copies did.)
// A page is num_pages -- outside the tensor, so the copy delivers zeros --
// where no row of the tile sees any of its keys, and where the table names no
// page of the cache, which is recorded.
struct PageFeed {
  const PagedParams& p;
  uint32_t slots;  // shared memory, 32 words
  int rows, per;   // keys of a page within a block; pages per block (at most 16)
  int next;        // this lane's entry of the next batch

  __device__ __forceinline__ PageFeed(const PagedParams& params, uint32_t smem) : p(params), slots(smem) {
    rows = p.page_shift < 7 ? 1 << p.page_shift : kPagedBlock;
    per = kPagedBlock / rows;
  }
  static constexpr int kNone = INT32_MIN;
  __device__ __forceinline__ int blocks_per_batch() const { return 32 / per; }
  __device__ __forceinline__ int entry(const PagedWalk& w, int step) const {
    if (step >= w.take * per) return kNone;
    const int j = step / per, key = w.blocks.key_block(w.off + j) * kPagedBlock + (step - j * per) * rows;
    const int at = key >> p.page_shift, k0 = at << p.page_shift;
    if (k0 >= w.blocks.end_key || (k0 + (1 << p.page_shift) <= w.blocks.first_key && k0 >= p.sinks)) return kNone;
    return at < p.width ? p.table[int64_t(w.r) * p.table_stride + at] : -1;
  }
  __device__ __forceinline__ void begin(const PagedWalk& w, uint32_t lane) { next = entry(w, int(lane)); }
  // The pages of blocks j .. j + blocks_per_batch() - 1, in order from j = 0.
  __device__ __forceinline__ void batch(const PagedWalk& w, int j, uint32_t lane) {
    int page = next;
    if (uint32_t(page) >= uint32_t(p.num_pages)) {
      if (page != kNone) paged_status(p, B200FA_DEV_PAGE, uint32_t(w.r));
      page = p.num_pages;
    }
    __syncwarp();  // the last batch has been read
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(slots + 4u * lane), "r"(page) : "memory");
    __syncwarp();
    next = entry(w, j * per + 32 + int(lane));
  }
  // Page i of the batch's block number b.
  __device__ __forceinline__ int operator()(int b, int i) const { return int(ld_volatile_shared(slots + 4u * uint32_t(b * per + i))); }
};

}  // namespace b200fa
