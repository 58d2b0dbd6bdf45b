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

// The page that holds key `key` of request r, for a load: num_pages (outside
// the tensor, so the copy delivers zeros) where no row of the tile sees any
// of the page's keys, or where the table names no page of the cache.
__device__ __forceinline__ int page_of(const PagedParams& p, int r, const PagedBlocks& b, int key) {
  const int size = 1 << p.page_shift, page = key >> p.page_shift, k0 = page << p.page_shift;
  if (k0 >= b.end_key || (k0 + size <= b.first_key && k0 >= p.sinks)) return p.num_pages;
  const int id = page < p.width ? p.table[int64_t(r) * p.table_stride + page] : -1;
  if (id >= 0 && id < p.num_pages) return id;
  paged_status(p, B200FA_DEV_PAGE, uint32_t(r));
  return p.num_pages;
}

}  // namespace b200fa
