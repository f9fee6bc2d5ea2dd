// TMA copies of a layer's pages into 128-byte swizzled tiles, and bounded waits,
// for the attention kernels on paged K/V.
#pragma once
#include <cuda.h>

#include "paged_attn.cuh"

namespace fa {

__device__ __forceinline__ void tma_2d(uint32_t dst, const void *map, int32_t x, int32_t y, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
               : "memory");
}

// Bounded wait of a whole warp; false, for all its lanes (they take the same
// way through later barriers and votes): it ran out here or elsewhere in the CTA
// (`abort`, in shared memory, is set).  The phase cannot pass while the warp
// waits: what completes the next one waits for the warp.  A try suspends the warp
// for 4 us at most, so 2^20 of them are four seconds (measured: 4.1).  The longest
// wait of a call that works is that of the warps that hold the next item's Q rows
// ready, for an item of 2^25 positions: 2^18 tiles of up to 4 us, a second.
constexpr uint32_t kWarpWaitTries = 1u << 20;
__device__ __forceinline__ bool wait_bar(uint32_t *abort, uint64_t *bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  uint32_t ok = 0;
  for (uint32_t i = 0; i < kWarpWaitTries && !ok; ++i) {
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(addr), "r"(parity)
                 : "memory");
    if ((i & 255) == 255 && *reinterpret_cast<volatile uint32_t *>(abort)) break;
  }
  if (__all_sync(0xFFFFFFFFu, ok)) return true;
  *reinterpret_cast<volatile uint32_t *>(abort) = 1;
  return false;
}

// The layer's pages as rows of a head: [page][k | v][kv head][16] x head_dim,
// boxes of `rows` rows x 64 elements, 128-byte swizzle.  False: the driver refused.
bool page_map(const AttnChunksParams &p, uint32_t rows, CUtensorMap *map);
// row of (page, k | v, head); a row past the end (zeros) for a bad or unused page
__device__ __forceinline__ int32_t map_row(const fa_pages &pg, uint32_t page, uint32_t is_v, uint32_t head) {
  return (int32_t)((page < pg.n_pages ? (page * 2 + is_v) * pg.n_kv_heads + head : pg.n_pages * 2 * pg.n_kv_heads) * kPageLen);
}

}  // namespace fa
