// Copies of pages (fork) and in-place compaction of kept positions, over every
// layer of a paged cache.  Both only move bytes: HBM bounds them, one read and
// one write of what moves.
#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {
namespace {

constexpr uint32_t kCopyThreads = 256, kCopyUnroll = 4;

// grid (pieces of a page, pairs, layers): a page of one layer is 2 n_kv blocks
// of 16 rows (head, K or V), contiguous; the first `slots` rows of each block
// are copied, 16 bytes a thread and four loads in flight.  64 tails of 1 to 16
// rows, 8 heads x 128 f16, 32 layers: 37 us, 5.8 TB/s.
__global__ void __launch_bounds__(kCopyThreads) k_page_copy(const PageCopyParams p, uint32_t row16) {
  const uint32_t pair = blockIdx.y;
  const uint32_t src = p.src[pair], dst = p.dst[pair], slots = p.slots ? p.slots[pair] : kPageLen;
  uint32_t bad = 0;
  if (src >= p.pg.n_pages || dst >= p.pg.n_pages) bad = kFlagPage;
  else if (slots > kPageLen) bad = kFlagRange;
  if (bad) {
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, bad);
    return;
  }
  const uint32_t esz = p.pg.dtype == FA_KV_F32 ? 4 : 2;
  const uint32_t block16 = kPageLen * row16, page16 = 2 * p.pg.n_kv_heads * block16, take = slots * row16;
  const uint64_t layer = (uint64_t)blockIdx.z * p.pg.layer_stride * esz;
  const uint4 *s = reinterpret_cast<const uint4 *>(static_cast<const char *>(p.pg.base) + layer) + (uint64_t)src * page16;
  uint4 *d = reinterpret_cast<uint4 *>(static_cast<char *>(p.pg.base) + layer) + (uint64_t)dst * page16;
  const uint32_t n = 2 * p.pg.n_kv_heads * take;  // 16-byte pieces that move
  const uint32_t step = gridDim.x * kCopyThreads;
  for (uint32_t i0 = blockIdx.x * kCopyThreads + threadIdx.x; i0 < n; i0 += kCopyUnroll * step) {
    uint4 v[kCopyUnroll];
    uint32_t at[kCopyUnroll];
#pragma unroll
    for (uint32_t j = 0; j < kCopyUnroll; ++j) {
      const uint32_t i = i0 + j * step;
      at[j] = slots == kPageLen ? i : i / take * block16 + i % take;
      if (i < n) v[j] = __ldcs(s + at[j]);
    }
#pragma unroll
    for (uint32_t j = 0; j < kCopyUnroll; ++j)
      if (i0 + j * step < n) __stcs(d + at[j], v[j]);
  }
}

// grid (n_kv heads, K or V, layers x sequences); one CTA moves all kept rows of
// one (sequence, layer, K or V, head) in ascending order, a tile of them at a
// time.  keep ascends, so row j comes from keep[j] >= j: what a tile writes lies
// at or below its own sources and below every later tile's.  So a tile may be
// written as soon as it and all before it are read: the next tile is read
// ahead, a barrier, this one written.  Four sequences of 2048 positions thinned
// to half, 8 heads x 128 f16, 32 layers: 111 us, 5.2 TB/s (without reading
// ahead 139).
constexpr uint32_t kCompactThreads = 256, kCompactUnroll = 4;
__global__ void __launch_bounds__(kCompactThreads) k_page_compact(const PageCompactParams p, uint32_t row16) {
  const uint32_t h = blockIdx.x, is_v = blockIdx.y, layer = blockIdx.z % p.pg.n_layers, i = blockIdx.z / p.pg.n_layers;
  const uint32_t seq = p.seq[i], k0 = p.start[i], k1 = p.start[i + 1];
  const uint32_t cap = p.pg.max_pages * kPageLen;
  if (seq >= p.pg.n_seq || k1 < k0 || k1 > p.n_keep || k1 - k0 > cap) {
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, kFlagRange);
    return;
  }
  const uint32_t *pt = p.pg.page_table + (uint64_t)seq * p.pg.max_pages, *keep = p.keep + k0;
  const uint32_t n = k1 - k0, esz = p.pg.dtype == FA_KV_F32 ? 4 : 2;
  uint4 *base = reinterpret_cast<uint4 *>(static_cast<char *>(p.pg.base) + (uint64_t)layer * p.pg.layer_stride * esz);
  const uint64_t page16 = (uint64_t)2 * p.pg.n_kv_heads * kPageLen * row16;
  const uint64_t block = (uint64_t)(is_v * p.pg.n_kv_heads + h) * kPageLen * row16;
  const uint32_t total = n * row16;  // below 2^25 * 64: checked on the host
  uint32_t bad = 0;
  constexpr uint64_t kNone = ~0ull;
  struct Tile {
    uint4 v[kCompactUnroll];
    uint64_t to[kCompactUnroll];
  } cur, nxt;
  auto read = [&](uint32_t e0, Tile &t) {
#pragma unroll
    for (uint32_t u = 0; u < kCompactUnroll; ++u) {
      const uint32_t e = e0 + u * kCompactThreads + threadIdx.x, j = e / row16, c = e - j * row16;
      t.to[u] = kNone;
      if (e0 >= total || e >= total) continue;
      const uint32_t from = __ldg(keep + j);
      if (from < j || from >= cap || (j && __ldg(keep + j - 1) >= from)) {
        bad |= kFlagRange;
        continue;
      }
      if (from == j) continue;
      const uint32_t sp = __ldg(pt + from / kPageLen), dp = __ldg(pt + j / kPageLen);
      if (sp >= p.pg.n_pages || dp >= p.pg.n_pages) {
        bad |= kFlagPage;
        continue;
      }
      t.v[u] = __ldcs(base + sp * page16 + block + (from % kPageLen) * row16 + c);
      t.to[u] = dp * page16 + block + (j % kPageLen) * row16 + c;
    }
  };
  read(0, cur);
  for (uint32_t e0 = 0; e0 < total; e0 += kCompactThreads * kCompactUnroll) {
    read(e0 + kCompactThreads * kCompactUnroll, nxt);
    __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < kCompactUnroll; ++u)
      if (cur.to[u] != kNone) __stcs(base + cur.to[u], cur.v[u]);
    cur = nxt;
  }
  if (bad && p.err) atomicOr(p.err, bad);
}

}  // namespace

int launch_page_copy(const PageCopyParams &p, cudaStream_t st) {
  const uint32_t row16 = p.pg.head_dim * elem_size(p.pg.dtype) / 16, page16 = 2 * p.pg.n_kv_heads * kPageLen * row16;
  uint32_t pieces = (page16 + kCopyThreads * kCopyUnroll - 1) / (kCopyThreads * kCopyUnroll);
  if (pieces > 4096) pieces = 4096;
  for (uint32_t n0 = 0; n0 < p.n; n0 += 65535) {  // grid y and z end at 65535
    for (uint32_t l0 = 0; l0 < p.pg.n_layers; l0 += 65535) {
      PageCopyParams q = p;
      q.src += n0;
      q.dst += n0;
      if (q.slots) q.slots += n0;
      q.pg.base = static_cast<char *>(q.pg.base) + (uint64_t)l0 * q.pg.layer_stride * elem_size(q.pg.dtype);
      const uint32_t ny = p.n - n0 < 65535 ? p.n - n0 : 65535, nz = p.pg.n_layers - l0 < 65535 ? p.pg.n_layers - l0 : 65535;
      k_page_copy<<<dim3(pieces, ny, nz), kCopyThreads, 0, st>>>(q, row16);
      if (cudaGetLastError() != cudaSuccess) return -1;
    }
  }
  return 0;
}

int launch_page_compact(const PageCompactParams &p, cudaStream_t st) {
  const uint32_t row16 = p.pg.head_dim * elem_size(p.pg.dtype) / 16;
  const uint32_t each = 65535 / p.pg.n_layers;  // sequences of a launch (n_layers <= 65535: checked by the caller)
  for (uint32_t n0 = 0; n0 < p.n; n0 += each) {
    PageCompactParams q = p;
    q.seq += n0;
    q.start += n0;
    const uint32_t m = p.n - n0 < each ? p.n - n0 : each;
    k_page_compact<<<dim3(p.pg.n_kv_heads, 2, m * p.pg.n_layers), kCompactThreads, 0, st>>>(q, row16);
    if (cudaGetLastError() != cudaSuccess) return -1;
  }
  return 0;
}

}  // namespace fa
