// Work split shared by the attention kernels on paged K/V.
//
// An item is (chunk, row tile, kv head): R rows of one kv head, row r of a
// chunk being query token r / rep and query head kvh * rep + r % rep, so the
// rows of an item read the same K and V.  It covers the positions that any of
// its rows sees, in units of U positions.  The units of all items, in chunk,
// row tile, head order, are one line, and each CTA takes an equal stretch of
// it: chunks of any lengths then load the GPU evenly, and a single long cache
// is spread over all of it.  A CTA finishes the items that lie inside its
// stretch; the ends of a stretch leave (max, sum, unnormalised output) in the
// CTA's two slots, and k_attn_join adds the pieces in the order of the
// positions, so results do not depend on timing.
#pragma once
#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {

struct Chunk {
  uint32_t q0, q_len, seq;
  int32_t first;  // position of its first token (kv_len - q_len; negative: tokens before the cache's start)
  uint32_t rows;  // q_len * rep; 0: not of this launch, or refused
};

// Chunk c as the kernels take it; a bad one has no rows and sets a flag.
__device__ __forceinline__ Chunk load_chunk(const AttnChunksParams &p, uint32_t c) {
  Chunk k;
  const uint32_t q0 = p.q_start[c], q1 = p.q_start[c + 1], kv = p.kv_len[c];
  k.seq = p.seq ? p.seq[c] : c;
  k.q0 = q0;
  k.q_len = q1 - q0;
  k.first = (int32_t)kv - (int32_t)k.q_len;
  k.rows = 0;
  if (q1 < q0 || q1 > p.n_tokens || k.q_len > p.max_q || kv > p.pg.max_pages * kPageLen || k.seq >= p.pg.n_seq) {
    if (p.err) atomicOr(p.err, kFlagRange);
    return k;
  }
  const uint32_t rows = k.q_len * p.rep;  // n_tokens * n_heads < 2^31: checked on the host
  if (rows >= p.rows_min && rows <= p.rows_max) k.rows = rows;
  return k;
}

// Positions [lo, hi) that the rows [r0, r1) of a chunk see (hi <= lo: none)
__device__ __forceinline__ void tile_range(const AttnChunksParams &p, const Chunk &k, uint32_t r0, uint32_t r1, uint32_t &lo,
                                           uint32_t &hi) {
  const int32_t last = k.first + (int32_t)((r1 - 1) / p.rep), first = k.first + (int32_t)(r0 / p.rep);
  hi = last < 0 ? 0u : (uint32_t)last + 1;
  lo = p.window && first >= (int32_t)p.window ? (uint32_t)first - p.window + 1 : 0u;
}

template <uint32_t U>
__device__ __forceinline__ uint32_t range_units(uint32_t lo, uint32_t hi) {
  return hi > lo ? (hi - 1) / U - lo / U + 1 : 1;  // at least one: somebody writes the zeros
}
template <uint32_t R, uint32_t U>
__device__ __forceinline__ uint32_t tile_units(const AttnChunksParams &p, const Chunk &k, uint32_t tile) {
  uint32_t lo, hi;
  tile_range(p, k, tile * R, min(k.rows, tile * R + R), lo, hi);
  return range_units<U>(lo, hi);
}
template <uint32_t R, uint32_t U>
__device__ __forceinline__ uint64_t chunk_units(const AttnChunksParams &p, const Chunk &k) {
  uint64_t n = 0;
  for (uint32_t t = 0; t * R < k.rows; ++t) n += tile_units<R, U>(p, k, t);
  return n * p.pg.n_kv_heads;
}

struct Segment {  // a piece of an item
  Chunk chunk;
  uint32_t tile, head;
  uint32_t r0, r1;       // rows of the item
  uint32_t lo, hi;       // positions the item sees
  uint32_t u0, u1, n;    // units [u0, u1) of the item's n
};

// A CTA's walk along its stretch.  Every thread holds the same state.
template <uint32_t R, uint32_t U, uint32_t THREADS>
struct Walk {
  uint32_t left, per;     // units of the stretch that are left, and of a whole one (below 2^32: the line has
                          // at most 2^31 rows / R items of 2^25 / U units for at least 100 CTAs)
  uint32_t c, tile, head;
  uint32_t rem;           // units into the current item
  Chunk chunk;

  // All threads of the CTA; `red` is scratch of THREADS / 32 + 2 words.
  __device__ void start(const AttnChunksParams &p, uint32_t min_units, uint64_t *red) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint64_t sum = 0;
    for (uint32_t i = tid; i < p.n_chunks; i += THREADS) {
      const Chunk k = load_chunk(p, i);
      sum += chunk_units<R, U>(p, k);
    }
    const uint64_t own = sum;  // of chunk tid, where a thread has one at most
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 32; ++w) total += red[w];
    per = (uint32_t)((total + gridDim.x - 1) / gridDim.x);
    if (per < min_units) per = min_units;
    const uint64_t at = (uint64_t)blockIdx.x * per;
    c = tile = head = rem = left = 0;
    if (at >= total) return;  // the same for all threads of the CTA
    left = (uint32_t)min((uint64_t)per, total - at);
    // the chunk that holds `at`: blocks of THREADS chunks, then a scan
    uint64_t before = 0;
    uint64_t *found = red + THREADS / 32;  // [0] chunk, [1] units before it
    for (uint32_t b = 0;; b += THREADS) {
      const uint32_t i = b + tid;
      uint64_t mine = 0;
      if (p.n_chunks <= THREADS) {
        mine = own;
      } else if (i < p.n_chunks) {
        const Chunk k = load_chunk(p, i);
        mine = chunk_units<R, U>(p, k);
      }
      uint64_t inc = mine;  // inclusive scan of the block
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= (uint32_t)o) inc += x;
      }
      __syncthreads();
      if (lane == 31) red[warp] = inc;
      __syncthreads();
      uint64_t prev = before, block = 0;
#pragma unroll
      for (uint32_t w = 0; w < THREADS / 32; ++w) {
        if (w < warp) prev += red[w];
        block += red[w];
      }
      inc += prev;
      if (mine && at >= inc - mine && at < inc) {
        found[0] = i;
        found[1] = inc - mine;
      }
      before += block;
      if (before > at) break;  // at < total: some block holds it
    }
    __syncthreads();
    c = (uint32_t)found[0];
    chunk = load_chunk(p, c);
    // from the units into the chunk to (tile, head, units into the item)
    uint64_t in = at - found[1];
    for (;; ++tile) {
      const uint32_t n = tile_units<R, U>(p, chunk, tile);
      const uint64_t all = (uint64_t)n * p.pg.n_kv_heads;
      if (in < all) {
        head = (uint32_t)(in / n);
        rem = (uint32_t)(in - (uint64_t)head * n);
        return;
      }
      in -= all;
    }
  }
  __device__ bool done() const { return left == 0; }
  // the next piece; moves on behind it
  __device__ Segment next(const AttnChunksParams &p) {
    Segment s;
    s.chunk = chunk;
    s.tile = tile;
    s.head = head;
    s.r0 = tile * R;
    s.r1 = min(chunk.rows, s.r0 + R);
    tile_range(p, chunk, s.r0, s.r1, s.lo, s.hi);
    s.n = range_units<U>(s.lo, s.hi);
    s.u0 = rem;
    const uint32_t take = min(s.n - s.u0, left);
    s.u1 = s.u0 + take;
    left -= take;
    rem = 0;
    if (s.u1 == s.n && left) {  // the next item
      if (++head == p.pg.n_kv_heads) {
        head = 0;
        if (++tile * R >= chunk.rows) {
          tile = 0;
          do chunk = load_chunk(p, ++c);
          while (!chunk.rows);  // units are left, so a chunk with rows follows
        }
      }
    }
    return s;
  }
  __device__ static bool whole(const Segment &s) { return s.u0 == 0 && s.u1 == s.n; }
  // What k_attn_join has to know of an item that this CTA begins and does not
  // end: its rows, its head, and the CTAs on it.
  __device__ uint4 describe(const Segment &s) const {
    return make_uint4(s.chunk.q0, s.r0, s.head | (s.r1 - s.r0) << 16, 1 + (s.n - s.u1 - 1) / per + 1);
  }
  // The slot of a piece that is not a whole item: slot 1 of the CTA that begins
  // the item, slot 0 of the others; R x hd outputs, then R x (max, sum)
  __device__ static float *slot(const AttnChunksParams &p, const Segment &s) {
    return p.part + ((uint64_t)blockIdx.x * 2 + (s.u0 ? 0 : 1)) * R * (p.pg.head_dim + 2);
  }
};
// Split items of one launch, as k_attn_join takes them.
struct JoinSet {
  const float *part;
  const uint4 *desc;
  uint32_t R, ctas;
  uint32_t parts;  // CTAs of the join to an item
};
// The kernels; each returns its grid, or 0 where the launch failed.
bool attn_mma_takes(const AttnChunksParams &p);
uint32_t launch_attn_any(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *R);
uint32_t launch_attn_mma(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *R);
uint32_t launch_attn_tc(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st);

// Most CTAs and rows of an item of the launch for few rows, and of the launch
// for many: what the workspace holds two slots of each for.
constexpr uint32_t kAttnMaxCtas = 480, kAttnMaxRows = 64;
constexpr uint32_t kTcMaxCtas = 160, kTcRows = 256;
// Where element d (a multiple of 4, and the three behind it) of row r is in a
// slot of the launch for many rows, whose threads have a row each; after the
// kTcRows x hd outputs come the pairs (max, sum).
__host__ __device__ constexpr uint32_t tc_part(uint32_t r, uint32_t d, uint32_t hd) {
  return ((r / 32) * (hd / 4) + d / 4) * 128 + (r % 32) * 4;
}

// element offset of (page, k | v, head, position in page) in a layer
__device__ __forceinline__ uint64_t page_row(const fa_pages &pg, uint32_t page, uint32_t is_v, uint32_t h, uint32_t slot) {
  return ((((uint64_t)page * 2 + is_v) * pg.n_kv_heads + h) * kPageLen + slot) * pg.head_dim;
}

}  // namespace fa
