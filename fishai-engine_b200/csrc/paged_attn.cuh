// Work split shared by the attention kernels on paged K/V.
//
// An item is (chunk, row tile, kv head): R rows of one kv head, row r of a
// chunk being query token r / rep and query head kvh * rep + r % rep, so the
// rows of an item read the same K and V.  It covers the positions that any of
// its rows sees, in units of U positions.  The items' costs, in chunk, row tile,
// head order, are one line, and each CTA takes an equal stretch of it: chunks of
// any lengths then load the GPU evenly, and a single long cache is spread over all
// of it.  A CTA finishes the items that lie inside its
// stretch; the ends of a stretch leave (max, sum, unnormalised output) in the
// CTA's two slots, and k_attn_join adds the pieces in the order of the
// positions, so results do not depend on timing.
#pragma once
#include <atomic>

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
// Cost of a row tile on the line: its units, and OVER for what an item costs
// apart from them (Q, filling the pipeline, the output), so that many short
// items do not make a CTA late.
template <uint32_t R, uint32_t U, uint32_t OVER>
__device__ __forceinline__ uint32_t tile_cost(const AttnChunksParams &p, const Chunk &k, uint32_t tile) {
  uint32_t lo, hi;
  tile_range(p, k, tile * R, min(k.rows, tile * R + R), lo, hi);
  return range_units<U>(lo, hi) + OVER;
}
// Cost of the lane's chunk, its row tiles times the heads; long chunks by the
// whole warp (a thread to itself took 6 us for the 16 tiles of 1024 tokens)
template <uint32_t R, uint32_t U, uint32_t OVER>
__device__ __forceinline__ uint64_t chunk_cost(const AttnChunksParams &p, const Chunk &k) {
  const uint32_t lane = threadIdx.x & 31;
  uint64_t mine = 0;
  const bool small = k.rows <= 2 * R;
  if (small)
    for (uint32_t t = 0; t * R < k.rows; ++t) mine += tile_cost<R, U, OVER>(p, k, t);
  for (uint32_t big = __ballot_sync(0xFFFFFFFFu, !small); big; big &= big - 1) {
    const uint32_t who = __ffs(big) - 1;
    Chunk c;
    c.rows = __shfl_sync(0xFFFFFFFFu, k.rows, who);
    c.first = __shfl_sync(0xFFFFFFFFu, k.first, who);
    uint64_t sum = 0;
    for (uint32_t t = lane; (uint64_t)t * R < c.rows; t += 32) sum += tile_cost<R, U, OVER>(p, c, t);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == who) mine = sum;
  }
  return mine * p.pg.n_kv_heads;
}

struct Segment {  // a piece of an item
  Chunk chunk;
  uint32_t tile, head;
  uint32_t r0, r1;       // rows of the item
  uint32_t lo, hi;       // positions the item sees
  uint32_t u0, u1, n;    // units [u0, u1) of the item's n
};

// A CTA's walk along its stretch.  Every thread holds the same state.
template <uint32_t R, uint32_t U, uint32_t OVER, uint32_t THREADS>
struct Walk {
  uint32_t left, per;     // cost of the stretch that is left, and of a whole one (start() refuses a line whose
                          // stretches need more bits)
  uint32_t c, tile, head;
  uint32_t rem;           // cost into the current item; its first OVER stand for no work
  Chunk chunk;

  // All threads of the CTA; `red` is scratch of THREADS / 32 + 2 words.
  __device__ void start(const AttnChunksParams &p, uint32_t min_cost, uint64_t *red) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto cost = [&](uint32_t i) -> uint64_t {  // of chunk i, whole warps
      Chunk k;
      k.rows = 0;
      if (i < p.n_chunks) k = load_chunk(p, i);
      return chunk_cost<R, U, OVER>(p, k);
    };
    uint64_t sum = 0;
    for (uint32_t b = 0; b < p.n_chunks; b += THREADS) sum += cost(b + tid);
    const uint64_t own = sum;  // of chunk tid, where a thread has one at most
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 32; ++w) total += red[w];
    c = tile = head = rem = left = 0;
    // 2^32 units a CTA, an hour of work and more: nothing is done (the same for all CTAs)
    const uint64_t share = (total + gridDim.x - 1) / gridDim.x;
    per = share > min_cost ? (uint32_t)share : min_cost;
    if (share > 0xFFFFFFFFull) {
      if (p.err && blockIdx.x == 0 && tid == 0) atomicOr(p.err, kFlagRange);
      return;
    }
    const uint64_t at = (uint64_t)blockIdx.x * per;
    if (at >= total) return;  // the same for all threads of the CTA
    left = (uint32_t)min((uint64_t)per, total - at);
    // the chunk that holds `at`: blocks of THREADS chunks, then a scan
    uint64_t before = 0;
    uint64_t *found = red + THREADS / 32;  // [0] chunk, [1] cost before it
    for (uint32_t b = 0;; b += THREADS) {
      const uint32_t i = b + tid;
      const uint64_t mine = p.n_chunks <= THREADS ? own : cost(i);
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
    // from the cost into the chunk to (tile, head, cost into the item), 32 tiles
    // at a time
    uint64_t in = at - found[1];
    for (uint32_t t0 = 0;; t0 += 32) {
      const uint32_t t = t0 + lane, n = (uint64_t)t * R < chunk.rows ? tile_cost<R, U, OVER>(p, chunk, t) : 0;
      uint64_t inc = (uint64_t)n * p.pg.n_kv_heads;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= (uint32_t)o) inc += x;
      }
      const uint32_t behind = __ballot_sync(0xFFFFFFFFu, inc > in);
      if (behind) {
        const uint32_t l = __ffs(behind) - 1;
        const uint32_t one = __shfl_sync(0xFFFFFFFFu, n, l);
        in -= __shfl_sync(0xFFFFFFFFu, inc, l) - (uint64_t)one * p.pg.n_kv_heads;
        tile = t0 + l;
        head = (uint32_t)(in / one);
        rem = (uint32_t)(in - (uint64_t)head * one);
        return;
      }
      in -= __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
  }
  __device__ bool done() const { return left == 0; }
  // the next piece with work in it; false: there is none left
  __device__ bool next(const AttnChunksParams &p, Segment &s) {
    while (left) {
      s.chunk = chunk;
      s.tile = tile;
      s.head = head;
      s.r0 = tile * R;
      s.r1 = min(chunk.rows, s.r0 + R);
      tile_range(p, chunk, s.r0, s.r1, s.lo, s.hi);
      s.n = range_units<U>(s.lo, s.hi);
      const uint32_t take = min(s.n + OVER - rem, left), end = rem + take;
      s.u0 = rem > OVER ? rem - OVER : 0;
      s.u1 = end > OVER ? end - OVER : 0;
      left -= take;
      rem = 0;
      if (end == s.n + OVER && left) {  // the next item
        if (++head == p.pg.n_kv_heads) {
          head = 0;
          if (++tile * R >= chunk.rows) {
            tile = 0;
            do chunk = load_chunk(p, ++c);
            while (!chunk.rows);  // some cost is left, so a chunk with rows follows
          }
        }
      }
      if (s.u1 > s.u0) return true;
    }
    return false;
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
// ---- an item on a cluster of CTAs, for few items ----
// The CTAs take the item's units in turn and add their pieces from one another's
// shared memory: no second launch, which is half of a short call's time.
constexpr uint32_t kOneCtas = 8;  // of a cluster (the portable most; of 16, the GPU holds 7 at once, for 8 kv heads)

// Most positions that a token of the call can see, as far as the host knows.
inline uint64_t one_span(const AttnChunksParams &p) {
  const uint64_t cap = (uint64_t)p.pg.max_pages * kPageLen, seen = (uint64_t)p.window + p.max_q;
  return p.window && seen < cap ? seen : cap;
}
inline uint64_t one_items(const AttnChunksParams &p) { return (uint64_t)p.n_chunks * p.pg.n_kv_heads; }
// Cluster blockIdx.x / kOneCtas takes (chunk, head); false: the chunk has no
// rows (the same for the whole cluster).
__device__ __forceinline__ bool one_item(const AttnChunksParams &p, Segment &s) {
  const uint32_t item = blockIdx.x / kOneCtas;
  s.chunk = load_chunk(p, item / p.pg.n_kv_heads);
  if (!s.chunk.rows) return false;
  s.tile = 0;
  s.head = item % p.pg.n_kv_heads;
  s.r0 = 0;
  s.r1 = s.chunk.rows;
  tile_range(p, s.chunk, 0, s.r1, s.lo, s.hi);
  return true;
}
// The cluster's rows from the CTAs' pieces, each (max, sum) [rows] and
// unnormalised outputs [rows][hd] in shared memory (16-byte aligned), as in
// k_attn_join, in the order of the CTAs: the threads of all CTAs share the
// elements, with the loads of all pieces in flight.  put(row, d, f32 x 4).
template <uint32_t THREADS, uint32_t C = kOneCtas, typename Put>
__device__ __forceinline__ void one_join(const Segment &s, uint32_t hd, const float *o, uint32_t ld, const float *ml, Put put) {
  cluster_sync();
  const uint32_t n4 = (s.r1 - s.r0) * (hd / 4), per = (n4 + C - 1) / C, i0 = cluster_ctarank() * per;
  for (uint32_t i = i0 + threadIdx.x; i < min(n4, i0 + per); i += THREADS) {
    const uint32_t r = i / (hd / 4), d = (i - r * (hd / 4)) * 4;
    float m[C], l[C];
    float4 x[C];
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) {
      asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(m[k]), "=f"(l[k]) : "r"(dsmem_addr(ml + 2 * r, k)) : "memory");
      asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(x[k].x), "=f"(x[k].y), "=f"(x[k].z), "=f"(x[k].w)
                   : "r"(dsmem_addr(o + r * ld + d, k))
                   : "memory");
    }
    float M = m[0], L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (uint32_t k = 1; k < C; ++k) M = fmaxf(M, m[k]);
    const float Ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) {
      const float e = exp2f(m[k] - Ms);
      L = fmaf(l[k], e, L);
      acc.x = fmaf(x[k].x, e, acc.x);
      acc.y = fmaf(x[k].y, e, acc.y);
      acc.z = fmaf(x[k].z, e, acc.z);
      acc.w = fmaf(x[k].w, e, acc.w);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    put(r, d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  }
  cluster_sync();  // the pieces have been read
}
// Launches a cluster for each of `items`, where the GPU holds that many at once; 1: it does not, -1: an error.
template <auto kern, uint32_t C = kOneCtas>
int launch_one(const AttnChunksParams &p, uint64_t items, uint32_t threads, uint32_t smem, cudaStream_t st) {
  static std::atomic<int> known[64];  // clusters at once, by device (0: not asked yet)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return -1;
  int device = 0, at_once = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return -1;
  const bool keep = device >= 0 && device < 64;
  if (keep) at_once = known[device].load(std::memory_order_relaxed);
  if (!at_once) {
    if (cudaOccupancyMaxActiveClusters(&at_once, kern, &cfg) != cudaSuccess) return -1;
    if (keep && at_once > 0) known[device].store(at_once, std::memory_order_relaxed);
  }
  if (items > (uint64_t)(at_once > 0 ? at_once : 0)) return 1;
  cfg.gridDim = dim3((uint32_t)items * C);
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? 0 : -1;
}

// Split items of one launch, as k_attn_join takes them.
struct JoinSet {
  const float *part;
  const uint4 *desc;
  uint32_t R, ctas;
  uint32_t parts;  // CTAs of the join to an item
};
// One launch for few items, each a cluster; 1: the call is not of that kind.
int launch_one_any(const AttnChunksParams &p, cudaStream_t st);
int launch_one_few(const AttnChunksParams &p, cudaStream_t st);
int launch_one_mma(const AttnChunksParams &p, cudaStream_t st);
int launch_short_mma(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st);
// The kernels; each returns its grid, or 0 where the launch failed.
bool attn_mma_takes(const AttnChunksParams &p);
uint32_t launch_attn_few(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *R);  // no chunk above 16 rows
uint32_t launch_attn_any(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *R);
uint32_t launch_attn_mma(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st);  // items of kMmaRows
// overlap: the launch before is launch_attn_mma's, with which this one may run at the same time
uint32_t launch_attn_tc(const AttnChunksParams &p, uint32_t n_sm, bool overlap, cudaStream_t st, uint32_t *R);

// Most CTAs and rows of an item of the launch for few rows (or of the f32 one),
// and of the launch for many: what the workspace holds two slots of each for.
constexpr uint32_t kAttnMaxCtas = 480, kAttnMaxRows = 32, kMmaRows = 16;
constexpr uint32_t kTcMaxCtas = 160, kTcRows = 256;  // or twice as many CTAs of 128 rows
// Where element d (a multiple of 4, and the three behind it) of row r is in a
// slot of the launch for many rows, whose threads have a row each; after the
// R x hd outputs come the pairs (max, sum).
__host__ __device__ constexpr uint32_t tc_part(uint32_t r, uint32_t d, uint32_t hd) {
  return ((r / 32) * (hd / 4) + d / 4) * 128 + (r % 32) * 4;
}

// element offset of (page, k | v, head, position in page) in a layer
__device__ __forceinline__ uint64_t page_row(const fa_pages &pg, uint32_t page, uint32_t is_v, uint32_t h, uint32_t slot) {
  return ((((uint64_t)page * 2 + is_v) * pg.n_kv_heads + h) * kPageLen + slot) * pg.head_dim;
}

}  // namespace fa
