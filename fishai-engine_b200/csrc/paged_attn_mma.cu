// Attention of chunks over paged f16 / bf16 K/V with up to 16 rows per kv head:
// single tokens and a few at a time, head sizes 64 and 128.  Same mathematics as
// paged_attn_any.cu, products on mma.sync m16n8k16 with f32 accumulators.  The
// weights p = 2^(s - m) <= 1 are rounded to the cache's type for the product
// with V (the type V itself was rounded to); their sum is taken before that
// rounding, in f32.  In f16 they are 2^15 times that, and so are their sums: f16
// has full precision down to 2^-14 and nothing below 2^-25, and beside one
// large weight the small ones of a long cache may be most of the output.
//
// HBM bounds it: every K and V row is used for at most 16 rows of Q, far below
// the 250 operations a byte where tensor cores would bind, so all that counts
// is copies in flight.  Sub-tiles of 32 positions (two pages) go to shared
// memory by cp.async in 16-byte pieces, XOR-swizzled by row so that ldmatrix
// reads eight rows from distinct banks; rows nobody sees are filled with
// zeros, so stale or NaN slots do not reach a product.  Each warp runs through
// its own sub-tiles and keeps its own (max, sum, output); the four of a CTA are
// merged at the end of a piece.  The next K is fetched as soon as the scores are
// formed, the next V after its product, so both buffers are nearly always in
// flight; three CTAs an SM.  64 sequences of 4096 positions, 32/8 heads x 128:
// 178 us, 6.0 TB/s; of 37 to 4096 positions: 95 us, 5.6 TB/s.  (One CTA an SM
// whose ring of copies a TMA warp keeps filled across items: 225 and 138 us.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_attn.cuh"

namespace fa {
namespace {

constexpr uint32_t kSub = 32;       // positions of a sub-tile
constexpr uint32_t kThreads = 128;  // 4 warps

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint32_t bytes) {  // 16 of them, or 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp; below 2^-126: 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (__is_same(T, __half)) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}
template <typename T>
constexpr float kLift = __is_same(T, __half) ? 15.0f : 0.0f;  // weights are 2^(s - m + kLift)
template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (__is_same(T, __half)) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// byte offset of 16-byte piece c of row r
template <uint32_t HD>
__device__ __forceinline__ uint32_t sw(uint32_t r, uint32_t c) {
  return r * (HD * 2) + ((c ^ (r & 7)) << 4);
}

// where the two pages of a sub-tile begin
struct Tile {
  uint32_t t[2];
};
// sub-tile h of unit u
template <uint32_t U, typename PR>
__device__ __forceinline__ Tile tile_at(const PR &p, uint32_t lo, uint32_t u, uint32_t h = 0) {
  const uint32_t t = unit_page<U>(p, lo, u, 2 * h);
  return {{t, PR::packed ? unit_page<U>(p, lo, u, 2 * h + 1) : t + kPageLen}};
}
// that of unit u + step, where unit u is a sub-tile at `at`
template <typename PR>
__device__ __forceinline__ Tile tile_after(const PR &p, uint32_t lo, uint32_t u, const Tile &at, uint32_t step) {
  if constexpr (PR::packed) return tile_at<kSub>(p, lo, u + step);
  const uint32_t t = unit_after<kSub>(p, lo, u, at.t[0], step);
  return {{t, t + kPageLen}};
}

// The rows of one warp: 16 rows of the item, this thread's rows g and g + 8
// (MMA fragment layout), with the running softmax and output.
template <typename T, uint32_t HD>
struct Rows {
  uint32_t qa[HD / 16][4];
  float o[HD / 8][4], m[2], l[2];
  int32_t pos[2];           // positions of the tokens; -1: no row (sees nothing)
  int32_t pos_min, pos_max; // over the warp's real rows

  __device__ void load(const AttnChunksParams &p, const Segment &s, uint32_t first_row) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const T *q[2];
    bool ok[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t row = first_row + g + 8 * i;
      ok[i] = row < s.r1;
      const uint32_t tok = ok[i] ? row / p.rep : 0, h = ok[i] ? row - tok * p.rep : 0;
      pos[i] = ok[i] ? s.chunk.first + (int32_t)tok : -1;
      q[i] = reinterpret_cast<const T *>(p.q) + (uint64_t)(s.chunk.q0 + tok) * p.qs + (s.head * p.rep + h) * HD;
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
    const uint32_t last = min(s.r1, first_row + 16) - 1;  // the caller's rows are not empty
    pos_min = s.chunk.first + (int32_t)(first_row / p.rep);
    pos_max = s.chunk.first + (int32_t)(last / p.rep);
#pragma unroll
    for (uint32_t kt = 0; kt < HD / 16; ++kt)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {  // rows g, g+8; columns 2c, 2c+8
        const T *x = q[e & 1] + 16 * kt + 2 * c + 8 * (e >> 1);
        uint32_t w = 0;
        if (ok[e & 1]) {
          if (p.aligned) w = *reinterpret_cast<const uint32_t *>(x);
          else w = (uint32_t)*reinterpret_cast<const uint16_t *>(x) | (uint32_t)*reinterpret_cast<const uint16_t *>(x + 1) << 16;
        }
        qa[kt][e] = w;
      }
#pragma unroll
    for (uint32_t j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  }

  // scores of 32 positions from t0 on
  __device__ void scores(uint32_t ktile, float (&s)[kSub / 8][4]) const {
    const uint32_t lane = threadIdx.x & 31, mi = lane >> 3;
#pragma unroll
    for (uint32_t j = 0; j < kSub / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
    for (uint32_t kt = 0; kt < HD / 16; ++kt)
#pragma unroll
      for (uint32_t j = 0; j < kSub / 8; j += 2) {
        uint32_t b0, b1, b2, b3;
        ldsm4(ktile + sw<HD>(8 * j + 8 * (mi >> 1) + (lane & 7), 2 * kt + (mi & 1)), b0, b1, b2, b3);
        mma16816<T>(s[j], qa[kt], b0, b1);
        mma16816<T>(s[j + 1], qa[kt], b2, b3);
      }
  }

  // s -> weights; the running maximum, sum and output follow
  template <typename PR>
  __device__ void softmax(const PR &p, const Tile &at, float (&s)[kSub / 8][4]) {
    const uint32_t c = threadIdx.x & 3;
    auto in = [&](uint32_t t) { return pos_max - (int32_t)t < (int32_t)p.window || t + kPageLen <= p.sinks; };
    const bool all = (int32_t)(at.t[1] + kPageLen - 1) <= pos_min && (!p.window || (in(at.t[0]) && (!PR::packed || in(at.t[1]))));
    float mx[2] = {-INFINITY, -INFINITY};
    if (!all) {
#pragma unroll
      for (uint32_t j = 0; j < kSub / 8; ++j)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          if (!token_sees(p, pos[e >> 1], (int32_t)(at.t[j / 2] + 8 * (j % 2) + 2 * c + (e & 1)))) s[j][e] = -INFINITY;
    }
#pragma unroll
    for (uint32_t j = 0; j < kSub / 8; ++j)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xFFFFFFFFu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xFFFFFFFFu, mx[i], 2));
      const float mn = fmaxf(m[i], mx[i] * p.scale_log2), ms = mn == -INFINITY ? 0.0f : mn;
      const float f = ex2(m[i] - ms);
      m[i] = mn;
      float sum = 0.0f;
#pragma unroll
      for (uint32_t j = 0; j < kSub / 8; ++j)
#pragma unroll
        for (uint32_t e = 2 * i; e < 2 * i + 2; ++e) {
          s[j][e] = ex2(fmaf(s[j][e], p.scale_log2, kLift<T> - ms));
          sum += s[j][e];
        }
      l[i] = fmaf(l[i], f, sum);  // of this thread's columns: summed over the four at the end
#pragma unroll
      for (uint32_t j = 0; j < HD / 8; ++j) {
        o[j][2 * i] *= f;
        o[j][2 * i + 1] *= f;
      }
    }
  }

  __device__ void add_values(uint32_t vtile, const float (&s)[kSub / 8][4]) {
    const uint32_t lane = threadIdx.x & 31, mi = lane >> 3;
#pragma unroll
    for (uint32_t kt = 0; kt < kSub / 16; ++kt) {
      const uint32_t a[4] = {pack2<T>(s[2 * kt][0], s[2 * kt][1]), pack2<T>(s[2 * kt][2], s[2 * kt][3]),
                             pack2<T>(s[2 * kt + 1][0], s[2 * kt + 1][1]), pack2<T>(s[2 * kt + 1][2], s[2 * kt + 1][3])};
#pragma unroll
      for (uint32_t j = 0; j < HD / 8; j += 2) {
        uint32_t b0, b1, b2, b3;
        ldsm4_t(vtile + sw<HD>(16 * kt + 8 * (mi & 1) + (lane & 7), j + (mi >> 1)), b0, b1, b2, b3);
        mma16816<T>(o[j], a, b0, b1);
        mma16816<T>(o[j + 1], a, b2, b3);
      }
    }
  }
  __device__ void finish() {
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
      l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
    }
  }
};

// Where a warp's copies of a sub-tile come from (looked up one sub-tile ahead).
struct PagePair {
  uint32_t page[2];
};
template <typename PR>
__device__ __forceinline__ PagePair look_up(const PR &p, const uint32_t *pt, const Tile &at, uint32_t lo, uint32_t hi) {
  PagePair r;
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t t = at.t[i];
    r.page[i] = item_reads(p, lo, hi, t) ? __ldg(pt + t / kPageLen) : 0u;  // only pages that are read are looked up
  }
  return r;
}
// K (is_v 0) or V rows of a sub-tile's positions to shared memory; THREADS threads,
// thread i of them.  Positions that the item does not see and bad pages become zeros.
template <typename T, uint32_t HD, typename PR>
__device__ __forceinline__ void stage(const PR &p, const T *base, const PagePair &pg, uint32_t head, uint32_t is_v,
                                      const Tile &at, uint32_t lo, uint32_t hi, uint32_t tile, uint32_t i, uint32_t threads) {
  constexpr uint32_t CH = HD / 8;  // pieces of a row
  const uint32_t c = i % CH, r0 = i / CH, step = threads / CH;
  // A bit for each row of a page that is seen: a shift and an "and" a row, and one path for all sub-tiles.  (Bounds
  // compared row by row were a third of a sub-tile's instructions where there are first positions beside a window.  With
  // a path of its own for sub-tiles that are seen whole one token over 4096 positions and 4 first ones took 10.4 us, 8.7
  // so, and calls of one short sub-tile, which fetch the code of both, 0.2 to 0.5 us more than the 4 to 6 they take.)
#pragma unroll
  for (uint32_t half = 0; half < 2; ++half) {
    const bool good = pg.page[half] < p.pg.n_pages;
    const T *src = base + page_row(p.pg, good ? pg.page[half] : 0, is_v, head, 0) + c * 8;
    const uint32_t t = at.t[half];
    auto below = [&](uint32_t x) { return (1u << (x > t ? min(x - t, kPageLen) : 0u)) - 1; };
    uint32_t m = ~below(lo);
    if (PR::packed) m |= below(p.sinks);
    m = good ? (m & below(hi)) >> r0 << 4 : 0;
#pragma unroll
    for (uint32_t r = 0; r < 16; r += step) cp16(tile + sw<HD>(16 * half + r + r0, c), src + (r + r0) * HD, m >> r & 16);
  }
}

template <typename T>
__device__ __forceinline__ T *out_row(const AttnChunksParams &p, const Segment &s, uint32_t row, uint32_t hd) {
  const uint32_t tok = row / p.rep;
  return reinterpret_cast<T *>(p.out) + (uint64_t)(s.chunk.q0 + tok) * p.os + (s.head * p.rep + row - tok * p.rep) * hd;
}

__device__ __forceinline__ void flag_bad_pages(const AttnChunksParams &p, const PagePair &pg) {
  if ((pg.page[0] >= p.pg.n_pages || pg.page[1] >= p.pg.n_pages) && p.err) atomicOr(p.err, kFlagPage);
}

// The warps' rows to shared memory, [warp][16][HD + 4], then (max, sum); over
// the tiles, which all warps have read
template <uint32_t HD, uint32_t WARPS>
struct Merge {
  static constexpr uint32_t LD = HD + 4, kBytes = WARPS * 16 * LD * 4 + WARPS * 16 * 8;
  float *o, *ml;
  template <typename T>
  __device__ Merge(uint8_t *at, const Rows<T, HD> &rows) : o(reinterpret_cast<float *>(at)), ml(o + WARPS * 16 * LD) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < HD / 8; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i)
        *reinterpret_cast<float2 *>(o + (warp * 16 + g + 8 * i) * LD + 8 * j + 2 * c) = make_float2(rows.o[j][2 * i], rows.o[j][2 * i + 1]);
    if (c == 0)
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        ml[(warp * 16 + g + 8 * i) * 2] = rows.m[i];
        ml[(warp * 16 + g + 8 * i) * 2 + 1] = rows.l[i];
      }
    __syncthreads();
  }
  // elements d .. d + 3 of row r, with its (max, sum), of all warps in order
  __device__ float4 sum(uint32_t r, uint32_t d, float &M, float &L) const {
    M = -INFINITY;
    L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (uint32_t v = 0; v < WARPS; ++v) M = fmaxf(M, ml[(v * 16 + r) * 2]);
    const float Ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (uint32_t v = 0; v < WARPS; ++v) {
      const float e = ex2(ml[(v * 16 + r) * 2] - Ms);
      const float4 x = *reinterpret_cast<const float4 *>(o + (v * 16 + r) * LD + d);
      L = fmaf(ml[(v * 16 + r) * 2 + 1], e, L);
      acc.x = fmaf(x.x, e, acc.x);
      acc.y = fmaf(x.y, e, acc.y);
      acc.z = fmaf(x.z, e, acc.z);
      acc.w = fmaf(x.w, e, acc.w);
    }
    return acc;
  }
};
template <typename T>
__device__ __forceinline__ void put4(const AttnChunksParams &p, T *o, float4 x) {
  if (p.aligned) {
    *reinterpret_cast<uint2 *>(o) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
  } else {
    o[0] = round_to<T>(x.x);
    o[1] = round_to<T>(x.y);
    o[2] = round_to<T>(x.z);
    o[3] = round_to<T>(x.w);
  }
}

// A warp's sub-tiles u, u + step, .. < n of an item (from its first one on), its
// K and V tiles the only ones it uses.  q: called once the first copies are on
// their way.
template <typename T, uint32_t HD, typename Q, typename PR>
__device__ __forceinline__ void walk_tiles(const PR &p, const T *base, const Segment &s, uint32_t u, uint32_t n, uint32_t step,
                                           uint32_t ktile, uint32_t vtile, Rows<T, HD> &rows, Q q) {
  const uint32_t *pt = p.pg.page_table + (uint64_t)s.chunk.seq * p.pg.max_pages;
  const uint32_t lane = threadIdx.x & 31;
  Tile at = tile_at<kSub>(p, s.lo, u);
  PagePair pg = look_up(p, pt, at, s.lo, s.hi);
  if (u < n) {
    flag_bad_pages(p, pg);
    stage<T, HD>(p, base, pg, s.head, 0, at, s.lo, s.hi, ktile, lane, 32);
    cp_commit();
    stage<T, HD>(p, base, pg, s.head, 1, at, s.lo, s.hi, vtile, lane, 32);
    cp_commit();
  }
  PagePair ahead = look_up(p, pt, tile_after(p, s.lo, u, at, step), s.lo, s.hi);
  q();
  for (; u < n; u += step) {
    const bool more = u + step < n;
    const Tile next = tile_after(p, s.lo, u, at, step);
    float sc[kSub / 8][4];
    cp_wait<1>();
    __syncwarp();
    rows.scores(ktile, sc);
    __syncwarp();
    pg = ahead;
    if (more) {
      flag_bad_pages(p, pg);
      stage<T, HD>(p, base, pg, s.head, 0, next, s.lo, s.hi, ktile, lane, 32);
    }
    cp_commit();
    ahead = look_up(p, pt, tile_after(p, s.lo, u + step, next, step), s.lo, s.hi);
    rows.softmax(p, at, sc);
    cp_wait<1>();
    __syncwarp();
    rows.add_values(vtile, sc);
    __syncwarp();
    if (more) stage<T, HD>(p, base, pg, s.head, 1, next, s.lo, s.hi, vtile, lane, 32);
    cp_commit();
    at = next;
  }
  cp_wait<0>();
  rows.finish();
}

// ------------------------------------------------------------ up to 16 rows
template <typename T, uint32_t HD, typename PR>
__global__ void __launch_bounds__(kThreads, 3) k_attn_rows16(const PR p) {
  extern __shared__ __align__(128) uint8_t dsm[];
  __shared__ uint64_t red[kThreads / 32 + 2];
  constexpr uint32_t kTileBytes = kSub * HD * 2;
  using W = Walk<kMmaRows, kSub, 6, kThreads>;
  const uint32_t tid = threadIdx.x, warp = tid >> 5;
  const uint32_t ktile = smem_u32(dsm) + warp * 2 * kTileBytes, vtile = ktile + kTileBytes;
  const T *base = reinterpret_cast<const T *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
  pdl_launch_dependents();
  W w;
  w.start(p, 4, red);
  if (tid == 0) p.desc[blockIdx.x].w = 0;
  for (Segment s; w.next(p, s);) {
    Rows<T, HD> rows;
    rows.load(p, s, s.r0);
    walk_tiles<T, HD>(p, base, s, s.hi > s.lo ? s.u0 + warp : s.u1, s.u1, kThreads / 32, ktile, vtile, rows, [] {});
    const Merge<HD, kThreads / 32> pieces(dsm, rows);
    const bool whole = W::whole(s);
    float *slot = W::slot(p, s);
    const uint32_t n_rows = s.r1 - s.r0;
    for (uint32_t i = tid; i < n_rows * (HD / 4); i += kThreads) {
      const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
      float M, L;
      const float4 acc = pieces.sum(r, d, M, L);
      if (whole) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        put4(p, out_row<T>(p, s, s.r0 + r, HD) + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      } else {
        *reinterpret_cast<float4 *>(slot + r * HD + d) = acc;
        if (d == 0) *reinterpret_cast<float2 *>(slot + 16 * HD + 2 * r) = make_float2(M, L);
      }
    }
    if (!whole && s.u0 == 0 && tid == 0) p.desc[blockIdx.x] = w.describe(s);
    __syncthreads();  // the next piece copies over the scratch
  }
}

template <typename T, uint32_t HD>
uint32_t launch_hd(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st) {
  // two tiles of 32 positions a warp, or the merge's 4 x 16 rows
  constexpr uint32_t kTiles = 4 * 2 * kSub * HD * 2, kMerge = Merge<HD, 4>::kBytes, kBytes = kTiles > kMerge ? kTiles : kMerge;
  const uint32_t grid = 3 * n_sm < kAttnMaxCtas ? 3 * n_sm : kAttnMaxCtas;
  return with_sinks<PackedParams>(p, [&](auto a) -> uint32_t {
    using PR = decltype(a);
    if (cudaFuncSetAttribute(k_attn_rows16<T, HD, PR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBytes) != cudaSuccess) return 0;
    k_attn_rows16<T, HD><<<grid, kThreads, kBytes, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? grid : 0;
  });
}

// ------------------------------------- few items of up to 16 rows: a cluster each
template <uint32_t HD, uint32_t WARPS>
struct OneCfg {
  static constexpr uint32_t kTiles = WARPS * 2 * kSub * HD * 2;  // a K and a V tile a warp
  static constexpr uint32_t kPiece = Merge<HD, WARPS>::kBytes;   // over them the warps' pieces, behind those the CTA's
  static constexpr uint32_t kEnd = kPiece + 16 * HD * 4 + 16 * 8, kBytes = kTiles > kEnd ? kTiles : kEnd;
};
template <typename T, uint32_t HD, uint32_t WARPS, typename PR>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 8 ? 1 : 2) k_attn_one16(const PR p) {
  extern __shared__ __align__(128) uint8_t dsm[];
  constexpr uint32_t kTileBytes = kSub * HD * 2;
  const uint32_t tid = threadIdx.x, warp = tid >> 5;
  const uint32_t ktile = smem_u32(dsm) + warp * 2 * kTileBytes, vtile = ktile + kTileBytes;
  const T *base = reinterpret_cast<const T *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
  Segment s;
  if (!one_item(p, s)) return;
  const uint32_t n = s.hi > s.lo ? range_units<kSub>(p, s.lo, s.hi) : 0;
  Rows<T, HD> rows;
  walk_tiles<T, HD>(p, base, s, cluster_ctarank() * WARPS + warp, n, kOneCtas * WARPS, ktile, vtile, rows, [&] { rows.load(p, s, 0); });
  const Merge<HD, WARPS> pieces(dsm, rows);
  float *o = reinterpret_cast<float *>(dsm + OneCfg<HD, WARPS>::kPiece), *ml = o + 16 * HD;
  for (uint32_t i = tid; i < s.r1 * (HD / 4); i += 32 * WARPS) {
    const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
    float M, L;
    *reinterpret_cast<float4 *>(o + r * HD + d) = pieces.sum(r, d, M, L);
    if (d == 0) *reinterpret_cast<float2 *>(ml + 2 * r) = make_float2(M, L);
  }
  one_join<32 * WARPS>(s, HD, o, HD, ml, [&](uint32_t r, uint32_t d, float4 x) { put4(p, out_row<T>(p, s, r, HD) + d, x); });
}
// Eight warps, one CTA an SM, or six and two CTAs: the former keep more copies in
// flight (8 kv heads over 8192 positions 11.9 us against 15.0), the latter take
// twice the items and are ahead where their first sub-tiles are all there is (1024
// positions: 5.8 us against 6.4).
template <typename T, uint32_t HD>
int launch_one_hd(const AttnChunksParams &p, uint64_t span, cudaStream_t st) {
  return with_sinks<PackedParams>(p, [&](auto a) {
    using PR = decltype(a);
    if (span > kOneCtas * 6 * kSub) {
      const int rc = launch_one<k_attn_one16<T, HD, 8, PR>>(a, one_items(p), 256, OneCfg<HD, 8>::kBytes, st);
      if (rc <= 0) return rc;
    }
    return launch_one<k_attn_one16<T, HD, 6, PR>>(a, one_items(p), 192, OneCfg<HD, 6>::kBytes, st);
  });
}

// --------------------------- short calls of more rows: a cluster to 64 rows each
// An item is 64 rows of a kv head, a warp has 16 of them, and all warps share
// tiles of 64 positions, the next one in flight.  The C CTAs of a cluster take the
// item's tiles in turn; one launch, no work split and no second kernel, which
// cost more than the work here.
constexpr uint32_t kShortRows = 64, kShortPos = 64;
template <uint32_t HD>
struct ShortCfg {
  static constexpr uint32_t kHalf = kSub * HD * 2, kTile = 2 * kHalf, LD = HD + 4;  // 32 positions, 64; floats of a row of a piece
  static constexpr uint32_t kTiles = 2 * 2 * kTile, kPiece = kShortRows * LD * 4 + kShortRows * 8, kBytes = kTiles > kPiece ? kTiles : kPiece;
};
template <typename T, uint32_t HD, uint32_t C, typename PR>
__global__ void __launch_bounds__(kThreads, 2) k_attn_short(const PR p) {
  using S = ShortCfg<HD>;
  extern __shared__ __align__(128) uint8_t dsm[];
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const T *base = reinterpret_cast<const T *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
  const uint32_t item = blockIdx.x / C, kvh = p.pg.n_kv_heads, tiles = (p.max_q * p.rep + kShortRows - 1) / kShortRows;
  Segment s;
  s.chunk = load_chunk(p, item / (kvh * tiles));
  s.tile = item / kvh % tiles;
  s.head = item % kvh;
  s.r0 = s.tile * kShortRows;
  if (s.r0 >= s.chunk.rows) return;  // the whole cluster
  s.r1 = min(s.chunk.rows, s.r0 + kShortRows);
  tile_range(p, s.chunk, s.r0, s.r1, s.lo, s.hi);
  const uint32_t n = s.hi > s.lo ? range_units<kShortPos>(p, s.lo, s.hi) : 0;
  const uint32_t *pt = p.pg.page_table + (uint64_t)s.chunk.seq * p.pg.max_pages;
  uint32_t u = cluster_ctarank();
  // K and V of tile u, whose pages are looked up a tile ahead, to buffer `which`
  PagePair ahead[2];
  auto pages = [&](uint32_t u) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) ahead[h] = look_up(p, pt, tile_at<kShortPos>(p, s.lo, u, h), s.lo, s.hi);
  };
  auto fetch = [&](uint32_t u, uint32_t which) {
    const uint32_t k = smem_u32(dsm) + which * 2 * S::kTile;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const Tile at = tile_at<kShortPos>(p, s.lo, u, h);
      flag_bad_pages(p, ahead[h]);
      stage<T, HD>(p, base, ahead[h], s.head, 0, at, s.lo, s.hi, k + h * S::kHalf, tid, kThreads);
      stage<T, HD>(p, base, ahead[h], s.head, 1, at, s.lo, s.hi, k + S::kTile + h * S::kHalf, tid, kThreads);
    }
    pages(u + C);
  };
  pages(u);
  if (u < n) fetch(u, 0);
  cp_commit();
  if (u + C < n) fetch(u + C, 1);
  cp_commit();
  const uint32_t first = s.r0 + 16 * warp;
  const bool mine = first < s.r1;
  Rows<T, HD> rows;
  rows.load(p, s, mine ? first : s.r0);
  for (uint32_t which = 0; u < n; u += C, which ^= 1) {
    cp_wait<1>();
    __syncthreads();
    const uint32_t k = smem_u32(dsm) + which * 2 * S::kTile;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const Tile at = tile_at<kShortPos>(p, s.lo, u, h);
      if (!mine || (int32_t)at.t[0] > rows.pos_max) continue;  // nothing of it is seen
      float sc[kSub / 8][4];
      rows.scores(k + h * S::kHalf, sc);
      rows.softmax(p, at, sc);
      rows.add_values(k + S::kTile + h * S::kHalf, sc);
    }
    __syncthreads();
    if (u + 2 * C < n) fetch(u + 2 * C, which);
    cp_commit();
  }
  cp_wait<0>();
  rows.finish();
  float *o = reinterpret_cast<float *>(dsm), *ml = o + kShortRows * S::LD;
  __syncthreads();
  if (mine) {
#pragma unroll
    for (uint32_t j = 0; j < HD / 8; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i)
        *reinterpret_cast<float2 *>(o + (warp * 16 + g + 8 * i) * S::LD + 8 * j + 2 * c) = make_float2(rows.o[j][2 * i], rows.o[j][2 * i + 1]);
    if (c == 0)
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) *reinterpret_cast<float2 *>(ml + (warp * 16 + g + 8 * i) * 2) = make_float2(rows.m[i], rows.l[i]);
  }
  one_join<kThreads, C>(s, HD, o, S::LD, ml, [&](uint32_t r, uint32_t d, float4 x) { put4(p, out_row<T>(p, s, s.r0 + r, HD) + d, x); });
}
template <typename T, uint32_t HD, uint32_t C>
int launch_short_c(const AttnChunksParams &p, uint64_t items, cudaStream_t st) {
  return with_sinks<PackedParams>(p, [&](auto a) { return launch_one<k_attn_short<T, HD, C, decltype(a)>, C>(a, items, kThreads, ShortCfg<HD>::kBytes, st); });
}
template <typename T, uint32_t HD>
int launch_short_hd(const AttnChunksParams &p, uint64_t items, uint32_t c, cudaStream_t st) {
  return c == 8 ? launch_short_c<T, HD, 8>(p, items, st) : c == 4 ? launch_short_c<T, HD, 4>(p, items, st)
       : c == 2 ? launch_short_c<T, HD, 2>(p, items, st) : launch_short_c<T, HD, 1>(p, items, st);
}

}  // namespace

int launch_short_mma(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st) {
  const uint64_t tiles = ((uint64_t)p.max_q * p.rep + kShortRows - 1) / kShortRows, items = one_items(p) * tiles;
  if (items > 2 * n_sm) return 1;
  const uint32_t c = items * 8 <= 2 * n_sm ? 8 : items * 4 <= 2 * n_sm ? 4 : items * 2 <= 2 * n_sm ? 2 : 1;
  const uint64_t units = (one_span(p) + kShortPos - 1) / kShortPos;
  // A tile takes some 2 us, and the tcgen05 kernel with its join 12 to 16 us before
  // its first.  32/8 heads x 128, here against there: 5 tokens of 100 positions 6.0
  // us against 11.8, of 1000 (2 tiles a CTA) 9.0 against 19.1, of 4000 (8) 20.1
  // against 22.3; 32 of 1000 (2) 12.5 against 20.4, of 4000 (8) 27.4 against 23.6; 128
  // over themselves 9.4 against 15.5, 512 (8) 25.9 against 24.8.
  if ((units + c - 1) / c > 6) return 1;
  if (p.pg.dtype == FA_KV_F16) return p.pg.head_dim == 64 ? launch_short_hd<__half, 64>(p, items, c, st) : launch_short_hd<__half, 128>(p, items, c, st);
  return p.pg.head_dim == 64 ? launch_short_hd<__nv_bfloat16, 64>(p, items, c, st) : launch_short_hd<__nv_bfloat16, 128>(p, items, c, st);
}

int launch_one_mma(const AttnChunksParams &p, cudaStream_t st) {
  if ((uint64_t)p.max_q * p.rep > kMmaRows) return 1;
  // A cluster streams some 0.7 TB/s, so the longer the cache the more of them
  // must run beside one another to keep up with the even split over all SMs, which
  // costs a join.  One token, kv heads x 128, clusters against split: 8 heads over
  // 1024, 8192, 16384 and 65536 positions 6.4, 11.9, 17.8 and 55 us against 9.8,
  // 17.0, 21.2 and 53; 2 heads over 1024, 8192 and 32768 6.1, 11.1 and 29.7 against
  // 9.2, 11.0 and 19.1; three sequences x 8 heads of 8192 21.6 against 26.8.
  const uint64_t span = one_span(p), items = (uint64_t)p.n_chunks * p.pg.n_kv_heads;
  if (span > (items >= 8 ? 16384 : 8192)) return 1;
  if (p.pg.dtype == FA_KV_F16) return p.pg.head_dim == 64 ? launch_one_hd<__half, 64>(p, span, st) : launch_one_hd<__half, 128>(p, span, st);
  return p.pg.head_dim == 64 ? launch_one_hd<__nv_bfloat16, 64>(p, span, st) : launch_one_hd<__nv_bfloat16, 128>(p, span, st);
}

// 16-bit types at head sizes 64 and 128; TMA counts the rows of a layer's pages
// in 31 bits
bool attn_mma_takes(const AttnChunksParams &p) {
  return p.pg.dtype != FA_KV_F32 && (p.pg.head_dim == 64 || p.pg.head_dim == 128) &&
         (uint64_t)p.pg.n_pages * 2 * p.pg.n_kv_heads * kPageLen < 0x7FFFFFFFull;
}

uint32_t launch_attn_mma(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st) {
  if (p.pg.dtype == FA_KV_F16) return p.pg.head_dim == 64 ? launch_hd<__half, 64>(p, n_sm, st) : launch_hd<__half, 128>(p, n_sm, st);
  return p.pg.head_dim == 64 ? launch_hd<__nv_bfloat16, 64>(p, n_sm, st) : launch_hd<__nv_bfloat16, 128>(p, n_sm, st);
}

}  // namespace fa
