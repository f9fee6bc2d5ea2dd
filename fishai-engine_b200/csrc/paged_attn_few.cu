// Attention of chunks over paged K/V with f32 arithmetic and up to 16 rows per kv
// head: single tokens and a few at a time over f32 caches, and over 16-bit ones of
// the head sizes that paged_attn_mma.cu is not made for.  Same mathematics as
// paged_attn_any.cu.
//
// Reads of shared memory bound it (each fills registers at 128 bytes a clock and
// SM, broadcast or not), so the operands are shared out to be read seldom.  Scores
// of a tile of 64 positions: a warp has half of the positions and every other
// group of four elements, a lane R/4 rows x 4 positions, and the two halves of the
// sums meet in shared memory.  Softmax: 16 threads a row, 4 positions each.
// Outputs: a warp has 16 of the positions, a lane DPL elements of all rows; the
// four warps' sums meet at the end of a piece.  The next K is on its way once the
// scores are formed, the next V once its product is done.  8 f32 sequences of 8192
// positions, 32/8 heads x 128: 146 us, 3.7 TB/s; one 32 us; of 64 positions 8.8.
// (paged_attn_any.cu's way for 8 rows: 210, 42 and 11.2; a warp to its own
// positions, a lane to one: 217, 38 and 12.8.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "paged_attn.cuh"

namespace fa {
namespace {

constexpr uint32_t kPos = 64, kThreads = 128, kWarps = 4, kRow = kPos + 8;  // kRow: floats of a row of scores, on distinct banks

// N consecutive elements as f32, aligned to their size (16 bytes at most)
template <uint32_t N, typename T>
__device__ __forceinline__ void load(const T *p, float (&x)[N]) {
  if constexpr (sizeof(T) * N > 16) {
    float a[N / 2], b[N / 2];
    load<N / 2>(p, a);
    load<N / 2>(p + N / 2, b);
#pragma unroll
    for (uint32_t i = 0; i < N / 2; ++i) x[i] = a[i], x[N / 2 + i] = b[i];
  } else {
    struct alignas(sizeof(T) * N) Vec {
      T v[N];
    };
    const Vec v = *reinterpret_cast<const Vec *>(p);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[i] = (float)v.v[i];
  }
}
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// R rows, DPL head elements of a lane (head_dim <= 32 DPL)
template <typename T, uint32_t R, uint32_t DPL>
struct FewCfg {
  static constexpr uint32_t kOver = 1;  // an item's own cost, in tiles
  static constexpr uint32_t row(uint32_t hd) { return hd + 16 / (uint32_t)sizeof(T); }  // elements: rows of a tile on distinct banks
  static constexpr uint32_t tiles(uint32_t hd) { return 2 * kPos * row(hd) * (uint32_t)sizeof(T); }
  // after a piece, over the tiles: the warps' outputs, then the CTA's with (max, sum)
  static constexpr uint32_t merge(uint32_t hd) { return kWarps * R * (hd + 4) * 4; }
  static constexpr uint32_t over(uint32_t hd) {
    const uint32_t m = merge(hd) + R * (hd + 2) * 4;
    return m > tiles(hd) ? m : tiles(hd);
  }
  // then the two halves of the scores, Q, and the rows' factors
  static constexpr uint32_t smem(uint32_t hd) { return over(hd) + 2 * R * kRow * 4 + R * (hd + 4) * 4 + R * 4; }
};

template <typename T, uint32_t R, uint32_t DPL>
struct FewRows {
  using C = FewCfg<T, R, DPL>;
  float m[R / 8], l[R / 8], o[R][DPL];  // m, l: of rows tid / 16 + 8 k; l: the thread's part

  // Units u, u + step, .. < n of an item.
  __device__ void run(const AttnChunksParams &p, const Segment &s, uint32_t u, uint32_t n, uint32_t step, uint8_t *sm) {
    __shared__ uint64_t at[2][kPos / kPageLen];  // element offsets of the tile's pages, and of the next tile's
    const uint32_t hd = p.pg.head_dim, ld = C::row(hd), ldq = hd + 4, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    T *sk = reinterpret_cast<T *>(sm), *sv = sk + kPos * ld;
    float *part = reinterpret_cast<float *>(sm + C::over(hd)), *sq = part + 2 * R * kRow, *sf = sq + R * ldq;
    const T *base = reinterpret_cast<const T *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
    const T *vbase = base + (uint64_t)p.pg.n_kv_heads * kPageLen * hd;  // V after the heads' K
    const uint32_t *pt = p.pg.page_table + (uint64_t)s.chunk.seq * p.pg.max_pages;
    if (s.hi <= s.lo) n = 0;
    // copies: piece c of row r, both carried along
    constexpr uint32_t kV = 16 / sizeof(T);
    const uint32_t per_row = hd / kV, r0 = tid / per_row, c0 = tid - r0 * per_row, dr = kThreads / per_row, dc = kThreads - dr * per_row;
    // thread j < 4: page j of the tile at t0; only pages that are read are looked up
    auto look_up = [&](uint32_t t0) -> uint32_t {
      const uint32_t t = t0 + tid * kPageLen;
      return tid < kPos / kPageLen && t < s.hi && t + kPageLen > s.lo ? __ldg(pt + t / kPageLen) : 0u;
    };
    auto note = [&](uint32_t page, uint32_t which) {
      if (tid >= kPos / kPageLen) return;
      const bool good = page < p.pg.n_pages;
      at[which][tid] = good ? page_row(p.pg, page, 0, s.head, 0) : ~0ull;
      if (!good && p.err) atomicOr(p.err, kFlagPage);
    };
    // positions outside [lo, hi) and of bad pages become zeros
    auto copy = [&](const T *src, uint32_t which, uint32_t t0, T *dst) {
      for (uint32_t r = r0, c = c0; r < kPos;) {
        const uint64_t row0 = at[which][r / kPageLen];
        const bool ok = t0 + r >= s.lo && t0 + r < s.hi && row0 != ~0ull;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * ld + c * kV)),
                     "l"(ok ? src + row0 + (r % kPageLen) * hd + c * kV : src), "r"(ok ? 16u : 0u)
                     : "memory");
        r += dr;
        c += dc;
        if (c >= per_row) {
          c -= per_row;
          ++r;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t t0 = (s.lo / kPos + u) * kPos;
    if (u < n) {
      note(look_up(t0), 0);
      __syncthreads();
      copy(base, 0, t0, sk);
      copy(vbase, 0, t0, sv);
    }
    // Q rows, past the item's zeros
    for (uint32_t r = warp; r < R; r += kWarps) {
      const uint32_t row = s.r0 + r, tok = row / p.rep;
      const T *x = reinterpret_cast<const T *>(p.q) + (uint64_t)(s.chunk.q0 + tok) * p.qs + (s.head * p.rep + row - tok * p.rep) * hd;
      for (uint32_t d = lane; d < hd; d += 32) sq[r * ldq + d] = row < s.r1 ? (float)x[d] : 0.0f;
    }
    const uint32_t c4 = tid % 16 * 4;
    int32_t pos[R / 8];  // of the tokens of the thread's rows in the softmax; -1: no row
#pragma unroll
    for (uint32_t k = 0; k < R / 8; ++k) {
      const uint32_t row = s.r0 + tid / 16 + 8 * k;
      m[k] = -INFINITY;
      l[k] = 0.0f;
      pos[k] = row < s.r1 ? s.chunk.first + (int32_t)(row / p.rep) : -1;
    }
#pragma unroll
    for (uint32_t r = 0; r < R; ++r)
#pragma unroll
      for (uint32_t e = 0; e < DPL; ++e) o[r][e] = 0.0f;
    for (uint32_t which = 0; u < n; u += step, which ^= 1) {
      const bool more = u + step < n;
      const uint32_t t1 = t0 + step * kPos, ahead = more ? look_up(t1) : 0;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      {
        const uint32_t rp = lane >> 3, p0 = (warp >> 1) * 32 + (lane & 7);
        float a[R / 4][4] = {};
#pragma unroll 2
        for (uint32_t d = 4 * (warp & 1); d < hd; d += 8) {
          float k[4][4];
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) load<4>(sk + (p0 + 8 * j) * ld + d, k[j]);
#pragma unroll
          for (uint32_t i = 0; i < R / 4; ++i) {
            const float4 q = *reinterpret_cast<const float4 *>(sq + (rp + 4 * i) * ldq + d);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) a[i][j] = fmaf(q.x, k[j][0], fmaf(q.y, k[j][1], fmaf(q.z, k[j][2], fmaf(q.w, k[j][3], a[i][j]))));
          }
        }
#pragma unroll
        for (uint32_t i = 0; i < R / 4; ++i)
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) part[((warp & 1) * R + rp + 4 * i) * kRow + p0 + 8 * j] = a[i][j];
      }
      if (more) note(ahead, which ^ 1);
      __syncthreads();
      if (more) copy(base, which ^ 1, t1, sk);
      else asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
      for (uint32_t k = 0; k < R / 8; ++k) {
        const uint32_t row = tid / 16 + 8 * k;
        float4 *w = reinterpret_cast<float4 *>(part + row * kRow + c4);
        const float4 x = *w, y = *reinterpret_cast<const float4 *>(part + (R + row) * kRow + c4);
        float a[4] = {x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w}, mx = -INFINITY;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          const int32_t t = (int32_t)(t0 + c4 + e);
          const bool see = t <= pos[k] && (!p.window || (uint32_t)(pos[k] - t) < p.window);
          a[e] = see ? a[e] * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, a[e]);
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, off));
        const float mn = fmaxf(m[k], mx), ms = mn == -INFINITY ? 0.0f : mn, f = exp2f(m[k] - ms);
        m[k] = mn;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) a[e] = exp2f(a[e] - ms);
        l[k] = fmaf(l[k], f, (a[0] + a[1]) + (a[2] + a[3]));
        *w = make_float4(a[0], a[1], a[2], a[3]);
        if (tid % 16 == 0) sf[row] = f;
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
#pragma unroll
      for (uint32_t r = 0; r < R; ++r) {
        const float f = sf[r];
#pragma unroll
        for (uint32_t e = 0; e < DPL; ++e) o[r][e] *= f;
      }
      if (lane * DPL < hd) {
#pragma unroll
        for (uint32_t i = 0; i < kPos / kWarps; i += 4) {
          const uint32_t t = warp * (kPos / kWarps) + i;
          float v[4][DPL];
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) load<DPL>(sv + (t + j) * ld + lane * DPL, v[j]);
#pragma unroll
          for (uint32_t r = 0; r < R; ++r) {
            const float4 w = *reinterpret_cast<const float4 *>(part + r * kRow + t);
#pragma unroll
            for (uint32_t e = 0; e < DPL; ++e) o[r][e] = fmaf(w.x, v[0][e], fmaf(w.y, v[1][e], fmaf(w.z, v[2][e], fmaf(w.w, v[3][e], o[r][e]))));
          }
        }
      }
      __syncthreads();
      if (more) copy(vbase, which ^ 1, t1, sv);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      t0 = t1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (uint32_t k = 0; k < R / 8; ++k)
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) l[k] += __shfl_xor_sync(0xFFFFFFFFu, l[k], off);
    // outputs of the warps, and the rows' (max, sum), over the tiles
    float *all = reinterpret_cast<float *>(sm), *ml = reinterpret_cast<float *>(sm + C::merge(hd)) + R * hd;
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < R; ++r)
      if (lane * DPL < hd)
#pragma unroll
        for (uint32_t e = 0; e < DPL; e += 2)
          *reinterpret_cast<float2 *>(all + (warp * R + r) * (hd + 4) + lane * DPL + e) = make_float2(o[r][e], o[r][e + 1]);
#pragma unroll
    for (uint32_t k = 0; k < R / 8; ++k)
      if (tid % 16 == 0) *reinterpret_cast<float2 *>(ml + 2 * (tid / 16 + 8 * k)) = make_float2(m[k], l[k]);
    __syncthreads();
  }
  // elements d .. d + 3 of row r after run(), and the row's (max, sum)
  __device__ static float4 sum(const uint8_t *sm, uint32_t hd, uint32_t r, uint32_t d) {
    const float *all = reinterpret_cast<const float *>(sm) + r * (hd + 4) + d;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (uint32_t v = 0; v < kWarps; ++v) {
      const float4 x = *reinterpret_cast<const float4 *>(all + v * R * (hd + 4));
      acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
    }
    return acc;
  }
  __device__ static float2 max_sum(const uint8_t *sm, uint32_t hd, uint32_t r) {
    return *reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(sm + C::merge(hd)) + R * hd + 2 * r);
  }
};
template <typename T>
__device__ __forceinline__ void put_row(const AttnChunksParams &p, const Segment &s, uint32_t row, uint32_t d, float4 x) {
  const uint32_t hd = p.pg.head_dim;
  T *o = reinterpret_cast<T *>(p.out) + (uint64_t)(s.chunk.q0 + row / p.rep) * p.os + (s.head * p.rep + row % p.rep) * hd + d;
  put(o, x.x);
  put(o + 1, x.y);
  put(o + 2, x.z);
  put(o + 3, x.w);
}

template <typename T, uint32_t R, uint32_t DPL>
__global__ void __launch_bounds__(kThreads) k_attn_few(const AttnChunksParams p) {
  using C = FewCfg<T, R, DPL>;
  extern __shared__ __align__(16) uint8_t few_sm[];
  __shared__ uint64_t red[kWarps + 2];
  const uint32_t hd = p.pg.head_dim, tid = threadIdx.x;
  using W = Walk<R, kPos, C::kOver, kThreads>;
  W w;
  w.start(p, 1, red);
  if (tid == 0) p.desc[blockIdx.x].w = 0;
  for (Segment s; w.next(p, s);) {
    FewRows<T, R, DPL> x;
    x.run(p, s, s.u0, s.u1, 1, few_sm);
    const bool whole = W::whole(s);
    float *slot = W::slot(p, s);
    for (uint32_t i = tid; i < (s.r1 - s.r0) * (hd / 4); i += kThreads) {
      const uint32_t r = i / (hd / 4), d = (i - r * (hd / 4)) * 4;
      const float4 acc = x.sum(few_sm, hd, r, d);
      const float2 ml = x.max_sum(few_sm, hd, r);
      if (whole) {
        const float inv = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
        put_row<T>(p, s, s.r0 + r, d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      } else {
        *reinterpret_cast<float4 *>(slot + r * hd + d) = acc;
        if (d == 0) *reinterpret_cast<float2 *>(slot + R * hd + 2 * r) = ml;
      }
    }
    if (!whole && s.u0 == 0 && tid == 0) p.desc[blockIdx.x] = w.describe(s);
    __syncthreads();  // the next piece copies over the scratch
  }
  pdl_launch_dependents();
}

// few items: a cluster each (paged_attn.cuh)
template <typename T, uint32_t R, uint32_t DPL>
__global__ void __launch_bounds__(kThreads) k_attn_few_one(const AttnChunksParams p) {
  using C = FewCfg<T, R, DPL>;
  extern __shared__ __align__(16) uint8_t few_sm[];
  const uint32_t hd = p.pg.head_dim, tid = threadIdx.x;
  Segment s;
  if (!one_item(p, s)) return;
  FewRows<T, R, DPL> x;
  x.run(p, s, cluster_ctarank(), range_units<kPos>(s.lo, s.hi), kOneCtas, few_sm);
  float *o = reinterpret_cast<float *>(few_sm + C::merge(hd));
  for (uint32_t i = tid; i < s.r1 * (hd / 4); i += kThreads) {
    const uint32_t r = i / (hd / 4), d = (i - r * (hd / 4)) * 4;
    *reinterpret_cast<float4 *>(o + r * hd + d) = x.sum(few_sm, hd, r, d);
  }
  one_join<kThreads>(s, hd, o, hd, o + R * hd, [&](uint32_t r, uint32_t d, float4 y) { put_row<T>(p, s, r, d, y); });
}

template <typename T, uint32_t R, uint32_t DPL>
struct LaunchFew {
  using C = FewCfg<T, R, DPL>;
  static uint32_t walk(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *rows) {
    const uint32_t smem = C::smem(p.pg.head_dim);
    if (cudaFuncSetAttribute(k_attn_few<T, R, DPL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::smem(32 * DPL)) != cudaSuccess) return 0;
    uint32_t per_sm = 228 * 1024 / (smem + 1024 + 256);  // 1 KB of the system, 256 bytes beside the tiles
    per_sm = per_sm > 3 ? 3 : per_sm;
    const uint32_t grid = n_sm * per_sm < kAttnMaxCtas ? n_sm * per_sm : kAttnMaxCtas;
    k_attn_few<T, R, DPL><<<grid, kThreads, smem, st>>>(p);
    *rows = R;
    return cudaGetLastError() == cudaSuccess ? grid : 0;
  }
  static int one(const AttnChunksParams &p, cudaStream_t st) {
    return launch_one<k_attn_few_one<T, R, DPL>>(p, one_items(p), kThreads, C::smem(32 * DPL), st);
  }
};
// f(LaunchFew of the call's type, rows and head size)
template <typename T, typename F>
auto with_hd(const AttnChunksParams &p, F f) {
  const uint32_t hd = p.pg.head_dim;
  const bool eight = (uint64_t)p.max_q * p.rep <= 8;
  auto with_rows = [&](auto dpl) {
    constexpr uint32_t DPL = decltype(dpl)::value;
    return eight ? f(LaunchFew<T, 8, DPL>()) : f(LaunchFew<T, 16, DPL>());
  };
  if (hd <= 64) return with_rows(std::integral_constant<uint32_t, 2>());
  if (hd <= 128) return with_rows(std::integral_constant<uint32_t, 4>());
  return with_rows(std::integral_constant<uint32_t, 8>());
}
template <typename F>
auto with_kind(const AttnChunksParams &p, F f) {
  switch (p.pg.dtype) {
    case FA_KV_F32: return with_hd<float>(p, f);
    case FA_KV_F16: return with_hd<__half>(p, f);
    default: return with_hd<__nv_bfloat16>(p, f);
  }
}

}  // namespace

uint32_t launch_attn_few(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *R) {
  return with_kind(p, [&](auto k) { return k.walk(p, n_sm, st, R); });
}
int launch_one_few(const AttnChunksParams &p, cudaStream_t st) {
  // While a CTA has two tiles at most: one f32 token over 1024 positions, 8 kv heads
  // x 128, 13.9 us against 14.4 in two launches, five chunks of 12 rows, 2 x 64,
  // 12.9 against 15.8; over 2048 22.9 against 16.4 and 19.5 against 18.1.
  if (one_span(p) > 2 * kOneCtas * kPos) return 1;
  return with_kind(p, [&](auto k) { return k.one(p, st); });
}

}  // namespace fa
