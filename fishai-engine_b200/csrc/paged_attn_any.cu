// Attention of chunks over paged K/V with f32 arithmetic and more than 16 rows per
// kv head, for every element type and every head size (a multiple of 8 up to
// 256): the path of f32 caches and of head sizes the tensor-core kernels are not
// made for.
//
//   o_r = sum_t e^(s_rt - m_r) v_t / sum_t e^(s_rt - m_r),  s_rt = scale q_r.k_t
//
// over one pass of the positions, with a running maximum m and sum l of a row:
// where m grows to m', l and o are multiplied by e^(m - m').
//
// An item is 32 rows of a kv head; tiles of 64 positions of K and V go through
// shared memory, copied one ahead.  Scores: a thread has 4 rows x 4 positions,
// outputs: 4 rows x hd/16 elements, each pair of operands read as float4, so 64 FMA
// per 8 loads of 16 bytes; the FMA pipes and shared memory bound it: 1024 f32
// tokens over themselves, 32/8 heads x 128, 716 us, 64 over 8192 positions 420.
// (Chunks of up to 16 rows: paged_attn_few.cu.  Its way of sharing the operands
// out, with 32 rows: 668 and 585 us.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_attn.cuh"

namespace fa {
namespace {

constexpr uint32_t kAnyThreads = 128, kAnyPos = 64, R = 32;  // R: rows of an item

// four elements, aligned to their size
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __half *p) {
  const uint2 a = *reinterpret_cast<const uint2 *>(p);
  const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&a.x)), y = __half22float2(*reinterpret_cast<const __half2 *>(&a.y));
  return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
  const uint2 a = *reinterpret_cast<const uint2 *>(p);
  const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&a.x)), y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&a.y));
  return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Copies of a tile's K or V rows, 16 bytes a thread and step: piece c of row r,
// both carried along (a division a piece took longer than the copies).
struct Copier {
  uint32_t r0, c0, dr, dc, per_row;
  __device__ Copier(uint32_t per_row) : per_row(per_row) {
    r0 = threadIdx.x / per_row, c0 = threadIdx.x - r0 * per_row;
    dr = kAnyThreads / per_row, dc = kAnyThreads - dr * per_row;
  }
  // src: rows of a page from at[page of the tile] on; positions that the item
  // does not see and bad pages (~0) become zeros
  template <typename T, typename PR>
  __device__ void copy(const PR &p, const T *src, const uint64_t *at, uint32_t t0, uint32_t lo, uint32_t hi, T *dst, uint32_t ld) const {
    constexpr uint32_t kV = 16 / sizeof(T);
    const uint32_t hd = p.pg.head_dim;
    for (uint32_t r = r0, c = c0; r < kAnyPos;) {
      const uint64_t row0 = at[r / kPageLen];
      const bool ok = item_sees(p, lo, hi, t0 + r) && row0 != ~0ull;
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
  }
};
__device__ __forceinline__ void copied_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// bytes: Q rows and weights in f32, K and V tiles in their own type, rows 16 bytes apart
template <typename T>
constexpr uint32_t any_smem(uint32_t hd) {
  return (R * (hd + 4) + R * (kAnyPos + 4)) * 4 + 2 * kAnyPos * (hd * (uint32_t)sizeof(T) + 16);
}

// HJ: groups of 64 head elements (hd <= 64 HJ).  A thread's rows are ty + 8 i, its
// elements 64 j + 4 tx + e.
template <typename T, uint32_t HJ>
struct AnyRows {
  static constexpr uint32_t RT = R / 8;
  float m[RT], l[RT], o[RT][HJ][4];

  // units u, u + step, .. < n of an item; the tile behind the one worked on is on
  // its way: its K once the scores are formed, its V once that product is done
  template <typename PR>
  __device__ void run(const PR &p, const Segment &s, uint32_t u, uint32_t n, uint32_t step, float *sm) {
    __shared__ uint64_t at[2][kAnyPos / kPageLen];  // element offsets of the tile's pages, and of the next tile's
    const uint32_t hd = p.pg.head_dim, ld = hd + 4, lds = kAnyPos + 4, ldk = hd + 16 / sizeof(T);
    float *sq = sm, *sp = sq + R * ld;
    T *sk = reinterpret_cast<T *>(sp + R * lds), *sv = sk + kAnyPos * ldk;
    const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const T *base = reinterpret_cast<const T *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
    const T *vbase = base + (uint64_t)p.pg.n_kv_heads * kPageLen * hd;  // V after the heads' K
    const uint32_t *pt = p.pg.page_table + (uint64_t)s.chunk.seq * p.pg.max_pages;
    if (s.hi <= s.lo) n = 0;
    const Copier copier(hd * sizeof(T) / 16);
    // thread j < 4: page j of the tile at t0; only pages that are read are looked up
    auto look_up = [&](uint32_t t0) -> uint32_t {
      const uint32_t t = t0 + tid * kPageLen;
      return tid < kAnyPos / kPageLen && item_reads(p, s.lo, s.hi, t) ? __ldg(pt + t / kPageLen) : 0u;
    };
    auto note = [&](uint32_t page, uint32_t which) {
      if (tid >= kAnyPos / kPageLen) return;
      const bool good = page < p.pg.n_pages;
      at[which][tid] = good ? page_row(p.pg, page, 0, s.head, 0) : ~0ull;
      if (!good && p.err) atomicOr(p.err, kFlagPage);
    };
    if (u < n) {
      const uint32_t t0 = unit_at<kAnyPos>(p, s.lo, u);
      note(look_up(t0), 0);
      __syncthreads();
      copier.copy(p, base, at[0], t0, s.lo, s.hi, sk, ldk);
      copier.copy(p, vbase, at[0], t0, s.lo, s.hi, sv, ldk);
    }
    // Q rows; past the item's: zeros
    for (uint32_t r = tid / 32; r < R; r += kAnyThreads / 32) {  // a warp a row
      const uint32_t row = s.r0 + r, tok = row / p.rep;
      const T *x = reinterpret_cast<const T *>(p.q) + (uint64_t)(s.chunk.q0 + tok) * p.qs + (s.head * p.rep + row - tok * p.rep) * hd;
#pragma unroll
      for (uint32_t j = 0; j < 2 * HJ; ++j) {
        const uint32_t d = tid % 32 + 32 * j;
        if (d < hd) sq[r * ld + d] = row < s.r1 ? (float)x[d] : 0.0f;
      }
    }
    int32_t pos[RT];  // position of each row's token
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
      const uint32_t row = s.r0 + ty + 8 * i;
      pos[i] = row < s.r1 ? s.chunk.first + (int32_t)(row / p.rep) : -1;
#pragma unroll
      for (uint32_t j = 0; j < HJ; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;
    }
    for (uint32_t which = 0; u < n; u += step, which ^= 1) {
      const uint32_t t0 = unit_at<kAnyPos>(p, s.lo, u), t1 = unit_after<kAnyPos>(p, s.lo, u, t0, step);
      const bool more = u + step < n;
      const uint32_t ahead = more ? look_up(t1) : 0;
      copied_but_one();
      __syncthreads();
      float a[RT][4];
#pragma unroll
      for (uint32_t i = 0; i < RT; ++i) a[i][0] = a[i][1] = a[i][2] = a[i][3] = 0.0f;
      for (uint32_t d = 0; d < hd; d += 4) {
        float4 kk[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) kk[j] = load4(sk + (tx + 16 * j) * ldk + d);
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
          const float4 q = *reinterpret_cast<const float4 *>(sq + (ty + 8 * i) * ld + d);
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j)
            a[i][j] = fmaf(q.x, kk[j].x, fmaf(q.y, kk[j].y, fmaf(q.z, kk[j].z, fmaf(q.w, kk[j].w, a[i][j]))));
        }
      }
      if (more) note(ahead, which ^ 1);
      __syncthreads();
      if (more) copier.copy(p, base, at[which ^ 1], t1, s.lo, s.hi, sk, ldk);
      else asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
      for (uint32_t i = 0; i < RT; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const int32_t t = (int32_t)(t0 + tx + 16 * j);
          a[i][j] = token_sees(p, pos[i], t) ? a[i][j] * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, a[i][j]);
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, off));
        const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: e^-inf = 0
        const float f = exp2f(m[i] - ms);
        float sum = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          a[i][j] = exp2f(a[i][j] - ms);
          sum += a[i][j];
          sp[(ty + 8 * i) * lds + tx + 16 * j] = a[i][j];
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
        l[i] = l[i] * f + sum;
        m[i] = mn;
#pragma unroll
        for (uint32_t j = 0; j < HJ; ++j) o[i][j][0] *= f, o[i][j][1] *= f, o[i][j][2] *= f, o[i][j][3] *= f;
      }
      copied_but_one();
      __syncthreads();
      for (uint32_t t = 0; t < kAnyPos; t += 4) {
        float4 pp[RT];
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) pp[i] = *reinterpret_cast<const float4 *>(sp + (ty + 8 * i) * lds + t);
#pragma unroll
        for (uint32_t j = 0; j < HJ; ++j) {
          const uint32_t d = 64 * j + 4 * tx;
          if (d >= hd) continue;
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            const float4 v = load4(sv + (t + e) * ldk + d);
#pragma unroll
            for (uint32_t i = 0; i < RT; ++i) {
              const float x = e == 0 ? pp[i].x : e == 1 ? pp[i].y : e == 2 ? pp[i].z : pp[i].w;
              o[i][j][0] = fmaf(x, v.x, o[i][j][0]);
              o[i][j][1] = fmaf(x, v.y, o[i][j][1]);
              o[i][j][2] = fmaf(x, v.z, o[i][j][2]);
              o[i][j][3] = fmaf(x, v.w, o[i][j][3]);
            }
          }
        }
      }
      __syncthreads();
      if (more) copier.copy(p, vbase, at[which ^ 1], t1, s.lo, s.hi, sv, ldk);
      else asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
};

template <typename T, uint32_t HJ, typename PR>
__global__ void __launch_bounds__(kAnyThreads) k_attn_any(const PR p) {
  extern __shared__ __align__(16) float sm[];
  __shared__ uint64_t red[kAnyThreads / 32 + 2];
  const uint32_t hd = p.pg.head_dim, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  using W = Walk<R, kAnyPos, 0, kAnyThreads>;
  W w;
  w.start(p, 1, red);
  if (tid == 0) p.desc[blockIdx.x].w = 0;
  for (Segment s; w.next(p, s);) {
    __syncthreads();
    AnyRows<T, HJ> x;
    x.run(p, s, s.u0, s.u1, 1, sm);
    const bool whole = W::whole(s);
    float *slot = W::slot(p, s);
#pragma unroll
    for (uint32_t i = 0; i < R / 8; ++i) {
      const uint32_t r = ty + 8 * i, row = s.r0 + r;
      if (row >= s.r1) continue;
      if (!whole && tx == 0) {
        slot[R * hd + 2 * r] = x.m[i];
        slot[R * hd + 2 * r + 1] = x.l[i];
      }
#pragma unroll
      for (uint32_t j = 0; j < HJ; ++j) {
        const uint32_t d = 64 * j + 4 * tx;
        if (d >= hd) continue;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          if (!whole) slot[r * hd + d + e] = x.o[i][j][e];
          else
            put(reinterpret_cast<T *>(p.out) + (uint64_t)(s.chunk.q0 + row / p.rep) * p.os +
                    (s.head * p.rep + row % p.rep) * hd + d + e,
                x.l[i] == 0.0f ? 0.0f : x.o[i][j][e] / x.l[i]);
        }
      }
    }
    if (!whole && s.u0 == 0 && tid == 0) p.desc[blockIdx.x] = w.describe(s);
  }
  pdl_launch_dependents();
}

// few items of up to 32 rows: a cluster each (paged_attn.cuh)
template <typename T, uint32_t HJ, typename PR>
__global__ void __launch_bounds__(kAnyThreads) k_attn_any_one(const PR p) {
  extern __shared__ __align__(16) float sm[];
  const uint32_t hd = p.pg.head_dim, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  Segment s;
  if (!one_item(p, s)) return;
  AnyRows<T, HJ> x;
  x.run(p, s, cluster_ctarank(), range_units<kAnyPos>(p, s.lo, s.hi), kOneCtas, sm);
  float *o = sm, *ml = o + R * hd;  // over Q and the weights, which have been read
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < R / 8; ++i) {
    const uint32_t r = ty + 8 * i;
    if (tx == 0) *reinterpret_cast<float2 *>(ml + 2 * r) = make_float2(x.m[i], x.l[i]);
#pragma unroll
    for (uint32_t j = 0; j < HJ; ++j) {
      const uint32_t d = 64 * j + 4 * tx;
      if (d < hd) *reinterpret_cast<float4 *>(o + r * hd + d) = make_float4(x.o[i][j][0], x.o[i][j][1], x.o[i][j][2], x.o[i][j][3]);
    }
  }
  one_join<kAnyThreads>(s, hd, o, hd, ml, [&](uint32_t r, uint32_t d, float4 y) {
    T *out = reinterpret_cast<T *>(p.out) + (uint64_t)(s.chunk.q0 + r / p.rep) * p.os + (s.head * p.rep + r % p.rep) * hd + d;
    put(out, y.x);
    put(out + 1, y.y);
    put(out + 2, y.z);
    put(out + 3, y.w);
  });
}

template <typename T, uint32_t HJ>
uint32_t launch_hj(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *rows) {
  const uint32_t smem = any_smem<T>(p.pg.head_dim);
  uint32_t per_sm = 224 * 1024 / (smem + 1024);
  per_sm = per_sm > 3 ? 3 : per_sm;
  const uint32_t grid = n_sm * per_sm < kAttnMaxCtas ? n_sm * per_sm : kAttnMaxCtas;
  *rows = R;
  return with_sinks<SinkParams>(p, [&](auto a) -> uint32_t {
    using PR = decltype(a);
    if (cudaFuncSetAttribute(k_attn_any<T, HJ, PR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)any_smem<T>(64 * HJ)) != cudaSuccess) return 0;
    k_attn_any<T, HJ><<<grid, kAnyThreads, smem, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? grid : 0;
  });
}
template <typename T, uint32_t HJ>
struct LaunchAny {
  static uint32_t walk(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *rows) { return launch_hj<T, HJ>(p, n_sm, st, rows); }
  static int one(const AttnChunksParams &p, cudaStream_t st) {
    return with_sinks<SinkParams>(p, [&](auto a) { return launch_one<k_attn_any_one<T, HJ, decltype(a)>>(a, one_items(p), kAnyThreads, any_smem<T>(64 * HJ), st); });
  }
};
// f(LaunchAny of the call's type, rows and head size)
template <typename T, typename F>
auto with_hd(const AttnChunksParams &p, F f) {
  const uint32_t hd = p.pg.head_dim;
  if (hd <= 64) return f(LaunchAny<T, 1>());
  if (hd <= 128) return f(LaunchAny<T, 2>());
  return f(LaunchAny<T, 4>());
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

uint32_t launch_attn_any(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *R) {
  return with_kind(p, [&](auto k) { return k.walk(p, n_sm, st, R); });
}
int launch_one_any(const AttnChunksParams &p, cudaStream_t st) {
  if ((uint64_t)p.max_q * p.rep > R) return 1;
  // While a CTA has one tile: 4 tokens of 8 heads each over 512 positions 20.6 us
  // against 29 in two launches; over 2048 59 against 38.
  if (one_span(p) > kOneCtas * kAnyPos) return 1;
  return with_kind(p, [&](auto k) { return k.one(p, st); });
}

}  // namespace fa
