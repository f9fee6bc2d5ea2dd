// Attention of chunks over paged K/V with f32 arithmetic, for every element
// type and every head size (a multiple of 8 up to 256): the path of f32 caches
// and of head sizes the tensor-core kernels are not made for.
//
//   o_r = sum_t e^(s_rt - m_r) v_t / sum_t e^(s_rt - m_r),  s_rt = scale q_r.k_t
//
// over one pass of the positions, with a running maximum m and sum l of a row:
// where m grows to m', l and o are multiplied by e^(m - m').
//
// An item is R rows of a kv head; tiles of 64 positions of K and V go through
// shared memory.  Scores: a thread has R/8 rows x 4 positions, outputs: R/8
// rows x hd/16 elements, each pair of operands read as float4, so 16 FMA per
// (R/8 + 4) loads of 16 bytes.  Few rows (decode) are bound by HBM, many by
// the FMA pipes and shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "paged_attn.cuh"

namespace fa {
namespace {

constexpr uint32_t kAnyThreads = 128, kAnyPos = 64;

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]);  // 16-byte aligned
template <>
__device__ __forceinline__ void load8<__half>(const __half *p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const __half2 *h = reinterpret_cast<const __half2 *>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// K and V of positions [t0, t0 + 64) to shared memory as f32; positions outside
// the item's range and bad pages as zeros.  The tile's four pages are looked up
// first and the copies are independent, so that they are all in flight: f32 by
// cp.async, 16-bit types through registers.  (A look-up with each 32-byte load
// took 19 us for a tile where this takes 8.)
template <typename T>
__device__ __forceinline__ void fetch(const AttnChunksParams &p, const T *base, const uint32_t *pt, const Segment &s, uint32_t t0,
                                      float *sk, float *sv, uint32_t ld, uint32_t tid) {
  constexpr uint32_t kV = 16 / sizeof(T);  // elements of a copy
  const uint32_t hd = p.pg.head_dim, per_row = hd / kV, total = 2 * kAnyPos * per_row;
  uint32_t page[kAnyPos / kPageLen];
#pragma unroll
  for (uint32_t j = 0; j < kAnyPos / kPageLen; ++j) {
    const uint32_t t = t0 + j * kPageLen;
    page[j] = t < s.hi && t + kPageLen > s.lo ? __ldg(pt + t / kPageLen) : 0u;
  }
  bool bad = false;
  uint64_t row0[kAnyPos / kPageLen];
#pragma unroll
  for (uint32_t j = 0; j < kAnyPos / kPageLen; ++j) {
    bad |= page[j] >= p.pg.n_pages;
    row0[j] = page[j] < p.pg.n_pages ? page_row(p.pg, page[j], 0, s.head, 0) : ~0ull;
  }
  if (bad && p.err) atomicOr(p.err, kFlagPage);
  const uint64_t v_off = (uint64_t)p.pg.n_kv_heads * kPageLen * hd;  // V after the heads' K
#pragma unroll 4
  for (uint32_t i = tid; i < total; i += kAnyThreads) {
    const uint32_t e = i / per_row, d = (i - e * per_row) * kV, is_v = e / kAnyPos, r = e % kAnyPos, t = t0 + r, j = r / kPageLen;
    const uint64_t r0 = j == 0 ? row0[0] : j == 1 ? row0[1] : j == 2 ? row0[2] : row0[3];
    const bool ok = t >= s.lo && t < s.hi && r0 != ~0ull;
    const T *src = base + (ok ? r0 + is_v * v_off + (t % kPageLen) * hd + d : 0);
    float *dst = (is_v ? sv : sk) + r * ld + d;
    if constexpr (sizeof(T) == 4) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16u : 0u) : "memory");
    } else {
      float x[8] = {};
      if (ok) load8(src, x);
      reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
  }
  if constexpr (sizeof(T) == 4) asm volatile("cp.async.wait_all;" ::: "memory");
}

constexpr uint32_t any_smem(uint32_t R, uint32_t hd) { return ((R + 2 * kAnyPos) * (hd + 4) + R * (kAnyPos + 4)) * 4; }

// HJ: groups of 64 head elements (hd <= 64 HJ).  A thread's rows are ty + 8 i, its
// elements 64 j + 4 tx + e.
template <typename T, uint32_t R, uint32_t HJ>
struct AnyRows {
  static constexpr uint32_t RT = R / 8;
  float m[RT], l[RT], o[RT][HJ][4];

  // units u, u + step, .. < n of an item
  __device__ void run(const AttnChunksParams &p, const Segment &s, uint32_t u, uint32_t n, uint32_t step, float *sm) {
    const uint32_t hd = p.pg.head_dim, ld = hd + 4, lds = kAnyPos + 4;
    float *sq = sm, *sk = sq + R * ld, *sv = sk + kAnyPos * ld, *sp = sv + kAnyPos * ld;
    const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const T *base = reinterpret_cast<const T *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
    const uint32_t *pt = p.pg.page_table + (uint64_t)s.chunk.seq * p.pg.max_pages;
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
    for (; u < n && s.hi > s.lo; u += step) {
      const uint32_t t0 = (s.lo / kAnyPos + u) * kAnyPos;
      __syncthreads();
      fetch<T>(p, base, pt, s, t0, sk, sv, ld, tid);
      __syncthreads();
      float a[RT][4];
#pragma unroll
      for (uint32_t i = 0; i < RT; ++i) a[i][0] = a[i][1] = a[i][2] = a[i][3] = 0.0f;
      for (uint32_t d = 0; d < hd; d += 4) {
        float4 kk[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) kk[j] = *reinterpret_cast<const float4 *>(sk + (tx + 16 * j) * ld + d);
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
          const float4 q = *reinterpret_cast<const float4 *>(sq + (ty + 8 * i) * ld + d);
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j)
            a[i][j] = fmaf(q.x, kk[j].x, fmaf(q.y, kk[j].y, fmaf(q.z, kk[j].z, fmaf(q.w, kk[j].w, a[i][j]))));
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < RT; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const int32_t t = (int32_t)(t0 + tx + 16 * j);
          const bool see = t <= pos[i] && (!p.window || (uint32_t)(pos[i] - t) < p.window);
          a[i][j] = see ? a[i][j] * p.scale_log2 : -INFINITY;
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
            const float4 v = *reinterpret_cast<const float4 *>(sv + (t + e) * ld + d);
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
    }
  }
};

template <typename T, uint32_t R, uint32_t HJ>
__global__ void __launch_bounds__(kAnyThreads) k_attn_any(const AttnChunksParams p) {
  extern __shared__ __align__(16) float sm[];
  __shared__ uint64_t red[kAnyThreads / 32 + 2];
  const uint32_t hd = p.pg.head_dim, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  using W = Walk<R, kAnyPos, 0, kAnyThreads>;
  W w;
  w.start(p, 1, red);
  if (tid == 0) p.desc[blockIdx.x].w = 0;
  for (Segment s; w.next(p, s);) {
    __syncthreads();
    AnyRows<T, R, HJ> x;
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

// few items of up to R rows: a cluster each (paged_attn.cuh)
template <typename T, uint32_t R, uint32_t HJ>
__global__ void __launch_bounds__(kAnyThreads) k_attn_any_one(const AttnChunksParams p) {
  extern __shared__ __align__(16) float sm[];
  const uint32_t hd = p.pg.head_dim, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  Segment s;
  if (!one_item(p, s)) return;
  AnyRows<T, R, HJ> x;
  x.run(p, s, cluster_ctarank(), range_units<kAnyPos>(s.lo, s.hi), kOneCtas, sm);
  float *o = sm + R * (hd + 4), *ml = o + R * hd;  // over K and V, which have been read
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
  one_join<kAnyThreads>(s, hd, o, ml, [&](uint32_t r, uint32_t d, float4 y) {
    T *out = reinterpret_cast<T *>(p.out) + (uint64_t)(s.chunk.q0 + r / p.rep) * p.os + (s.head * p.rep + r % p.rep) * hd + d;
    put(out, y.x);
    put(out + 1, y.y);
    put(out + 2, y.z);
    put(out + 3, y.w);
  });
}

template <typename T, uint32_t R, uint32_t HJ>
uint32_t launch_hj(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *rows) {
  const uint32_t smem = any_smem(R, p.pg.head_dim);
  if (cudaFuncSetAttribute(k_attn_any<T, R, HJ>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)any_smem(R, 64 * HJ)) !=
      cudaSuccess)
    return 0;
  uint32_t per_sm = 224 * 1024 / (smem + 1024);
  per_sm = per_sm > 3 ? 3 : per_sm;
  const uint32_t grid = n_sm * per_sm < kAttnMaxCtas ? n_sm * per_sm : kAttnMaxCtas;
  k_attn_any<T, R, HJ><<<grid, kAnyThreads, smem, st>>>(p);
  *rows = R;
  return cudaGetLastError() == cudaSuccess ? grid : 0;
}
template <typename T, uint32_t R, uint32_t HJ>
struct LaunchAny {
  static uint32_t walk(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st, uint32_t *rows) { return launch_hj<T, R, HJ>(p, n_sm, st, rows); }
  static int one(const AttnChunksParams &p, cudaStream_t st) {
    return launch_one<k_attn_any_one<T, R, HJ>>(p, kAnyThreads, any_smem(R, 64 * HJ), st);
  }
};
// f(LaunchAny of the call's type, rows and head size)
template <typename T, typename F>
auto with_hd(const AttnChunksParams &p, F f) {
  const uint32_t hd = p.pg.head_dim;
  // items of 8 or 16 rows while no chunk has more: few rows would leave most of
  // 32 idle in the FMA loops
  const uint64_t rows = (uint64_t)p.max_q * p.rep;
  auto with_rows = [&](auto hj) {
    constexpr uint32_t HJ = decltype(hj)::value;
    return rows <= 8 ? f(LaunchAny<T, 8, HJ>()) : rows <= 16 ? f(LaunchAny<T, 16, HJ>()) : f(LaunchAny<T, 32, HJ>());
  };
  if (hd <= 64) return with_rows(std::integral_constant<uint32_t, 1>());
  if (hd <= 128) return with_rows(std::integral_constant<uint32_t, 2>());
  return with_rows(std::integral_constant<uint32_t, 4>());
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
  if ((uint64_t)p.max_q * p.rep > 32) return 1;
  // While a CTA has one tile: 5 sequences of 512 positions with 12 rows, 2 kv heads
  // x 64, 13.1 us against 18.1 in two launches; of 2048 36.7 against 23.3.
  if (one_span(p) > kOneCtas * kAnyPos) return 1;
  return with_kind(p, [&](auto k) { return k.one(p, st); });
}

}  // namespace fa
