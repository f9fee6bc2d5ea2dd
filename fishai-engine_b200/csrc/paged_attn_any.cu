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

#include "paged_attn.cuh"

namespace fa {
namespace {

constexpr uint32_t kAnyThreads = 128, kAnyPos = 64;

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]);  // 16-byte aligned
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
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

constexpr uint32_t any_smem(uint32_t R, uint32_t hd) { return ((R + 2 * kAnyPos) * (hd + 4) + R * (kAnyPos + 4)) * 4; }

// HJ: groups of 64 head elements (hd <= 64 HJ)
template <typename T, uint32_t R, uint32_t HJ>
__global__ void __launch_bounds__(kAnyThreads) k_attn_any(const AttnChunksParams p) {
  extern __shared__ __align__(16) float sm[];
  __shared__ uint64_t red[kAnyThreads / 32 + 2];
  constexpr uint32_t RT = R / 8;
  const uint32_t hd = p.pg.head_dim, ld = hd + 4, lds = kAnyPos + 4;
  float *sq = sm, *sk = sq + R * ld, *sv = sk + kAnyPos * ld, *sp = sv + kAnyPos * ld;
  const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const T *base = reinterpret_cast<const T *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
  using W = Walk<R, kAnyPos, kAnyThreads>;
  W w;
  w.start(p, 1, red);
  if (tid == 0) p.desc[blockIdx.x].w = 0;
  while (!w.done()) {
    const Segment s = w.next(p);
    const uint32_t *pt = p.pg.page_table + (uint64_t)s.chunk.seq * p.pg.max_pages;
    __syncthreads();
    // Q rows times the scale (log2 domain); rows past the item's are zero
    for (uint32_t i = tid; i < R * hd; i += kAnyThreads) {
      const uint32_t r = i / hd, d = i - r * hd, row = s.r0 + r;
      float x = 0.0f;
      if (row < s.r1)
        x = (float)reinterpret_cast<const T *>(p.q)[(uint64_t)(s.chunk.q0 + row / p.rep) * p.qs +
                                                   (s.head * p.rep + row % p.rep) * hd + d];
      sq[r * ld + d] = x;
    }
    float m[RT], l[RT], o[RT][HJ][4];
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
    for (uint32_t u = s.u0; u < s.u1 && s.hi > s.lo; ++u) {
      const uint32_t t0 = (s.lo / kAnyPos + u) * kAnyPos;
      __syncthreads();
      for (uint32_t i = tid; i < 2 * kAnyPos * (hd / 8); i += kAnyThreads) {
        const uint32_t is_v = i >= kAnyPos * (hd / 8), e = i - is_v * kAnyPos * (hd / 8), r = e / (hd / 8), d = e % (hd / 8) * 8;
        const uint32_t t = t0 + r;
        float x[8] = {};
        if (t >= s.lo && t < s.hi) {
          const uint32_t page = pt[t / kPageLen];
          if (page < p.pg.n_pages) load8(base + page_row(p.pg, page, is_v, s.head, t % kPageLen) + d, x);
          else if (p.err) atomicOr(p.err, kFlagPage);
        }
        float4 *dst = reinterpret_cast<float4 *>((is_v ? sv : sk) + r * ld + d);
        dst[0] = make_float4(x[0], x[1], x[2], x[3]);
        dst[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
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
    const bool whole = W::whole(s);
    float *slot = W::slot(p, s);
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
      const uint32_t r = ty + 8 * i, row = s.r0 + r;
      if (row >= s.r1) continue;
      if (!whole && tx == 0) {
        slot[R * hd + 2 * r] = m[i];
        slot[R * hd + 2 * r + 1] = l[i];
      }
#pragma unroll
      for (uint32_t j = 0; j < HJ; ++j) {
        const uint32_t d = 64 * j + 4 * tx;
        if (d >= hd) continue;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          if (!whole) slot[r * hd + d + e] = o[i][j][e];
          else
            put(reinterpret_cast<T *>(p.out) + (uint64_t)(s.chunk.q0 + row / p.rep) * p.os +
                    (s.head * p.rep + row % p.rep) * hd + d + e,
                l[i] == 0.0f ? 0.0f : o[i][j][e] / l[i]);
        }
      }
    }
    if (!whole && s.u0 == 0 && tid == 0) p.desc[blockIdx.x] = w.describe(s);
  }
  pdl_launch_dependents();
}

// The item that CTA blockIdx.x of the launch before began and others finished.
// A row at a time: warp w adds the pieces w, w + 8, .. in the order of the
// positions (four loads in flight each), then the warps' sums are added in
// order.  With a warp to a whole row the 60 pieces of one long cache were one
// chain of loads: 44 us for 8 kv heads x 4 rows, against 4 us so.
constexpr uint32_t kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) k_attn_join(const AttnChunksParams p, uint32_t R) {
  __shared__ float part[kJoinWarps][kMaxHeadDim];
  __shared__ float wm[kJoinWarps], wl[kJoinWarps];
  pdl_wait();
  const uint4 d = p.desc[blockIdx.x];
  if (!d.w) return;
  const uint32_t hd = p.pg.head_dim, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = d.z & 0xFFFF, rows = d.z >> 16;
  const uint64_t slot = (uint64_t)R * (hd + 2);
  const float *first = p.part + ((uint64_t)blockIdx.x * 2 + 1) * slot;
  // piece i: slot 1 of this CTA, then slot 0 of the next ones
  auto piece = [&](uint32_t i) { return i ? first + (2 * (uint64_t)i - 1) * slot : first; };
  for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y) {
    // running maximum, sum and output of this warp's pieces (a piece's maximum
    // is -inf where its row saw nothing there: weight 0)
    float m = -INFINITY, l = 0.0f, acc[kMaxHeadDim / 32] = {};
    for (uint32_t i0 = warp; i0 < d.w; i0 += 4 * kJoinWarps) {
      float2 ml[4];
      float x[4][kMaxHeadDim / 32];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t i = i0 + k * kJoinWarps;
        ml[k] = make_float2(-INFINITY, 0.0f);
        if (i < d.w) {
          const float *q = piece(i);
          ml[k] = __ldcg(reinterpret_cast<const float2 *>(q + R * hd + 2 * r));
#pragma unroll
          for (uint32_t j = 0; j < kMaxHeadDim / 32; ++j)
            x[k][j] = lane + 32 * j < hd ? __ldcg(q + r * hd + lane + 32 * j) : 0.0f;
        } else {
#pragma unroll
          for (uint32_t j = 0; j < kMaxHeadDim / 32; ++j) x[k][j] = 0.0f;
        }
      }
      const float mn = fmaxf(fmaxf(fmaxf(m, ml[0].x), fmaxf(ml[1].x, ml[2].x)), ml[3].x), ms = mn == -INFINITY ? 0.0f : mn;
      const float f = exp2f(m - ms);
      l *= f;
#pragma unroll
      for (uint32_t j = 0; j < kMaxHeadDim / 32; ++j) acc[j] *= f;
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        const float e = exp2f(ml[k].x - ms);
        l = fmaf(ml[k].y, e, l);
#pragma unroll
        for (uint32_t j = 0; j < kMaxHeadDim / 32; ++j) acc[j] = fmaf(x[k][j], e, acc[j]);
      }
      m = mn;
    }
    __syncthreads();  // the row before has been read
    if (lane == 0) {
      wm[warp] = m;
      wl[warp] = l;
    }
#pragma unroll
    for (uint32_t j = 0; j < kMaxHeadDim / 32; ++j)
      if (lane + 32 * j < hd) part[warp][lane + 32 * j] = acc[j];
    __syncthreads();
    const uint32_t row = d.y + r;
    T *out = reinterpret_cast<T *>(p.out) + (uint64_t)(d.x + row / p.rep) * p.os + (head * p.rep + row % p.rep) * hd;
    float M = wm[0], L = 0.0f, e[kJoinWarps];
#pragma unroll
    for (uint32_t w = 1; w < kJoinWarps; ++w) M = fmaxf(M, wm[w]);
    const float Ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (uint32_t w = 0; w < kJoinWarps; ++w) {
      e[w] = exp2f(wm[w] - Ms);
      L = fmaf(wl[w], e[w], L);
    }
    for (uint32_t x = threadIdx.x; x < hd; x += kJoinWarps * 32) {
      float y = 0.0f;
#pragma unroll
      for (uint32_t w = 0; w < kJoinWarps; ++w) y = fmaf(part[w][x], e[w], y);
      put(out + x, L == 0.0f ? 0.0f : y / L);
    }
  }
}

template <typename T, uint32_t R, uint32_t HJ>
int launch_hj(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st) {
  const uint32_t smem = any_smem(R, p.pg.head_dim);
  if (cudaFuncSetAttribute(k_attn_any<T, R, HJ>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)any_smem(R, 64 * HJ)) !=
      cudaSuccess)
    return -1;
  uint32_t per_sm = 224 * 1024 / (smem + 1024);
  per_sm = per_sm > 3 ? 3 : per_sm;
  const uint32_t grid = n_sm * per_sm < kAttnMaxCtas ? n_sm * per_sm : kAttnMaxCtas;
  k_attn_any<T, R, HJ><<<grid, kAnyThreads, smem, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return -1;
  return launch_attn_join(p, R, grid, st);
}
template <typename T>
int launch_any_t(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st) {
  const uint32_t hd = p.pg.head_dim;
  // items of 8 rows while no chunk has more: a decode's 1 to 8 rows would leave
  // most of 32 idle in the FMA loops
  const bool few = (uint64_t)p.max_q * p.rep <= 8;
  if (hd <= 64) return few ? launch_hj<T, 8, 1>(p, n_sm, st) : launch_hj<T, 32, 1>(p, n_sm, st);
  if (hd <= 128) return few ? launch_hj<T, 8, 2>(p, n_sm, st) : launch_hj<T, 32, 2>(p, n_sm, st);
  return few ? launch_hj<T, 8, 4>(p, n_sm, st) : launch_hj<T, 32, 4>(p, n_sm, st);
}

}  // namespace

int launch_attn_any(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st) {
  switch (p.pg.dtype) {
    case FA_KV_F32: return launch_any_t<float>(p, n_sm, st);
    case FA_KV_F16: return launch_any_t<__half>(p, n_sm, st);
    default: return launch_any_t<__nv_bfloat16>(p, n_sm, st);
  }
}

int launch_attn_join(const AttnChunksParams &p, uint32_t R, uint32_t ctas, cudaStream_t st) {
  const dim3 grid(ctas, R < 8 ? R : 8), block(kJoinWarps * 32);
  switch (p.pg.dtype) {
    case FA_KV_F32: return launch_pdl(k_attn_join<float>, grid, block, 0, st, p, R);
    case FA_KV_F16: return launch_pdl(k_attn_join<__half>, grid, block, 0, st, p, R);
    default: return launch_pdl(k_attn_join<__nv_bfloat16>, grid, block, 0, st, p, R);
  }
}

size_t attn_chunks_ws(uint32_t head_dim) {
  return kAttnMaxCtas * (sizeof(uint4) + (size_t)2 * kAttnMaxRows * (head_dim + 2) * 4);
}

uint32_t attn_max_ctas() { return kAttnMaxCtas; }

int launch_attn_chunks(const AttnChunksParams &p, uint32_t n_sm, cudaStream_t st) {
  AttnChunksParams a = p;
  a.rows_min = 1;
  a.rows_max = 0xFFFFFFFFu;
  if (attn_mma_takes(a)) return launch_attn_mma(a, n_sm, st);
  return launch_attn_any(a, n_sm, st);
}

}  // namespace fa
