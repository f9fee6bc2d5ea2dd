// Rotary positions of q and k with the append of k and v to the pages
// (src/tensor.rs:331-392 turns, src/kv_cache.rs:50-54 appends):
//   (a, b) -> m (a cos x - b sin x, a sin x + b cos x),  x = pos f_i
//
// One pass: every element of q, k, v is read once and written once, so HBM
// bounds it for many tokens and the launch for few.  A CTA takes one token
// and a group of its heads.  It forms the token's rot / 2 sines and cosines
// once in shared memory, from the position in turns: pos * (f_i / 2 pi) in 64
// bits (exact to 2^-53 of the turn count), its fraction in [-1/2, 1/2] in 32
// bits, sincospi of that.  In 32 bits the product alone would be wrong by
// 2^-24 * pos radians, 0.06 at position 10^6.  Then each thread turns or
// copies units of 4 pairs or 8 elements.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};
// N consecutive elements; V: in one access (the address is a multiple of its size)
template <bool V, int N, typename T>
__device__ __forceinline__ void load_n(const T *p, float (&x)[N]) {
  if constexpr (V) {
    const Vec<T, N> w = *reinterpret_cast<const Vec<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f(w.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f(p[i]);
  }
}
template <bool V, int N, typename T>
__device__ __forceinline__ void store_n(T *p, const float (&x)[N]) {
  if constexpr (V) {
    Vec<T, N> w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.v[i] = from_f<T>(x[i]);
    *reinterpret_cast<Vec<T, N> *>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f<T>(x[i]);
  }
}

// W: pairs of a unit (4: every address a unit touches is aligned to 4 elements;
// 1: any).  A head is hd / (2 W) units: the first rot / (2 W) turn W pairs,
// the others copy 2 W elements.
template <typename TI, typename TO, int W>
__global__ void __launch_bounds__(256) k_rope_append(const RopeAppendParams p, const __grid_constant__ RopeTable tab) {
  __shared__ float cs[kMaxHeadDim / 2], sn[kMaxHeadDim / 2];
  const uint32_t t = blockIdx.x, hd = p.pg.head_dim, half = p.rot / 2, H = p.n_heads, KVH = p.pg.n_kv_heads;
  const uint32_t seq = p.seq[t], pos = p.pos[t], slot = p.slot ? p.slot[t] : pos;
  if (seq == FA_NO_TOKEN) return;
  uint32_t bad = 0, page = 0;
  if (seq >= p.pg.n_seq || slot / kPageLen >= p.pg.max_pages) bad = kFlagRange;
  else if ((page = p.pg.page_table[(uint64_t)seq * p.pg.max_pages + slot / kPageLen]) >= p.pg.n_pages) bad = kFlagPage;
  if (bad) {
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, bad);
    return;
  }
  for (uint32_t i = threadIdx.x; i < half; i += blockDim.x) {
    const double x = (double)pos * tab.turns[i];
    float s, c;
    sincospif(2.0f * (float)(x - rint(x)), &s, &c);
    cs[i] = c * tab.scale;
    sn[i] = s * tab.scale;
  }
  __syncthreads();
  constexpr bool V = W == 4;
  const uint32_t upr = half / W, uph = hd / (2 * W);
  const uint32_t n_units = (H + 2 * KVH) * uph;
  TO *base = reinterpret_cast<TO *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride;
  for (uint32_t u = blockIdx.y * blockDim.x + threadIdx.x; u < n_units; u += gridDim.y * blockDim.x) {
    const uint32_t head = u / uph, w = u - head * uph;
    const TI *src;
    TO *dst;
    const bool is_v = head >= H + KVH;
    if (head < H) {
      src = reinterpret_cast<const TI *>(p.q) + t * p.qs + head * hd;
      dst = reinterpret_cast<TO *>(p.out) + t * p.os + head * hd;
    } else {
      const uint32_t h = head - H - (is_v ? KVH : 0);
      src = is_v ? reinterpret_cast<const TI *>(p.v) + t * p.vs + h * hd
                 : reinterpret_cast<const TI *>(p.k) + t * p.ks + h * hd;
      dst = base + ((((uint64_t)page * 2 + is_v) * KVH + h) * kPageLen + slot % kPageLen) * hd;
    }
    float a[W], b[W];
    const bool turn = !is_v && w < upr;
    // offsets of the unit's two halves: pairs (a[j], b[j]) of the half layout,
    // else 2 W consecutive elements
    const uint32_t o0 = turn && p.half_layout ? w * W : w * 2 * W;
    const uint32_t o1 = turn && p.half_layout ? half + w * W : w * 2 * W + W;
    load_n<V>(src + o0, a);
    load_n<V>(src + o1, b);
    if (turn) {
      if (p.half_layout) {
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const float c = cs[w * W + j], s = sn[w * W + j], x = a[j], y = b[j];
          a[j] = x * c - y * s;
          b[j] = x * s + y * c;
        }
      } else {
        float e[2 * W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
          e[j] = a[j];
          e[W + j] = b[j];
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const float c = cs[w * W + j], s = sn[w * W + j], x = e[2 * j], y = e[2 * j + 1];
          e[2 * j] = x * c - y * s;
          e[2 * j + 1] = x * s + y * c;
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
          a[j] = e[j];
          b[j] = e[W + j];
        }
      }
    }
    store_n<V>(dst + o0, a);
    store_n<V>(dst + o1, b);
  }
}

template <typename TI, typename TO>
int launch_io(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st) {
  const uint32_t esi = sizeof(TI), eso = sizeof(TO), half = p.rot / 2;
  auto al = [](const void *q, uint64_t stride, uint32_t es) {
    return reinterpret_cast<uintptr_t>(q) % (4 * es) == 0 && stride % 4 == 0;
  };
  // four pairs a unit where every unit starts on a multiple of four elements
  const bool wide = half % 4 == 0 && al(p.q, p.qs, esi) && al(p.k, p.ks, esi) && al(p.v, p.vs, esi) &&
                    al(p.out, p.os, eso);
  const uint32_t units = (p.n_heads + 2 * p.pg.n_kv_heads) * (p.pg.head_dim / (wide ? 8 : 2));
  const uint32_t parts = (units + 255) / 256;
  // few tokens: one unit a thread, the heads spread over more CTAs; many: a CTA
  // a token, whose angles then serve all heads
  const dim3 grid(p.n_tokens, p.n_tokens >= 512 ? 1 : (parts < 64 ? parts : 64));
  if (wide) k_rope_append<TI, TO, 4><<<grid, 256, 0, st>>>(p, t);
  else k_rope_append<TI, TO, 1><<<grid, 256, 0, st>>>(p, t);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}
template <typename TI>
int launch_in(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st) {
  switch (p.pg.dtype) {
    case FA_KV_F32: return launch_io<TI, float>(p, t, st);
    case FA_KV_F16: return launch_io<TI, __half>(p, t, st);
    default: return launch_io<TI, __nv_bfloat16>(p, t, st);
  }
}

}  // namespace

int launch_rope_append(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st) {
  switch (p.in_dtype) {
    case FA_KV_F32: return launch_in<float>(p, t, st);
    case FA_KV_F16: return launch_in<__half>(p, t, st);
    default: return launch_in<__nv_bfloat16>(p, t, st);
  }
}

}  // namespace fa
