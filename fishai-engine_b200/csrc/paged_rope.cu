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
// copies a unit of up to 8 pairs or 16 elements.  With several axes (images and
// video) a pair's position is that of its axis; all else is the same.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>

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

// N consecutive elements; V: in one access (the address is a multiple of its size)
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};
template <bool V, int N, typename T>
__device__ __forceinline__ Vec<T, N> load_n(const T *p) {
  Vec<T, N> w;
  if constexpr (V) w = *reinterpret_cast<const Vec<T, N> *>(p);
  else
#pragma unroll
    for (int i = 0; i < N; ++i) w.v[i] = p[i];
  return w;
}
template <bool V, int N, typename T>
__device__ __forceinline__ void store_n(T *p, const float (&x)[N]) {
  Vec<T, N> w;
#pragma unroll
  for (int i = 0; i < N; ++i) w.v[i] = from_f<T>(x[i]);
  if constexpr (V) *reinterpret_cast<Vec<T, N> *>(p) = w;
  else
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = w.v[i];
}

// 16-bit elements two at a time, from and to a 32-bit word
__device__ __forceinline__ float2 unpack(const __half *p, uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float2 unpack(const __nv_bfloat16 *p, uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ uint32_t pack(const __half *p, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack(const __nv_bfloat16 *p, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// W: pairs of a unit (8 or 4: every address a unit touches is aligned to W
// elements; 1: any).  A head is hd / (2 W) units: the first rot / (2 W) turn W
// pairs, the others copy 2 W elements.  A CTA takes `each` tokens (up to 4) and
// as many units as it has threads: it forms all their angles at once, with one
// barrier, while each thread's first unit is already on its way; then the next
// token's is always in flight while one is turned and stored.  (A CTA a token,
// loading after its angles: 46 us for 8192 tokens of 48 heads.)
constexpr uint32_t kRopeTokens = 4;
template <typename TI, typename TO, int W, bool AXES, int HALF>
__global__ void __launch_bounds__(512, 3) k_rope_append(const RopeAppendParams p, const __grid_constant__ RopeTable tab, uint32_t each) {
  __shared__ __align__(16) float cs[kRopeTokens][kMaxHeadDim / 2], sn[kRopeTokens][kMaxHeadDim / 2];
  __shared__ uint64_t place[kRopeTokens];  // element offset of the token's slot in a (K, head 0) block
  const uint32_t hd = p.pg.head_dim, half = p.rot / 2, H = p.n_heads, KVH = p.pg.n_kv_heads;
  constexpr bool V = W > 1;
  constexpr uint64_t kSkip = ~0ull;
  const uint32_t t0 = blockIdx.x * each, nt = min(each, p.n_tokens - t0);
  const uint32_t upr = half / W, uph = hd / (2 * W), n_units = (H + 2 * KVH) * uph;
  const uint32_t u = blockIdx.y * blockDim.x + threadIdx.x;
  const bool live = u < n_units;
  const uint32_t head = u / uph, w = u - head * uph;
  const bool turn = head < H + KVH && w < upr, is_q = head < H, is_v = head >= H + KVH;
  // offsets of the unit's two parts: pairs of the half layout, else 2 W
  // consecutive elements, or (16-bit types) W in each half of the head, so that
  // the accesses of neighbours adjoin
  constexpr bool kWords = W == 8 && sizeof(TI) == 2 && sizeof(TO) == 2;
  const bool in_halves = HALF < 0 ? p.half_layout : HALF, spread = kWords && (is_v || !in_halves);
  const uint32_t o0 = (turn && in_halves) || spread ? w * W : w * 2 * W;
  const uint32_t o1 = spread ? hd / 2 + w * W : turn && in_halves ? half + w * W : w * 2 * W + W;
  const uint64_t ss = is_q ? p.qs : is_v ? p.vs : p.ks;
  const TI *src = reinterpret_cast<const TI *>(is_q ? p.q : is_v ? p.v : p.k) + t0 * ss + (head - (is_q ? 0 : is_v ? H + KVH : H)) * hd;
  Vec<TI, W> a0{}, a1{};
  if (live) {
    a0 = load_n<V, W>(src + o0);
    a1 = load_n<V, W>(src + o1);
  }
  if (threadIdx.x < nt) {
    const uint32_t t = t0 + threadIdx.x, seq = p.seq[t], slot = p.slot ? p.slot[t] : p.pos[t];
    uint64_t at = kSkip;
    if (seq != FA_NO_TOKEN) {
      uint32_t bad = 0, page = 0;
      if (seq >= p.pg.n_seq || slot / kPageLen >= p.pg.max_pages) bad = kFlagRange;
      else if ((page = p.pg.page_table[(uint64_t)seq * p.pg.max_pages + slot / kPageLen]) >= p.pg.n_pages) bad = kFlagPage;
      else at = ((uint64_t)page * 2 * KVH * kPageLen + slot % kPageLen) * hd;
      if (bad && p.err) atomicOr(p.err, bad);
    }
    place[threadIdx.x] = at;
  }
  for (uint32_t i = threadIdx.x; i < nt * half; i += blockDim.x) {
    const uint32_t k = i / half, j = i - k * half;
    const double a = (double)p.pos[t0 + k + (AXES ? tab.axis[j] * p.pos_stride : 0)] * tab.turns[j];
    float s, c;
    sincospif(2.0f * (float)(a - rint(a)), &s, &c);
    // half layout in 16-bit types: units 4 to 7 find their angles' two pieces swapped, and the eight units of a head
    // read from 32 banks (8192 tokens: 42.7 us unswapped, 41.2 so)
    const uint32_t at = HALF == 1 ? j ^ (j >> 3 & 4) : j;
    cs[k][at] = c * tab.scale;
    sn[k][at] = s * tab.scale;
  }
  __syncthreads();
  if (!live) return;
  TO *out = is_q ? reinterpret_cast<TO *>(p.out) + t0 * p.os + head * hd
                 : reinterpret_cast<TO *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride +
                       (uint64_t)(head - H) * kPageLen * hd;  // K heads, then V heads of a page
  if constexpr (kWords) {
    // word by word, and at most 42 registers: more threads hold loads on their way (8192 tokens of 48 heads x
    // 128: 39 us interleaved, 41 halves with three axes; all 16 elements as f32 at once in 61 registers 49 and 51; in
    // 32 registers 49; all four tokens' pieces to shared memory by cp.async at the start 51 and 41; CTAs that stay
    // and go through 14 tokens one after another 58 and 60.  Interleaved in accesses to every other 16 bytes, as
    // two pieces that adjoin would be: 44.  A copy of as many bytes takes 34.)
    const TI *ti = nullptr;
    const TO *to = nullptr;
    for (uint32_t k = 0; k < nt; ++k) {
      uint32_t r[2][4], o[2][4];
      memcpy(r[0], &a0, 16);
      memcpy(r[1], &a1, 16);
      if (k + 1 < nt) {
        src += ss;
        a0 = load_n<V, W>(src + o0);
        a1 = load_n<V, W>(src + o1);
      }
      if (HALF == 1 && turn) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {  // elements of two pairs in a word of each part
          const float4 c = *reinterpret_cast<const float4 *>(&cs[k][(w * W + 4 * h) ^ (w & 4)]), s = *reinterpret_cast<const float4 *>(&sn[k][(w * W + 4 * h) ^ (w & 4)]);
          const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (uint32_t i = 0; i < 2; ++i) {
            const float2 va = unpack(ti, r[0][2 * h + i]), vb = unpack(ti, r[1][2 * h + i]);
            o[0][2 * h + i] = pack(to, va.x * cv[2 * i] - vb.x * sv[2 * i], va.y * cv[2 * i + 1] - vb.y * sv[2 * i + 1]);
            o[1][2 * h + i] = pack(to, va.x * sv[2 * i] + vb.x * cv[2 * i], va.y * sv[2 * i + 1] + vb.y * cv[2 * i + 1]);
          }
        }
      } else {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          const uint32_t e = h ? o1 : o0;
          if (!HALF && !is_v && e < p.rot) {  // a pair in a word
            const float4 c = *reinterpret_cast<const float4 *>(&cs[k][e / 2]), s = *reinterpret_cast<const float4 *>(&sn[k][e / 2]);
            const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
              const float2 v = unpack(ti, r[h][i]);
              o[h][i] = pack(to, v.x * cv[i] - v.y * sv[i], v.x * sv[i] + v.y * cv[i]);
            }
          } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
              const float2 v = unpack(ti, r[h][i]);
              o[h][i] = __is_same(TI, TO) ? r[h][i] : pack(to, v.x, v.y);
            }
          }
        }
      }
      const uint64_t at = place[k];
      TO *dst = is_q ? out : out + at;
      if (at != kSkip) {
        *reinterpret_cast<uint4 *>(dst + o0) = make_uint4(o[0][0], o[0][1], o[0][2], o[0][3]);
        *reinterpret_cast<uint4 *>(dst + o1) = make_uint4(o[1][0], o[1][1], o[1][2], o[1][3]);
      }
      if (is_q) out += p.os;
    }
    return;
  }
  for (uint32_t k = 0; k < nt; ++k) {
    float x[2][W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      x[0][j] = to_f(a0.v[j]);
      x[1][j] = to_f(a1.v[j]);
    }
    if (k + 1 < nt) {
      src += ss;
      a0 = load_n<V, W>(src + o0);
      a1 = load_n<V, W>(src + o1);
    }
    if (turn) {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float c = cs[k][w * W + j], s = sn[k][w * W + j];
        if (p.half_layout) {
          const float va = x[0][j], vb = x[1][j];
          x[0][j] = va * c - vb * s;
          x[1][j] = va * s + vb * c;
        } else {
          const int i = 2 * j;
          const float va = x[i / W][i % W], vb = x[(i + 1) / W][(i + 1) % W];
          x[i / W][i % W] = va * c - vb * s;
          x[(i + 1) / W][(i + 1) % W] = va * s + vb * c;
        }
      }
    }
    const uint64_t at = place[k];
    TO *dst = is_q ? out : out + at;
    if (at != kSkip) {
      store_n<V>(dst + o0, x[0]);
      store_n<V>(dst + o1, x[1]);
    }
    if (is_q) out += p.os;
  }
}

template <typename TI, typename TO, bool AXES>
int launch_io(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st) {
  const uint32_t half = p.rot / 2, hd = p.pg.head_dim;
  // every unit starts on a multiple of n elements of every buffer (pages: hd is
  // a multiple of 8 and their base is aligned)
  auto fits = [&](uint32_t n) {
    auto al = [&](const void *q, uint64_t stride, size_t es) {
      return reinterpret_cast<uintptr_t>(q) % (n * es) == 0 && stride % n == 0;
    };
    return half % n == 0 && hd % (2 * n) == 0 && al(p.q, p.qs, sizeof(TI)) && al(p.k, p.ks, sizeof(TI)) &&
           al(p.v, p.vs, sizeof(TI)) && al(p.out, p.os, sizeof(TO));
  };
  const uint32_t W = sizeof(TI) == 2 && sizeof(TO) == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;  // accesses of up to 16 bytes
  const uint32_t units = (p.n_heads + 2 * p.pg.n_kv_heads) * (hd / (2 * W));
  // few tokens: small CTAs, the heads spread over the SMs; many: up to four
  // tokens a CTA as long as two CTAs an SM remain, one CTA for all heads where it
  // can be (2000 tokens: 20.8 us with one token a CTA, 17.0 with four; 8192: 43
  // with four, 51 with two, 45 with eight)
  const uint32_t each = p.n_tokens < 600 ? 1 : p.n_tokens < 1200 ? 2 : kRopeTokens;
  uint32_t block = p.n_tokens < 296 ? 128 : (units + 31) / 32 * 32;
  if (block > 512) block = (units / ((units + 511) / 512) + 31) / 32 * 32;
  if ((units + block - 1) / block > 65535) block = 512;  // grid y (thousands of heads)
  const dim3 grid((p.n_tokens + each - 1) / each, (units + block - 1) / block);
  if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) {
    if (W == 8 && p.half_layout) k_rope_append<TI, TO, 8, AXES, 1><<<grid, block, 0, st>>>(p, t, each);
    if (W == 8 && !p.half_layout) k_rope_append<TI, TO, 8, AXES, 0><<<grid, block, 0, st>>>(p, t, each);
  }
  if (W == 4) k_rope_append<TI, TO, 4, AXES, -1><<<grid, block, 0, st>>>(p, t, each);
  if (W == 1) k_rope_append<TI, TO, 1, AXES, -1><<<grid, block, 0, st>>>(p, t, each);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}
template <typename TI, bool AXES>
int launch_in(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st) {
  switch (p.pg.dtype) {
    case FA_KV_F32: return launch_io<TI, float, AXES>(p, t, st);
    case FA_KV_F16: return launch_io<TI, __half, AXES>(p, t, st);
    default: return launch_io<TI, __nv_bfloat16, AXES>(p, t, st);
  }
}

template <bool AXES>
int launch_axes(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st) {
  switch (p.in_dtype) {
    case FA_KV_F32: return launch_in<float, AXES>(p, t, st);
    case FA_KV_F16: return launch_in<__half, AXES>(p, t, st);
    default: return launch_in<__nv_bfloat16, AXES>(p, t, st);
  }
}

}  // namespace

int launch_rope_append(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st) {
  return p.pos_stride ? launch_axes<true>(p, t, st) : launch_axes<false>(p, t, st);
}

}  // namespace fa
