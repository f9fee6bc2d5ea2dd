// Beam search selection: the k best of score_b + x_bv - log sum_v exp(x_bv)
// over the beams b and tokens v of each request, equal scores by lowest (b, v).
//
// The logits are read once and bound it by HBM when there are many rows, by
// latency when there are few, so a row is split over CTAs until they fill the
// GPU.  k_beam_scan: each CTA keeps, over its range of one row, a running
// (max, sum of exp) per thread and the k best (value, token) of the range.
// Within a row the score grows with the logit, so the best of a row need no
// log-sum-exp.  k_beam_pick: one CTA per request joins the ranges' sums in 64
// bits and picks the k best of beams x ranges x k candidates.
//
// The candidates of a tile of 4096 logits: a thread's largest value that does
// not beat the range's k-th best so far ends the matter for its 16 elements,
// and a tile in which nothing does is passed by.  Else the k-th largest of the
// 256 threads' largest bounds the tile's k-th best from below; what reaches the
// bound (at most 16 k elements) is ranked against the list by counting.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {
namespace {

constexpr uint32_t kScanThreads = 256, kScanElems = 16, kTile = kScanThreads * kScanElems;
constexpr uint32_t kPickThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;

// (ordered value, lower token first) as one number; 0: no candidate
__device__ __forceinline__ unsigned long long cand_key(float x, uint32_t token) {
  return ((unsigned long long)float_key(x) << 32) | (uint32_t)~token;
}

template <typename T>
__device__ __forceinline__ float logit(T x) {
  const float f = (float)x;
  return f == f ? fminf(f, FLT_MAX) : -INFINITY;  // NaN: no candidate; +inf: the largest f32
}

// 16 logits of a thread: four groups of four, group j at (j * 256 + tid) * 4
template <typename T, bool VEC>
__device__ __forceinline__ void load_tile(const T *row, uint32_t v0, uint32_t end, float (&x)[kScanElems]) {
  struct alignas(4 * sizeof(T)) T4 {
    T e[4];
  };
  T4 raw[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint32_t v = v0 + (j * kScanThreads + threadIdx.x) * 4;
    if (VEC && v + 4 <= end) {
      raw[j] = *reinterpret_cast<const T4 *>(row + v);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) raw[j].e[e] = v + e < end ? row[v + e] : (T)(-INFINITY);
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) x[4 * j + e] = logit(raw[j].e[e]);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kScanThreads) k_beam_scan(const BeamParams p) {
  pdl_launch_dependents();
  __shared__ unsigned long long list[2][kBeamMaxK], tops[kScanThreads], buf[kScanElems * kBeamMaxK + kBeamMaxK];
  __shared__ uint32_t n_buf;
  __shared__ unsigned long long bound;
  __shared__ float wm[kScanThreads / 32], wsum[kScanThreads / 32];
  const uint32_t row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, K = p.k;
  if (!isfinite(p.scores[row]) || (p.done && p.done[row])) return;
  const uint32_t begin = split * p.per, end = min(p.vocab, begin + p.per);
  const T *x_row = reinterpret_cast<const T *>(p.logits) + row * p.ld;
  for (uint32_t i = tid; i < K; i += kScanThreads) list[0][i] = 0;
  if (tid == 0) n_buf = 0;
  uint32_t cur = 0;
  float m = -INFINITY, s = 0.0f;
  __syncthreads();
  for (uint32_t v0 = begin; v0 < end; v0 += kTile) {
    float x[kScanElems];
    load_tile<T, VEC>(x_row, v0, end, x);
    float t = x[0];
#pragma unroll
    for (uint32_t i = 1; i < kScanElems; ++i) t = fmaxf(t, x[i]);
    if (t != -INFINITY) {
      if (t > m) {
        s *= exp2f((m - t) * kLog2e);
        m = t;
      }
#pragma unroll
      for (uint32_t i = 0; i < kScanElems; ++i) s += exp2f((x[i] - m) * kLog2e);
    }
    // the thread's best element (the lowest token among equals)
    unsigned long long best = 0;
    const unsigned long long kth = list[cur][K - 1];
    if (t != -INFINITY && float_key(t) > (uint32_t)(kth >> 32)) {  // a later equal token does not beat the list's
#pragma unroll
      for (int i = kScanElems - 1; i >= 0; --i)
        if (x[i] == t) best = cand_key(t, v0 + (i / 4 * kScanThreads + tid) * 4 + i % 4);
    }
    if (!__syncthreads_or(best != 0)) continue;
    tops[tid] = best;
    __syncthreads();
    uint32_t above = 0;
    for (uint32_t i = 0; i < kScanThreads; ++i) above += tops[i] > best;
    if (best && above == K - 1) bound = best;
    const uint32_t n_tops = __syncthreads_count(best != 0);
    const unsigned long long low = n_tops >= K ? bound : 1;
    if (best >= low && best) {
#pragma unroll
      for (uint32_t i = 0; i < kScanElems; ++i) {
        const unsigned long long c =
            x[i] == -INFINITY ? 0 : cand_key(x[i], v0 + (i / 4 * kScanThreads + tid) * 4 + i % 4);
        if (c >= low && c > kth) buf[atomicAdd(&n_buf, 1u)] = c;
      }
    }
    __syncthreads();
    // the list and the tile's candidates, ranked by counting (all keys differ)
    const uint32_t n = n_buf;
    if (tid < K && list[cur][tid]) buf[n + tid] = list[cur][tid];
    __shared__ uint32_t n_old;
    if (tid == 0) n_old = 0;
    __syncthreads();
    if (tid < K && list[cur][tid] && (tid + 1 == K || !list[cur][tid + 1])) n_old = tid + 1;
    if (tid < K) list[cur ^ 1][tid] = 0;
    __syncthreads();
    const uint32_t all = n + n_old;
    for (uint32_t i = tid; i < all; i += kScanThreads) {
      const unsigned long long c = buf[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < all; ++j) rank += buf[j] > c;
      if (rank < K) list[cur ^ 1][rank] = c;
    }
    __syncthreads();
    cur ^= 1;
    if (tid == 0) n_buf = 0;
    __syncthreads();
  }
  // the range's (max, sum), warps then lanes in a fixed order
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, o), s2 = __shfl_xor_sync(0xFFFFFFFFu, s, o), mm = fmaxf(m, m2);
    if (mm != -INFINITY) s = s * exp2f((m - mm) * kLog2e) + s2 * exp2f((m2 - mm) * kLog2e);
    m = mm;
  }
  if (tid % 32 == 0) {
    wm[tid / 32] = m;
    wsum[tid / 32] = s;
  }
  __syncthreads();
  if (tid == 0) {
    float M = -INFINITY, S = 0.0f;
    for (uint32_t w = 0; w < kScanThreads / 32; ++w) M = fmaxf(M, wm[w]);
    if (M != -INFINITY)
      for (uint32_t w = 0; w < kScanThreads / 32; ++w) S += wsum[w] * exp2f((wm[w] - M) * kLog2e);
    p.stats[row * p.splits + split] = make_float2(M, S);
  }
  for (uint32_t i = tid; i < K; i += kScanThreads) {
    const unsigned long long c = list[cur][i];
    p.cand[((uint64_t)row * p.splits + split) * K + i] = make_uint2((uint32_t)(c >> 32), ~(uint32_t)c);
  }
}

// A candidate: an ordered score, then the lowest beam, the largest logit and the
// lowest token; hi 0: none.  (Scores of one beam order as its logits do, also
// where 64 bits no longer tell them apart, as beside a logit of 10^38.)
struct Best {
  unsigned long long hi, mid;  // mid: ~beam, ordered logit
  uint32_t lo;                 // ~token
};
__device__ __forceinline__ bool better(const Best &a, const Best &b) {
  return a.hi != b.hi ? a.hi > b.hi : a.mid != b.mid ? a.mid > b.mid : a.lo > b.lo;
}
__device__ __forceinline__ unsigned long long double_key(double f) {
  const unsigned long long b = __double_as_longlong(f);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_double(unsigned long long k) {
  return __longlong_as_double((k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k);
}

__global__ void __launch_bounds__(kPickThreads) k_beam_pick(const BeamParams p) {
  pdl_wait();
  __shared__ double base[kBeamMaxBeams], lse[kBeamMaxBeams];  // score, log sum exp
  __shared__ uint32_t kind[kBeamMaxBeams];                    // 0 out, 1 open, 2 done
  __shared__ Best wbest[kPickThreads / 32];
  __shared__ uint32_t wthread[kPickThreads / 32];
  __shared__ Best won[kBeamMaxK];
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, NB = p.n_beams, K = p.k;
  for (uint32_t j = warp; j < NB; j += kPickThreads / 32) {
    const uint32_t row = b * NB + j;
    const float sc = p.scores[row];
    const uint32_t kd = !isfinite(sc) ? 0 : (p.done && p.done[row]) ? 2 : 1;
    if (kd == 1) {
      const float2 st = lane < p.splits ? p.stats[row * p.splits + lane] : make_float2(-INFINITY, 0.0f);
      float M = st.x;
#pragma unroll
      for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
      double S = st.x == -INFINITY ? 0.0 : (double)st.y * exp((double)st.x - (double)M);
#pragma unroll
      for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(0xFFFFFFFFu, S, o);
      if (lane == 0) lse[j] = (double)M + log(S);
    }
    if (lane == 0) {
      base[j] = sc;
      kind[j] = kd;
    }
  }
  __syncthreads();
  const uint32_t each = p.splits * K, N = NB * each;
  const uint2 *cand = p.cand + (uint64_t)b * N;
  // candidate i of the request; a done beam's only one stands in its first place
  auto get = [&](uint32_t i) -> Best {
    const uint32_t j = i / each;
    if (kind[j] == 1) {
      const uint2 c = cand[i];
      if (!c.x) return {0, 0, 0};
      return {double_key(base[j] + ((double)key_float(c.x) - lse[j])), (unsigned long long)~j << 32 | c.x, ~c.y};
    }
    if (kind[j] == 2 && i == j * each) return {double_key(base[j]), (unsigned long long)~j << 32, ~p.pad};
    return {0, 0, 0};
  };
  // k rounds: the best of the threads' own best; the winner looks for its next
  auto scan = [&](const Best &below) -> Best {
    Best r{0, 0, 0};
    for (uint32_t i = tid; i < N; i += kPickThreads) {
      const Best c = get(i);
      if (better(below, c) && better(c, r)) r = c;
    }
    return r;
  };
  Best mine = scan(Best{~0ull, ~0ull, ~0u});
  for (uint32_t r = 0; r < K; ++r) {
    Best w = mine;
    uint32_t who = tid;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      Best x;
      x.hi = __shfl_xor_sync(0xFFFFFFFFu, w.hi, o);
      x.mid = __shfl_xor_sync(0xFFFFFFFFu, w.mid, o);
      x.lo = __shfl_xor_sync(0xFFFFFFFFu, w.lo, o);
      const uint32_t xw = __shfl_xor_sync(0xFFFFFFFFu, who, o);
      if (better(x, w)) {
        w = x;
        who = xw;
      }
    }
    if (lane == 0) {
      wbest[warp] = w;
      wthread[warp] = who;
    }
    __syncthreads();
    w = wbest[0];
    who = wthread[0];
#pragma unroll
    for (uint32_t i = 1; i < kPickThreads / 32; ++i)
      if (better(wbest[i], w)) {
        w = wbest[i];
        who = wthread[i];
      }
    if (tid == 0) won[r] = w;
    if (w.hi == 0) {  // nothing is left: the same for every thread
      if (tid == 0)
        for (uint32_t i = r; i < K; ++i) won[i] = Best{0, 0, 0};
      break;
    }
    if (tid == who) mine = scan(w);
    __syncthreads();
  }
  __syncthreads();
  for (uint32_t r = tid; r < K; r += kPickThreads) {
    const Best w = won[r];
    const bool some = w.hi != 0;
    const uint32_t parent = some ? ~(uint32_t)(w.mid >> 32) : r % NB, token = some ? ~w.lo : p.pad;
    const uint64_t o = (uint64_t)b * K + r;
    p.out_scores[o] = some ? (float)key_double(w.hi) : -INFINITY;
    p.out_parents[o] = parent;
    p.out_tokens[o] = token;
    if (p.out_done) p.out_done[o] = !some || kind[parent] == 2 || token == p.eos;
  }
}

template <typename T>
int launch_t(const BeamParams &p, cudaStream_t st) {
  const uint32_t rows = p.n_batch * p.n_beams;
  const bool vec = reinterpret_cast<uintptr_t>(p.logits) % (4 * sizeof(T)) == 0 && p.ld % 4 == 0;
  for (uint32_t r0 = 0; r0 < rows; r0 += 65535) {  // grid y ends at 65535
    BeamParams q = p;
    q.logits = reinterpret_cast<const T *>(p.logits) + r0 * p.ld;
    q.scores += r0;
    if (q.done) q.done += r0;
    q.stats += (uint64_t)r0 * p.splits;
    q.cand += (uint64_t)r0 * p.splits * p.k;
    const dim3 grid(p.splits, rows - r0 < 65535 ? rows - r0 : 65535);
    if (vec) k_beam_scan<T, true><<<grid, kScanThreads, 0, st>>>(q);
    else k_beam_scan<T, false><<<grid, kScanThreads, 0, st>>>(q);
    if (cudaGetLastError() != cudaSuccess) return -1;
  }
  return launch_pdl(k_beam_pick, dim3(p.n_batch), dim3(kPickThreads), 0, st, p);
}

}  // namespace

// Ranges of a row: enough CTAs to fill the GPU twice over, none smaller than a
// tile.
uint32_t beam_splits(uint32_t rows, uint32_t vocab, uint32_t *per) {
  const uint32_t tiles = (vocab + kTile - 1) / kTile;
  uint32_t want = rows ? (4 * 148 + rows - 1) / rows : 1;
  if (want > kBeamMaxSplits) want = kBeamMaxSplits;
  if (want > tiles) want = tiles;
  if (!want) want = 1;
  const uint32_t each = (tiles + want - 1) / want;
  *per = each * kTile;
  return (tiles + each - 1) / each;
}

int launch_beam_select(const BeamParams &p, cudaStream_t st) {
  switch (p.dtype) {
    case FA_KV_F32: return launch_t<float>(p, st);
    case FA_KV_F16: return launch_t<__half>(p, st);
    default: return launch_t<__nv_bfloat16>(p, st);
  }
}

}  // namespace fa
