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
// The sum of a range is f32, so that an exponential is one instruction: the scan
// is bound by its instructions.  With e = 2^-24: an exponential is good to 4 e and
// its argument to 3 e times its distance d from the maximum, which over a row's
// weights costs 3 e ln(vocab) at most (their mean d is below their entropy); a
// tile's 16 add 9 e, each tile of a thread 5 e (the sum, and a factor where the
// maximum moves), the warp's, the CTA's and the ranges' joins 48 e.  In all less than
// (128 + vocab / 512) e in the log, which only the order of different beams feels
// (measured over rows of 100 to 10^6 normal logits: 2.5e-7 at most).
//
// Candidates of a range: what beats the k-th best of the list so far goes to a
// buffer, and the list is made anew, by counting ranks, after the first tile of
// 4096 logits and then after groups of 1, 2, 4, .. tiles: in random order each
// group has about k candidates.  Within a group nothing waits for other warps; a
// group that fills the buffer (rows that rise) is gone through once more, tile by
// tile.  256 rows of 128256 f32, k = 8: 31 us, of which the stream of logits is 24
// (5.4 TB/s), the first tile, the lists and the pick the rest; bf16 35, k = 64 62.
// (A barrier a tile, a list whenever the buffer might overflow and a pick in k
// rounds: 41, 63 and 111.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {
namespace {

constexpr uint32_t kScanThreads = 256, kScanElems = 16, kTile = kScanThreads * kScanElems;
constexpr uint32_t kBuf = kScanElems * kBeamMaxK;  // candidates of a tile
constexpr uint32_t kPickThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// A value's place in the order; + 0 makes +0.0 of -0.0: the two are equal, here
// as in the comparisons and maxima that the bounds below are taken with.
__device__ __forceinline__ uint32_t value_key(float x) { return float_key(x + 0.0f); }
// (ordered value, lower token first) as one number; 0: no candidate
__device__ __forceinline__ unsigned long long cand_key(float x, uint32_t token) {
  return ((unsigned long long)value_key(x) << 32) | (uint32_t)~token;
}

__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two f32 in a register pair
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 16 logits of a thread as they are stored: four groups of four, group j at
// (j * 256 + tid) * 4; past the end: -inf
template <typename T>
struct Raw {
  struct alignas(4 * sizeof(T)) T4 {
    T e[4];
  } g[4];
};
template <typename T>
__device__ __forceinline__ void load_tile(const T *row, uint32_t v0, uint32_t end, Raw<T> &raw) {
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint32_t v = v0 + (j * kScanThreads + threadIdx.x) * 4;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) raw.g[j].e[e] = v + e < end ? row[v + e] : (T)(-INFINITY);
  }
}

// The same to a slot of shared memory, by cp.async where rows are aligned to four
// elements; a thread reads only what it copied, so its own wait is all it needs.
template <typename T>
__device__ __forceinline__ void stage_tile(const T *row, uint32_t v0, uint32_t end, Raw<T> *slot) {
  using T4 = typename Raw<T>::T4;
  T4 *to = reinterpret_cast<T4 *>(slot) + threadIdx.x;
  const T *from = row + v0 + threadIdx.x * 4;
  auto copy = [&](uint32_t j) {
    if constexpr (sizeof(T) == 4)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to + j * kScanThreads)), "l"(from + j * kScanThreads * 4) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(to + j * kScanThreads)), "l"(from + j * kScanThreads * 4) : "memory");
  };
  if (v0 + kTile <= end) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) copy(j);
  } else if (v0 < end) {
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t v = v0 + (j * kScanThreads + threadIdx.x) * 4;
      if (v + 4 <= end) {
        copy(j);
        continue;
      }
      T4 x;
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) x.e[e] = v + e < end ? row[v + e] : (T)(-INFINITY);
      to[j * kScanThreads] = x;
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kScanThreads, 4) k_beam_scan(const BeamParams p) {
  pdl_launch_dependents();
  __shared__ __align__(16) unsigned long long tops[kScanThreads];
  __shared__ unsigned long long list[2][kBeamMaxK];
  __shared__ __align__(16) unsigned long long buf[kBuf + kBeamMaxK + 2];
  __shared__ uint32_t n_buf, n_list;
  __shared__ unsigned long long bound;
  __shared__ float wm[kScanThreads / 32], wsum[kScanThreads / 32];
  const uint32_t row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, K = p.k;
  const uint32_t begin = split * p.per, end = min(p.vocab, begin + p.per);
  const T *x_row = reinterpret_cast<const T *>(p.logits) + row * p.ld;
  const bool open = isfinite(p.scores[row]) && !(p.done && p.done[row]);
  // the next tile, on its way over the work on one (two of them: 38 -> 41 us for
  // 256 rows of 128256)
  __shared__ __align__(16) Raw<T> slot[VEC ? kScanThreads : 1];
  Raw<T> ahead;
  if (open) {
    if constexpr (VEC) stage_tile(x_row, begin, end, slot);
    else load_tile(x_row, begin, end, ahead);
  }
  for (uint32_t i = tid; i < K; i += kScanThreads) list[0][i] = 0;
  if (tid == 0) n_buf = n_list = 0;
  if (!open) return;
  uint32_t cur = 0;
  float m = -INFINITY, s = 0.0f, kv = -INFINITY;  // kv: the list's k-th value
  __syncthreads();
  // The list and the buffer, ranked by counting (all keys differ), become the
  // list; the buffer is empty after it.  Starts with the buffer complete.
  auto flush = [&] {
    const uint32_t n = n_buf, n_old = n_list, all = n + n_old;
    if (tid < n_old) buf[n + tid] = list[cur][tid];
    if (tid >= 64 && tid < 64 + K) list[cur ^ 1][tid - 64] = 0;
    if (tid == 128) buf[all] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < all; i += kScanThreads) {
      const unsigned long long c = buf[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < all; j += 2) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(buf + j);
        rank += (o.x > c) + (o.y > c);
      }
      if (rank < K) list[cur ^ 1][rank] = c;
    }
    if (tid == 0) {
      n_buf = 0;
      n_list = min(all, K);
    }
    __syncthreads();
    cur ^= 1;
    const unsigned long long kth = list[cur][K - 1];
    kv = kth ? key_float((uint32_t)(kth >> 32)) : -INFINITY;
  };
  float x[kScanElems], t;  // a tile's values of the thread, and their largest
  auto largest = [&] {
    t = x[0];
#pragma unroll
    for (uint32_t i = 1; i + 1 < kScanElems; i += 2) t = fmaxf(t, fmaxf(x[i], x[i + 1]));
    t = fmaxf(t, x[kScanElems - 1]);
  };
  auto clean = [&] {
#pragma unroll
    for (uint32_t i = 0; i < kScanElems; ++i) x[i] = x[i] == x[i] ? fminf(x[i], FLT_MAX) : -INFINITY;
  };
  auto take = [&](const Raw<T> &raw) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) x[4 * j + e] = (float)raw.g[j].e[e];
  };
  // the next tile to x and t, and into (m, s); the one behind it on its way
  auto next = [&](uint32_t v0) {
    if constexpr (VEC) {
      asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) ahead.g[j] = reinterpret_cast<const typename Raw<T>::T4 *>(slot)[j * kScanThreads + tid];
      take(ahead);
      stage_tile(x_row, v0 + kTile, end, slot);
    } else {
      take(ahead);
      if (v0 + kTile < end) load_tile(x_row, v0 + kTile, end, ahead);
    }
    float add;
    for (;;) {  // a second time where there is a NaN or +inf among the 16
      largest();
      const float r = t == -INFINITY ? 0.0f : t;
      const uint64_t less = pair(-r, -r), l2e = pair(kLog2e, kLog2e);
      uint64_t a = 0;
#pragma unroll
      for (uint32_t i = 0; i < kScanElems; i += 2) {
        float u, w;
        unpair(mul2(add2(pair(x[i], x[i + 1]), less), l2e), u, w);
        a = add2(a, pair(ex2(u), ex2(w)));
      }
      float a0, a1;
      unpair(a, a0, a1);
      add = a0 + a1;
      if (add == add) break;  // +inf - +inf is NaN too
      clean();
    }
    if (t > m) {
      s = fmaf(s, ex2((m - t) * kLog2e), add);
      m = t;
    } else if (t != -INFINITY) {
      s = fmaf(add, ex2((t - m) * kLog2e), s);
    }
  };
  // what beats the list goes to the buffer (a later token of an equal value does
  // not beat it), as far as it has room
  auto append = [&](uint32_t v0, unsigned long long low) {
    if (t > kv) {
#pragma unroll
      for (uint32_t i = 0; i < kScanElems; ++i)
        if (x[i] > kv) {
          const unsigned long long c = cand_key(x[i], v0 + (i / 4 * kScanThreads + tid) * 4 + i % 4);
          if (c < low) continue;
          const uint32_t to = atomicAdd(&n_buf, 1u);
          if (to < kBuf) buf[to] = c;
        }
    }
  };
  // a tile by itself, however many of its values beat the list; starts and ends
  // with an empty buffer
  auto choose = [&](uint32_t v0) {
    const uint32_t n_tops = __syncthreads_count(t > kv);
    if (!n_tops) return;
    const bool many = n_tops * kScanElems > kBuf;  // the first tile, rising rows
    for (bool exact = many && K > kScanThreads / 32;; exact = true) {
      unsigned long long low = 1;
      if (exact) {
        // the k-th largest of the threads' largest, which at most 16 k elements reach
        unsigned long long best = 0;
        if (t > kv) {
#pragma unroll
          for (int i = kScanElems - 1; i >= 0; --i)
            if (x[i] == t) best = cand_key(t, v0 + (i / 4 * kScanThreads + tid) * 4 + i % 4);
        }
        tops[tid] = best;
        if (tid == 0) n_buf = 0;
        __syncthreads();
        uint32_t above = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < kScanThreads; i += 2) {
          const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(tops + i);
          above += (o.x > best) + (o.y > best);
        }
        if (best && above == K - 1) bound = best;  // n_tops > 64 >= K: one thread's
        __syncthreads();
        low = bound;
      } else if (many) {
        // the least of the warps' largest, which 8 elements reach
        float g = t;
#pragma unroll
        for (uint32_t o = 16; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
        if (tid % 32 == 0) tops[tid / 32] = value_key(g);
        __syncthreads();
        unsigned long long v = tops[0];
#pragma unroll
        for (uint32_t i = 1; i < kScanThreads / 32; ++i) v = min(v, tops[i]);
        low = max(v << 32, 1ull);
      }
      append(v0, low);
      __syncthreads();
      if (exact || n_buf <= kBuf) break;
      __syncthreads();  // still too many
    }
    flush();
  };
  next(begin);
  choose(begin);
  uint32_t group = 1;
  for (uint32_t v0 = begin + kTile; v0 < end; v0 += group * kTile, group *= 2) {
    const uint32_t g_end = min(end, v0 + group * kTile);
    bool some = false;
    for (uint32_t v = v0; v < g_end; v += kTile) {
      next(v);
      some = some || t > kv;
      append(v, 1);
    }
    if (!__syncthreads_count(some)) continue;
    if (n_buf <= kBuf) {
      flush();
      continue;
    }
    // more than the buffer holds: the group again, tile by tile
    __syncthreads();
    if (tid == 0) n_buf = 0;
    for (uint32_t v = v0; v < g_end; v += kTile) {
      Raw<T> raw;
      load_tile(x_row, v, g_end, raw);
      take(raw);
      clean();
      largest();
      choose(v);
    }
  }
  // the range's (max, sum), warps then lanes in a fixed order
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, o), s2 = __shfl_xor_sync(0xFFFFFFFFu, s, o), mm = fmaxf(m, m2);
    if (mm != -INFINITY) s = s * ex2((m - mm) * kLog2e) + s2 * ex2((m2 - mm) * kLog2e);
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
      for (uint32_t w = 0; w < kScanThreads / 32; ++w) S += wsum[w] * ex2((wm[w] - M) * kLog2e);
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
  const unsigned long long b = __double_as_longlong(f + 0.0);  // zeros of both signs are equal
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_double(unsigned long long k) {
  return __longlong_as_double((k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k);
}

// The lane of the warp's best candidate.  Field by field (scores differ in
// their first 32 bits almost always): a maximum and a ballot each.
__device__ __forceinline__ uint32_t best_lane(const Best &x) {
  const uint32_t f[5] = {(uint32_t)(x.hi >> 32), (uint32_t)x.hi, (uint32_t)(x.mid >> 32), (uint32_t)x.mid, x.lo};
  uint32_t in = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const bool mine = (in >> (threadIdx.x & 31)) & 1;
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, mine ? f[i] : 0u);
    in = __ballot_sync(0xFFFFFFFFu, mine && f[i] == top);
    if (!(in & (in - 1))) break;  // the same for the whole warp
  }
  return __ffs(in) - 1;
}

// The ranges' lists stand in descending order.  Of the threads' best candidates
// (each thread has some of the lists' first ones, or of all) the k-th is a bound
// that at least k candidates reach; what reaches it, from each list's beginning,
// goes to shared memory, and a candidate's place is the number of better ones.
// (k rounds of the best of the threads' best, each followed by a scan: 1 x 12
// beams, k = 16: 161 us, 19 so; 1 x 64, k = 64: 2.9 ms, 50 so.)
constexpr uint32_t kPlaced = 1024;  // candidates that are placed by counting; in random order some 2 k reach the bound
template <bool MANY>  // more candidates than threads
__global__ void __launch_bounds__(kPickThreads) k_beam_pick(const BeamParams p) {
  constexpr uint32_t kWarps = kPickThreads / 32, kHold = MANY ? 8 : 1, kRoom = MANY ? kPlaced : kPickThreads;
  __shared__ double base[kBeamMaxBeams], lse[kBeamMaxBeams];  // score, log sum exp
  __shared__ uint32_t kind[kBeamMaxBeams];                    // 0 out, 1 open, 2 done
  __shared__ __align__(16) unsigned long long hi[kRoom + 2];
  __shared__ unsigned long long mid[kRoom];
  __shared__ uint32_t lo[kRoom];
  __shared__ uint32_t bound, n_placed, n_reach;
  __shared__ __align__(16) uint32_t tops[MANY ? kPickThreads : 1];
  __shared__ uint16_t reach[MANY ? kBeamMaxBeams * kBeamMaxSplits : 1];  // lists
  __shared__ Best wbest[2][kWarps];
  __shared__ uint32_t wthread[2][kWarps];
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, NB = p.n_beams, K = p.k;
  // the inputs, which the scan does not write: before it ends
  for (uint32_t j = tid; j < NB; j += kPickThreads) {
    const float sc = p.scores[b * NB + j];
    const uint32_t dn = p.done ? p.done[b * NB + j] : 0;
    base[j] = sc;
    kind[j] = !isfinite(sc) ? 0 : dn ? 2 : 1;
  }
  const uint32_t each = p.splits * K, N = NB * each, lists = NB * p.splits;
  const uint2 *cand = p.cand + (uint64_t)b * N;
  pdl_wait();
  // the thread's candidates tid, tid + 256, ..; the first ones of lists where
  // there are enough of them (2048 at most)
  const bool heads = MANY && lists >= kPickThreads;
  const uint32_t step = heads ? K : 1, have = heads ? lists : N;
  uint2 raw[kHold];
#pragma unroll
  for (uint32_t h = 0; h < kHold; ++h) {
    const uint32_t i = tid + h * kPickThreads;
    raw[h] = i < have ? __ldcg(cand + i * step) : make_uint2(0, 0);  // of a beam that is not open: not used
  }
  for (uint32_t j = warp; j < NB; j += kWarps) {
    const float2 st = lane < p.splits ? __ldcg(p.stats + (b * NB + j) * p.splits + lane) : make_float2(-INFINITY, 0.0f);
    float M = st.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
    double S = M == -INFINITY ? 0.0 : (double)(st.y * ex2((st.x - M) * kLog2e));
#pragma unroll
    for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(0xFFFFFFFFu, S, o);
    if (lane == 0) lse[j] = (double)M + log(S);
  }
  if (tid == 0) n_placed = n_reach = 0;
  __syncthreads();
  // candidate i of the request; a done beam's only one stands in its first place
  auto make = [&](uint32_t i, const uint2 &c) -> Best {
    const uint32_t j = i / each;
    if (kind[j] == 1) {
      if (!c.x) return {0, 0, 0};
      return {double_key(base[j] + ((double)key_float(c.x) - lse[j])), (unsigned long long)~j << 32 | c.x, ~c.y};
    }
    if (kind[j] == 2 && i == j * each) return {double_key(base[j]), (unsigned long long)~j << 32, ~p.pad};
    return {0, 0, 0};
  };
  auto write = [&](uint32_t r, const Best &w) {
    const bool some = w.hi != 0;
    const uint32_t parent = some ? ~(uint32_t)(w.mid >> 32) : r % NB, token = some ? ~w.lo : p.pad;
    const uint64_t o = (uint64_t)b * K + r;
    p.out_scores[o] = some ? (float)key_double(w.hi) : -INFINITY;
    p.out_parents[o] = parent;
    p.out_tokens[o] = token;
    if (p.out_done) p.out_done[o] = !some || kind[parent] == 2 || token == p.eos;
  };
  auto keep = [&](uint32_t at, const Best &c) {
    hi[at] = c.hi;
    mid[at] = c.mid;
    lo[at] = c.lo;
  };
  // Candidate `at` of the first n (0 in hi[n]) by the number of better ones
  auto place = [&](uint32_t at, uint32_t n) {
    const Best c{hi[at], mid[at], lo[at]};
    uint32_t r = 0, same = 0;
    for (uint32_t j = 0; j < n; j += 2) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(hi + j);
      r += (x.x > c.hi) + (x.y > c.hi);
      same += (x.x == c.hi) + (x.y == c.hi);
    }
    if (same > 1)
      for (uint32_t j = 0; j < n; ++j) r += hi[j] == c.hi && (mid[j] > c.mid || (mid[j] == c.mid && lo[j] > c.lo));
    if (r < K) write(r, c);
  };
  if constexpr (!MANY) {  // all of them, a thread each
    const Best c = tid < N ? make(tid, raw[0]) : Best{0, 0, 0};
    keep(tid, c);
    if (tid < 2) hi[kPickThreads + tid] = 0;
    const uint32_t some = __syncthreads_count(c.hi != 0);
    if (c.hi) place(tid, N);
    if (tid >= some && tid < K) write(tid, Best{0, 0, 0});
    return;
  }
  // the scores' first 32 bits do for the bound
  uint32_t top = 0;
#pragma unroll
  for (uint32_t h = 0; h < kHold; ++h) {
    const uint32_t i = tid + h * kPickThreads;
    if (i < have) top = max(top, (uint32_t)(make(i * step, raw[h]).hi >> 32));
  }
  for (uint32_t i = tid + kHold * kPickThreads; i < have; i += kPickThreads) top = max(top, (uint32_t)(make(i, __ldcg(cand + i)).hi >> 32));
  tops[tid] = top;
  __syncthreads();
  uint32_t above = 0;
#pragma unroll 4
  for (uint32_t j = 0; j < kPickThreads; j += 4) {
    const uint4 x = *reinterpret_cast<const uint4 *>(tops + j);
    above += (x.x > top || (x.x == top && j < tid)) + (x.y > top || (x.y == top && j + 1 < tid)) + (x.z > top || (x.z == top && j + 2 < tid)) +
             (x.w > top || (x.w == top && j + 3 < tid));
  }
  if (above == K - 1) bound = top;  // one thread's
  __syncthreads();
  const uint32_t low = max(bound, 1u);  // of a candidate it is never 0
  auto gather = [&](uint32_t i, const uint2 &c) {
    const Best x = make(i, c);
    if ((uint32_t)(x.hi >> 32) < low) return;
    const uint32_t at = atomicAdd(&n_placed, 1u);
    if (at < kPlaced) keep(at, x);
  };
#pragma unroll
  for (uint32_t h = 0; h < kHold; ++h) {
    const uint32_t i = tid + h * kPickThreads;
    if (i >= have) continue;
    if (!heads) gather(i, raw[h]);
    else if ((uint32_t)(make(i * step, raw[h]).hi >> 32) >= low) reach[atomicAdd(&n_reach, 1u)] = i;
  }
  for (uint32_t i = tid + kHold * kPickThreads; i < have; i += kPickThreads) gather(i, __ldcg(cand + i));
  if (heads) {  // the lists whose first one reaches it
    __syncthreads();
    for (uint32_t i = tid; i < n_reach * K; i += kPickThreads) {
      const uint32_t at = reach[i / K] * K + i % K;
      gather(at, __ldcg(cand + at));
    }
  }
  __syncthreads();
  const uint32_t found = n_placed;
  if (found <= kPlaced) {
    if (tid < 2) hi[found + tid] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < found; i += kPickThreads) place(i, found);
    for (uint32_t r = found + tid; r < K; r += kPickThreads) write(r, Best{0, 0, 0});
    return;
  }
  // More (equal scores, or most of the best in few ranges): k rounds, the best of
  // the threads' own best; the winner looks for its next
  auto scan = [&](const Best &below) -> Best {
    Best r{0, 0, 0};
#pragma unroll 4
    for (uint32_t i = tid; i < N; i += kPickThreads) {
      const Best c = make(i, __ldcg(cand + i));
      if (better(below, c) && better(c, r)) r = c;
    }
    return r;
  };
  Best mine = scan(Best{~0ull, ~0ull, ~0u});
  for (uint32_t r = 0; r < K; ++r) {  // found > k: every round has a winner
    const uint32_t buf = r & 1;
    uint32_t l = best_lane(mine);
    if (lane == l) {
      wbest[buf][warp] = mine;
      wthread[buf][warp] = tid;
    }
    __syncthreads();
    const Best w = lane < kWarps ? wbest[buf][lane] : Best{0, 0, 0};
    l = best_lane(w);
    const Best best = wbest[buf][l];
    if (tid == 0) write(r, best);
    if (tid == wthread[buf][l]) mine = scan(best);
  }
}

// How a kernel's SMs split their memory.  Before k_beam_pick<true>, which has 27 KB
// of shared memory, the scan takes the same split, or the pick's CTAs wait for
// the SMs to empty: 4 x 8 beams 24.4 us, 18.6 so.  Else its own: 32 x 8 beams 31.2
// us, and 34.2 with the smaller L1.
template <typename K>
bool split_memory(K kern, bool shared) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                              shared ? cudaSharedmemCarveoutMaxShared : cudaSharedmemCarveoutDefault) == cudaSuccess;
}
template <typename T>
int launch_t(const BeamParams &p, cudaStream_t st) {
  const uint32_t rows = p.n_batch * p.n_beams;
  const bool vec = reinterpret_cast<uintptr_t>(p.logits) % (4 * sizeof(T)) == 0 && p.ld % 4 == 0;
  const bool many = p.n_beams * p.splits * p.k > kPickThreads;
  if (!(vec ? split_memory(k_beam_scan<T, true>, many) : split_memory(k_beam_scan<T, false>, many))) return -1;
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
  if (!many) return launch_pdl(k_beam_pick<false>, dim3(p.n_batch), dim3(kPickThreads), 0, st, p);
  if (!split_memory(k_beam_pick<true>, true)) return -1;
  return launch_pdl(k_beam_pick<true>, dim3(p.n_batch), dim3(kPickThreads), 0, st, p);
}

}  // namespace

// Ranges of a row: as many CTAs as the GPU holds at once (four an SM), none
// smaller than a tile.  (One more range a row than that, for 256 rows, ran a
// second wave of a third of the SMs: 75 us.)
uint32_t beam_splits(uint32_t rows, uint32_t vocab, uint32_t *per) {
  const uint32_t tiles = (vocab + kTile - 1) / kTile;
  uint32_t want = rows ? 4 * 148 / rows : 1;
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
