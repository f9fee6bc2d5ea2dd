// The plan of a step: which pages the sequences of a step give back and get, where
// its rows are, what the attention and the append of the step are to be given.
//
// With request i keeping k_i of the len positions of its sequence and adding a_i,
// and P(x) = ceil(x / 16) pages of x positions,
//   taken_i  <=>  sum_{j <= i} a_j <= rows  and
//                 sum_{j <= i} max(0, P(k_j + a_j) - P(len_j)) <= free + sum_j max(0, P(len_j) - P(k_j + a_j)),
// so two prefix sums decide, and requests from the first one on that does not fit
// are left out together (their k stays).  A second pass of sums places the pages on
// the stack of free ones.
//
// Latency bounds it: a few words a request and three a row.  One launch of one
// cluster: every CTA forms the sums of all requests (they are few, and stay in shared
// memory), then all threads of the cluster share out the pages that come back, the
// pages that are taken, and the rows, each finding its request by a binary search in
// the sums, so that one long sequence does not keep a warp while the others wait;
// a barrier of the cluster stands where one's writes are another's reads.
// Eight decode requests 6.2 us, 512 requests with 66000 rows 14.4 (a warp to a request's
// pages and a thread to a row, eight CTAs of 512 threads: 28.7).
#include <type_traits>

#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {
namespace {

constexpr uint32_t kCluster = 8;
constexpr uint32_t kNone = FA_NO_TOKEN;

__device__ __forceinline__ uint32_t pages_of(uint32_t positions) { return (positions + kPageLen - 1) / kPageLen; }
// sums that stay at 2^32 - 1 once they reach it: still associative, and above every limit they are compared with
__device__ __forceinline__ uint32_t sat(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < a ? 0xFFFFFFFFu : s;
}

struct Request {
  uint32_t seq, keep, add, have, want;  // pages: have now, want with all of add
  bool ok;
};
__device__ __forceinline__ Request load_request(const StepPlanParams &p, uint32_t i) {
  Request r;
  r.seq = p.seq ? p.seq[i] : i;
  r.add = p.add[i];
  const uint32_t keep = p.keep ? p.keep[i] : 0, most = p.max_pages * kPageLen;
  r.ok = r.seq < p.n_seq;
  const uint32_t len = r.ok ? p.len[r.seq] : 0;
  r.keep = p.keep ? keep : len;
  r.ok = r.ok && len <= most && r.keep <= len && r.add <= most - r.keep;
  r.have = pages_of(len);
  r.want = pages_of(r.keep + r.add);
  return r;
}

// what every CTA keeps of the requests in shared memory
struct Shared {
  uint32_t *start;         // [n + 1] first row (before that: exclusive sums of add)
  uint32_t *gain, *back;   // exclusive sums of the pages that requests take, and give back
  uint32_t *seq;           // their sequences; kNone: left out
  uint32_t *have, *now;    // pages before, length after
  uint32_t *once, *twice;  // a bit a sequence: named, named again
};
// the last i < n with sums[i] <= x
__device__ __forceinline__ uint32_t find(const uint32_t *sums, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// words r0 .. r0 + 3 of an array of n, at once where it is aligned
__device__ __forceinline__ void put4(uint32_t *to, uint32_t r0, uint32_t n, const uint32_t *v) {
  if (reinterpret_cast<uintptr_t>(to) % 16 == 0 && r0 + 4 <= n) {
    *reinterpret_cast<uint4 *>(to + r0) = make_uint4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e)
    if (r0 + e < n) to[r0 + e] = v[e];
}

// inclusive sums over a warp's lanes
template <int N>
__device__ __forceinline__ void scan_lanes(uint32_t (&v)[N]) {
  const uint32_t lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, v[k], o);
      if (lane >= (uint32_t)o) v[k] = sat(v[k], x);
    }
}
// over the CTA's threads, and the totals; scratch of N x kWarps words
template <uint32_t kWarps, int N>
__device__ __forceinline__ void scan(uint32_t (&v)[N], uint32_t (&total)[N], uint32_t (*red)[kWarps]) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  scan_lanes(v);
  __syncthreads();
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < N; ++k) red[k][warp] = v[k];
  __syncthreads();
  uint32_t of[N];  // the warps' totals, summed by every warp
#pragma unroll
  for (int k = 0; k < N; ++k) of[k] = lane < kWarps ? red[k][lane] : 0;
  scan_lanes(of);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    total[k] = __shfl_sync(0xFFFFFFFFu, of[k], kWarps - 1);
    const uint32_t before = __shfl_sync(0xFFFFFFFFu, of[k], (warp + 31) % 32);
    if (warp) v[k] = sat(v[k], before);
  }
}

template <uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) k_step_plan(const StepPlanParams p) {
  constexpr uint32_t kWarps = THREADS / 32;
  extern __shared__ uint32_t words[];
  __shared__ uint32_t red[3][kWarps];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.n, marks = p.seq ? (p.n_seq + 31) / 32 : 0;
  const uint32_t at = cluster_ctarank() * THREADS + tid, all = gridDim.x * THREADS;  // of the cluster's threads
  Shared s;
  s.start = words;
  s.gain = s.start + n + 1;
  s.back = s.gain + n;
  s.seq = s.back + n;
  s.have = s.seq + n;
  s.now = s.have + n;
  s.once = s.now + n;
  s.twice = s.once + marks;
  const uint32_t free0 = *p.n_free;
  uint32_t flags = 0;
  Request mine{};  // request tid
  if (tid < n) mine = load_request(p, tid);
  if (p.seq) {  // a sequence that is named twice is left out both times
    for (uint32_t i = tid; i < 2 * marks; i += THREADS) s.once[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += THREADS) {
      const uint32_t q = i == tid ? mine.seq : p.seq[i], bit = 1u << (q & 31);
      if (q < p.n_seq && (atomicOr(&s.once[q >> 5], bit) & bit)) atomicOr(&s.twice[q >> 5], bit);
    }
    __syncthreads();
  }
  auto request = [&](uint32_t i) {
    Request r{};
    if (i >= n) return r;
    r = i == tid ? mine : load_request(p, i);
    if (p.seq && r.ok && (s.twice[r.seq >> 5] >> (r.seq & 31) & 1)) r.ok = false;
    return r;
  };
  // sums of add and of the pages needed, all given back
  uint32_t rows = 0, need = 0, room = free0;
  for (uint32_t b = 0; b < n; b += THREADS) {
    const uint32_t i = b + tid;
    const Request r = request(i);
    if (i < n && !r.ok) flags |= kFlagRange;
    uint32_t v[3] = {r.ok ? r.add : 0, r.ok && r.want > r.have ? r.want - r.have : 0, r.ok && r.have > r.want ? r.have - r.want : 0}, total[3];
    scan<kWarps>(v, total, red);
    if (i < n) {
      s.start[i] = sat(rows, v[0]);  // inclusive for now
      s.gain[i] = sat(need, v[1]);
    }
    rows = sat(rows, total[0]);
    need = sat(need, total[1]);
    room = sat(room, total[2]);
  }
  // who is taken; where the pages go that come back
  uint32_t freed = 0, T = 0, A = 0;
  for (uint32_t b = 0; b < n; b += THREADS) {
    const uint32_t i = b + tid;
    const Request r = request(i);
    uint32_t end = 0, now = 0;
    bool taken = false;
    if (r.ok) {
      taken = s.start[i] <= p.n_rows && s.gain[i] <= room;
      now = taken ? r.keep + r.add : r.keep;
      end = pages_of(now);
      if (!taken && r.add) flags |= FA_FLAG_FULL;
    }
    uint32_t v[1] = {r.ok && r.have > end ? r.have - end : 0}, total[1];
    const uint32_t own = v[0];
    scan<kWarps>(v, total, red);
    if (i < n) {
      s.back[i] = sat(freed, v[0]) - own;
      s.seq[i] = r.ok ? r.seq : kNone;
      s.have[i] = r.have;
      s.now[i] = now;
      if (taken) {
        T = s.start[i];
        A = s.gain[i];
      }
      // exclusive (a sum that is stuck at its top belongs to a request that is left out)
      s.start[i] -= r.ok ? r.add : 0;
      s.gain[i] -= r.ok && r.want > r.have ? r.want - r.have : 0;
    }
    freed = sat(freed, total[0]);
  }
  // rows and pages of all that are taken: the sums up to the last of them
  T = __reduce_max_sync(0xFFFFFFFFu, T);
  A = __reduce_max_sync(0xFFFFFFFFu, A);
  __syncthreads();
  if (lane == 0) {
    red[0][warp] = T;
    red[1][warp] = A;
  }
  __syncthreads();
  T = __reduce_max_sync(0xFFFFFFFFu, red[0][lane % kWarps]);
  A = __reduce_max_sync(0xFFFFFFFFu, red[1][lane % kWarps]);
  // a stack that is longer than its array, or would be: nothing is done
  const bool bad = free0 > p.free_cap || sat(free0, freed) > p.free_cap;
  if (bad) {
    flags |= kFlagRange;
    T = A = freed = 0;
  }
  for (uint32_t i = tid; i < n; i += THREADS) {
    s.start[i] = min(s.start[i], T);
    if (bad) s.seq[i] = kNone;
  }
  if (tid == 0) s.start[n] = T;
  __syncthreads();
  const uint32_t top = free0 + freed;
  for (uint32_t f = at; f < freed; f += all) {
    const uint32_t i = find(s.back, n, f);
    const uint32_t page = p.table[(uint64_t)s.seq[i] * p.max_pages + pages_of(s.now[i]) + (f - s.back[i])];
    if (page >= p.n_pages) flags |= kFlagPage;
    p.free_pages[free0 + f] = page;
  }
  // all CTAs have read the lengths and the stack's height, which may be written in place, and the stack is complete
  cluster_sync();
  for (uint32_t k = at; k < A; k += all) {
    const uint32_t i = find(s.gain, n, k);
    const uint32_t page = __ldcg(p.free_pages + (top - 1 - k));
    if (page >= p.n_pages) flags |= kFlagPage;
    p.table[(uint64_t)s.seq[i] * p.max_pages + s.have[i] + (k - s.gain[i])] = page;
  }
  for (uint32_t i = at; i < n; i += all) {
    const uint32_t q = s.seq[i], a = s.start[i], b = s.start[i + 1];
    p.q_start[i] = a;
    p.kv_len[i] = q != kNone ? s.now[i] : 0;
    if (p.last) p.last[i] = b > a ? b - 1 : kNone;
    if (q != kNone) {
      p.len_out[q] = s.now[i];
    } else if (p.len_out != p.len) {  // left out: its sequence keeps its length (all that name it write the same)
      const uint32_t named = p.seq ? p.seq[i] : i;
      if (named < p.n_seq) p.len_out[named] = p.len[named];
    }
  }
  if (at == 0) {
    p.q_start[n] = T;
    *p.n_free_out = top - A;
  }
  if (p.slot) cluster_sync();  // the table is complete
  // Rows, four or eight in a row a thread: one search in the sums, then all their looks at the table at once
  // (one where a page begins, each waited for, took twice as long).
  auto put_rows = [&](auto count) {
    constexpr uint32_t N = decltype(count)::value;
    for (uint32_t r0 = N * at; r0 < p.n_rows; r0 += N * all) {
      uint32_t pos[N], q[N], slot[N], i = r0 < T ? find(s.start, n, r0) : 0, end = r0 < T ? s.start[i + 1] : 0;
#pragma unroll
      for (uint32_t e = 0; e < N; ++e) {
        const uint32_t r = r0 + e;
        pos[e] = 0;
        q[e] = slot[e] = kNone;
        if (r < T) {
          while (end <= r) end = s.start[++i + 1];
          pos[e] = s.now[i] - (end - r);
          q[e] = s.seq[i];
        }
      }
      if (p.slot) {
#pragma unroll
        for (uint32_t e = 0; e < N; ++e)
          if (r0 + e < T) slot[e] = __ldcg(p.table + (uint64_t)q[e] * p.max_pages + pos[e] / kPageLen);
#pragma unroll
        for (uint32_t e = 0; e < N; ++e)
          if (r0 + e < T) slot[e] = slot[e] * kPageLen + pos[e] % kPageLen;
      }
#pragma unroll
      for (uint32_t e = 0; e < N; e += 4) {
        put4(p.pos, r0 + e, p.n_rows, pos + e);
        put4(p.row_seq, r0 + e, p.n_rows, q + e);
        if (p.slot) put4(p.slot, r0 + e, p.n_rows, slot + e);
      }
    }
  };
  if (p.n_rows <= 4 * all) put_rows(std::integral_constant<uint32_t, 4>());
  else put_rows(std::integral_constant<uint32_t, 8>());
  if (flags && p.err && (at < THREADS || (flags & kFlagPage))) atomicOr(p.err, flags);
}

template <uint32_t THREADS>
int launch(const StepPlanParams &p, uint32_t ctas, cudaStream_t st) {
  if (cudaFuncSetAttribute(k_step_plan<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanMaxSmem) != cudaSuccess) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = 4 * ((size_t)6 * p.n + 1 + (p.seq ? 2 * ((p.n_seq + 31) / 32) : 0));
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_step_plan<THREADS>, p) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_step_plan(const StepPlanParams &p, cudaStream_t st) {
  static_assert(4 * (6 * kPlanMaxRequests + 1 + 2 * (kPlanMaxSeqs / 32)) <= kPlanMaxSmem, "shared memory of the largest call");
  // few rows and requests: one small CTA, whose barriers are cheaper
  return p.n_rows <= 512 && p.n <= 128 ? launch<128>(p, 1, st) : launch<1024>(p, kCluster, st);
}

}  // namespace fa
