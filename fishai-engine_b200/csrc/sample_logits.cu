// Draws a token from each row of logits, with cuts of the row's own:
//   w_v = 2^(-z_v),  z_v = (max x - x_v) log2(e) / T       (0 where z_v > 64)
//   order: x descending, equal ones by id;  top-k: the first k;
//   top-p: the shortest beginning of those whose mass is at least p of theirs;
//   min-p: those with w >= min_p;
//   the token: the first by id at which the mass of the kept ones exceeds u times all of it.
// Every cut keeps a beginning of the same order, so a row's cuts are one place in it.
//
// Each row is read once: a cluster of up to eight CTAs holds it in shared memory (in
// f32) and exchanges sums over distributed shared memory.  A thread owns consecutive
// ids, an odd number of them, so that the lanes' reads fall on distinct banks and a
// prefix sum over threads is one over ids.  Masses are 64-bit sums of 64-bit
// exponentials in a fixed order: which token is drawn from a flat row of 10^5 tokens
// depends on 17 bits more than f32 has.
//
// A cut's place is found without sorting the row: a histogram over z in 1/16 octave
// (of counts, or of masses to 2^-15, which bracket the place), then the few elements of the
// bins around it, which CTA 0 sorts.  Where few elements in all are above the place (top-k
// and top-p as they mostly are), they are all in that list and the rest happens there; where
// more are in the bracket than the list holds (flat rows, equal logits), its range of values is
// halved until it holds them, or one value is left and the place is an id.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {
namespace {

constexpr uint32_t kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kList = 1024, kMaxCtas = 8;
constexpr float kOctaves = 64.0f, kPerOctave = kBins / kOctaves;
constexpr double kHistError = 1.0 / 32768;  // of a prefix of the histogram's masses: each is rounded to 2^-15 of its bin's largest, and 2^-21 in exponentials

struct Msg {  // what a CTA tells the others
  double a, b;
  uint32_t c, d, e, f;
};
struct Small {
  Msg msg[2][kMaxCtas];
  double red[kWarps];
  uint32_t redu[4][kWarps];
  uint32_t bin, count;
  double before;
};

__device__ __forceinline__ float to_logit(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f) + 0.0f; }  // -0 to +0

template <typename T>
struct alignas(16) Vec {
  T v[16 / sizeof(T)];
};

__device__ __forceinline__ void st_cluster(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint64_t ld_cluster64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_cluster32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// A cluster's work on one row.
struct Row {
  const SampleParams &p;
  Small &s;
  float *x;         // this CTA's part of the row
  uint32_t *hist;   // [kBins], or over it
  uint64_t *list;   // [kList] (ordered value, ~id)
  uint32_t tid, lane, warp, rank, ctas, n_own, first;  // first: the thread's first element; n_own: how many it has
  uint32_t id0;     // id of the CTA's first element
  uint32_t turn = 0;
  float mx, cf;     // the maximum, log2(e) / T
  double mxd, cd;
  // kept so far: value above the key, or equal and id at most cut_id
  uint32_t cut_key = 0, cut_id = 0xFFFFFFFFu;

  __device__ Row(const SampleParams &p, Small &s) : p(p), s(s) {}

  __device__ float z(float v) const { return (mx - v) * cf; }
  __device__ double weight(float v) const { return exp2(((double)v - mxd) * cd); }
  __device__ bool kept(float v, uint32_t id) const {
    const uint32_t k = float_key(v);
    return z(v) <= kOctaves && (k > cut_key || (k == cut_key && id <= cut_id));
  }
  // f(value, id) of the thread's elements that are kept, in the order of ids
  template <typename F>
  __device__ void each(F f) const {
    for (uint32_t j = 0; j < n_own; ++j) {
      const float v = x[first + j];
      const uint32_t id = id0 + first + j;
      if (kept(v, id)) f(v, id);
    }
  }

  // what every CTA says, from thread 0's m; valid until the call after the next
  __device__ const Msg *share(const Msg &m) {
    const uint32_t t = turn;
    turn ^= 1;
    if (tid == 0) s.msg[t][rank] = m;
    __syncthreads();
    if (tid < 4 * ctas && tid / 4 != rank) {
      const uint64_t *w = reinterpret_cast<const uint64_t *>(&s.msg[t][rank]) + tid % 4;
      st_cluster(dsmem_addr(w, tid / 4), *w);
    }
    cluster_sync();
    return s.msg[t];
  }
  // sums over the CTA, the same for all threads
  __device__ double sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if (lane == 0) s.red[warp] = v;
    __syncthreads();
    double t = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) t += s.red[w];
    return t;
  }
  // (sum of a, sum of b, smallest of c, largest of d)
  __device__ void sums(uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) {
    a = __reduce_add_sync(0xFFFFFFFFu, a);
    b = __reduce_add_sync(0xFFFFFFFFu, b);
    c = __reduce_min_sync(0xFFFFFFFFu, c);
    d = __reduce_max_sync(0xFFFFFFFFu, d);
    __syncthreads();
    if (lane == 0) {
      s.redu[0][warp] = a;
      s.redu[1][warp] = b;
      s.redu[2][warp] = c;
      s.redu[3][warp] = d;
    }
    __syncthreads();
    a = b = d = 0;
    c = 0xFFFFFFFFu;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      a += s.redu[0][w];
      b += s.redu[1][w];
      c = min(c, s.redu[2][w]);
      d = max(d, s.redu[3][w]);
    }
  }
  // inclusive sum over the CTA's threads, and the total
  __device__ double scan(double v, double &total) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= (uint32_t)o) v += y;
    }
    __syncthreads();
    if (lane == 31) s.red[warp] = v;
    __syncthreads();
    double before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w == warp) before = total;
      total += s.red[w];
    }
    return before + v;
  }

  // The histogram over the kept elements: of counts, or of masses, where elements
  // above z_most only count for the whole mass, which is returned (0 for counts).
  template <bool MASS>
  __device__ double fill(float z_most) {
    for (uint32_t i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    double w = 0;
    uint32_t bin = 0, n = 0;  // elements of one bin in a row are added at once
    each([&](float v, uint32_t) {
      const float zv = z(v);
      if (MASS) w += weight(v);
      if (MASS && zv > z_most) return;
      const uint32_t b = min((uint32_t)(zv * kPerOctave), kBins - 1);
      if (b != bin) {
        if (n) atomicAdd(hist + bin, n);
        bin = b;
        n = 0;
      }
      n += MASS ? __float2uint_rn(exp2f((float)b * (1.0f / kPerOctave) - zv) * 32768.0f) : 1u;
    });
    if (n) atomicAdd(hist + bin, n);
    return MASS ? sum(w) : 0.0;
  }
  // The cluster's sums over bins: hist becomes, in CTA r, the inclusive sums (f64) of its share of the bins.
  template <bool MASS>
  __device__ double reduce_bins() {
    const uint32_t nb = kBins / ctas, per = nb > kThreads ? 2 : 1;
    double v[2] = {0, 0};
    cluster_sync();
    for (uint32_t j = 0; j < per; ++j) {
      const uint32_t b = rank * nb + tid * per + j;
      if (tid * per + j >= nb) continue;
      uint64_t t = 0;
      for (uint32_t r = 0; r < ctas; ++r) t += ld_cluster32(dsmem_addr(hist + b, r));
      v[j] = MASS ? (double)t * exp2(-(double)b / kPerOctave - 15.0) : (double)t;
    }
    double total;
    const double in = scan(v[0] + v[1], total);
    cluster_sync();  // all have read their shares of all CTAs' bins
    double *sums = reinterpret_cast<double *>(hist);
    for (uint32_t j = 0; j < per; ++j)
      if (tid * per + j < nb) sums[tid * per + j] = j + 1 == per ? in : in - v[1];
    return total;
  }
  // the first bin whose inclusive sum reaches `target` (the last bin where none does)
  __device__ uint32_t find_bin(const Msg *all, double target) {
    const uint32_t nb = kBins / ctas;
    double before = 0;
    uint32_t r = 0;
    while (r + 1 < ctas && before + all[r].a < target) before += all[r++].a;
    if (tid == 0) s.bin = nb - 1;
    __syncthreads();
    const double *sums = reinterpret_cast<const double *>(hist);
    for (uint32_t i = tid; i < nb; i += kThreads)
      if (before + __longlong_as_double((long long)ld_cluster64(dsmem_addr(sums + i, r))) >= target) atomicMin(&s.bin, i);
    __syncthreads();
    const uint32_t b = r * nb + s.bin;
    __syncthreads();
    return b;
  }
  __device__ void note(uint32_t key, uint32_t id) {
    const uint32_t at = atomicAdd(&s.count, 1u);
    if (at < kList) list[at] = (uint64_t)key << 32 | (uint32_t)~id;
  }
  // sorts list[0 .. n) in descending order, n a power of two
  __device__ void sort(uint32_t n) {
    for (uint32_t k = 2; k <= n; k <<= 1)
      for (uint32_t j = k >> 1; j; j >>= 1) {
        __syncthreads();
        if (tid < n / 2) {
          const uint32_t i = (tid / j) * 2 * j + tid % j;
          const uint64_t a = list[i], b = list[i + j];
          if ((a < b) == ((i & k) == 0)) {
            list[i] = b;
            list[i + j] = a;
          }
        }
      }
    __syncthreads();
  }
  // CTA 0 brings all CTAs' lists together in its own, sorted; true there.  After it
  // no CTA reads another's memory.
  __device__ bool gather(const Msg *all, uint32_t &n) {
    uint64_t mine[2] = {0, 0};
    n = 0;
    for (uint32_t r = 0; r < ctas; ++r) n += all[r].c;
    if (rank == 0)
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e) {
        uint32_t i = tid + e * kThreads;
        if (i >= n) continue;
        uint32_t r = 0;
        while (i >= all[r].c) i -= all[r++].c;
        mine[e] = ld_cluster64(dsmem_addr(list + i, r));
      }
    cluster_sync();
    if (rank) return false;
    list[tid] = mine[0];
    list[tid + kThreads] = mine[1];
    uint32_t n2 = 2;
    while (n2 < n) n2 <<= 1;
    sort(n2);
    return true;
  }
  __device__ double list_weight(uint64_t e) const { return e ? weight(key_float((uint32_t)(e >> 32))) : 0.0; }

  __device__ void answer(uint32_t row, uint32_t id, double prob) {
    p.ids[row] = id;
    if (p.logprobs) p.logprobs[row] = (float)log(prob);
  }
  // The rest of a row whose candidates are all in CTA 0's sorted list: the first k of
  // them, of those the beginning with the mass p * whole (whole < 0: their own), min-p, the draw.
  __device__ void finish_list(uint32_t row, uint32_t n, uint32_t k, double pp, double whole, double min_p, double u) {
    const uint64_t e[2] = {list[2 * tid], list[2 * tid + 1]};
    double w[2];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) w[j] = 2 * tid + j < min(n, k) ? list_weight(e[j]) : 0.0;
    double total;
    const double in = scan(w[0] + w[1], total), target = pp * (whole < 0 ? total : whole);
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t i = 2 * tid + j;
      const double before = j ? in - w[1] : in - w[1] - w[0];
      const bool stay = i < min(n, k) && (i == 0 || pp >= 1.0 || before < target) && w[j] >= min_p;
      list[i] = stay ? (e[j] & 0xFFFFFFFFull) << 32 | (uint32_t)(e[j] >> 32) : 0;  // (~id, value): by id
    }
    uint32_t n2 = 2;
    while (n2 < n) n2 <<= 1;
    sort(n2);
    const uint64_t f[2] = {list[2 * tid], list[2 * tid + 1]};
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) w[j] = f[j] ? weight(key_float((uint32_t)f[j])) : 0.0;
    const double incl = scan(w[0] + w[1], total), at = u * total;
    if (tid == 0) s.bin = 0xFFFFFFFFu;
    __syncthreads();
    const double in0 = incl - w[1];
    if (f[0] && in0 > at) atomicMin(&s.bin, 2 * tid);
    else if (f[1] && incl > at) atomicMin(&s.bin, 2 * tid + 1);
    if (tid == 0) s.count = 0;
    __syncthreads();
    if (s.bin == 0xFFFFFFFFu) {  // rounding: the last one
      if (f[0]) atomicMax(&s.count, f[1] ? 2 * tid + 1 : 2 * tid);
      __syncthreads();
      if (tid == 0) s.bin = s.count;
      __syncthreads();
    }
    if (s.bin / 2 == tid) {
      const uint32_t j = s.bin & 1;
      answer(row, ~(uint32_t)(f[j] >> 32), w[j] / total);
    }
  }

  // Finds the place of a cut whose bracket is the bins [b0, b1]: the shortest beginning with
  // the count or mass `target`, and takes it over into cut_key and cut_id.
  // True: the row is finished (its elements up to b1 were few).
  template <bool MASS>
  __device__ bool cut(uint32_t row, uint32_t b0, uint32_t b1, double target, uint32_t k, double pp, double whole, double min_p, double u) {
    if (tid == 0) s.count = 0;
    __syncthreads();
    double a = 0;
    uint32_t above = 0, m = 0, kmin = 0xFFFFFFFFu, kmax = 0;
    each([&](float v, uint32_t id) {
      const uint32_t b = min((uint32_t)(z(v) * kPerOctave), kBins - 1), key = float_key(v);
      if (b > b1) return;
      note(key, id);
      if (b < b0) {
        ++above;
        if (MASS) a += weight(v);
      } else {
        ++m;
        kmin = min(kmin, key);
        kmax = max(kmax, key);
      }
    });
    sums(above, m, kmin, kmax);
    if (MASS) a = sum(a);
    Msg msg{MASS ? a : (double)above, 0, above + m, m, kmin, kmax};
    const Msg *all = share(msg);
    double A = 0;
    uint32_t total = 0;
    m = 0;
    for (uint32_t r = 0; r < ctas; ++r) {
      A += all[r].a;
      total += all[r].c;
      m += all[r].d;
      kmin = min(kmin, all[r].e);
      kmax = max(kmax, all[r].f);
    }
    if (total <= kList) {
      uint32_t n;
      if (gather(all, n)) finish_list(row, n, k, pp, whole, min_p, u);
      return true;
    }
    // halve the range of values until the list holds it, or one value is left
    while (m > kList && kmin < kmax) {
      const uint32_t mid = kmin + (kmax - kmin + 1) / 2;
      double b = 0;
      uint32_t up = 0, o0 = 0, o1 = 0xFFFFFFFFu, o2 = 0;
      each([&](float v, uint32_t) {
        const uint32_t key = float_key(v);
        if (key < mid || key > kmax) return;
        ++up;
        if (MASS) b += weight(v);
      });
      sums(up, o0, o1, o2);
      if (MASS) b = sum(b);
      all = share(Msg{MASS ? b : (double)up, 0, up, 0, 0, 0});
      double B = 0;
      uint32_t n = 0;
      for (uint32_t r = 0; r < ctas; ++r) {
        B += all[r].a;
        n += all[r].c;
      }
      if (A + B >= target) {
        kmin = mid;
        m = n;
      } else {
        kmax = mid - 1;
        m -= n;
        A += B;
      }
    }
    if (kmin == kmax) {  // equal values: the first `need` ids of them
      const double w = MASS ? weight(key_float(kmin)) : 1.0, ratio = ceil((target - A) / w);
      const uint32_t need = ratio < 1.0 ? 1 : ratio >= (double)m ? m : (uint32_t)ratio;
      uint32_t own = 0;
      each([&](float v, uint32_t) { own += float_key(v) == kmin; });
      double sum_all;
      const uint32_t in = (uint32_t)scan((double)own, sum_all);
      all = share(Msg{0, 0, (uint32_t)sum_all, 0, 0, 0});
      uint32_t before = 0;
      for (uint32_t r = 0; r < rank; ++r) before += all[r].c;
      uint32_t found = 0xFFFFFFFFu, at = before + in - own, o0 = 0, o1 = 0, o3 = 0;
      if (at < need && need <= before + in)
        each([&](float v, uint32_t id) {
          if (float_key(v) == kmin && ++at == need) found = id;
        });
      sums(o0, o1, found, o3);
      all = share(Msg{0, 0, found, 0, 0, 0});
      for (uint32_t r = 0; r < ctas; ++r) found = min(found, all[r].c);
      cut_key = kmin;
      cut_id = found;
      return false;
    }
    if (tid == 0) s.count = 0;
    __syncthreads();
    each([&](float v, uint32_t id) {
      const uint32_t key = float_key(v);
      if (key >= kmin && key <= kmax) note(key, id);
    });
    __syncthreads();
    all = share(Msg{0, 0, s.count, 0, 0, 0});
    uint32_t n;
    Msg place{};
    if (gather(all, n)) {
      const uint64_t e[2] = {list[2 * tid], list[2 * tid + 1]};
      double w[2];
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) w[j] = 2 * tid + j >= n ? 0.0 : MASS ? list_weight(e[j]) : 1.0;
      double t;
      const double in = scan(w[0] + w[1], t);
      if (tid == 0) s.bin = n - 1;
      __syncthreads();
      if (2 * tid < n && A + (in - w[1]) >= target) atomicMin(&s.bin, 2 * tid);
      else if (2 * tid + 1 < n && A + in >= target) atomicMin(&s.bin, 2 * tid + 1);
      __syncthreads();
      const uint64_t at = list[s.bin];
      place.c = (uint32_t)(at >> 32);
      place.d = ~(uint32_t)at;
    }
    all = share(place);
    cut_key = all[0].c;
    cut_id = all[0].d;
    return false;
  }

  // the draw from what is kept, by id
  __device__ void draw(uint32_t row, double min_p, double u) {
    double own = 0;
    each([&](float v, uint32_t) {
      const double w = weight(v);
      if (w >= min_p) own += w;
    });
    double total;
    const double in = scan(own, total);
    const Msg *all = share(Msg{total, 0, 0, 0, 0, 0});
    double M = 0, before = 0, at;
    for (uint32_t r = 0; r < ctas; ++r) M += all[r].a;
    at = u * M;
    uint32_t r = 0, last = 0;  // the CTA with the token; rounding: the last one with any mass
    for (uint32_t i = 0; i < ctas; ++i)
      if (all[i].a > 0) last = i;
    while (r < last && before + all[r].a <= at) before += all[r++].a;
    if (rank != r) return;
    at -= before;
    // its thread: the first whose sum is above, or the last with any mass
    if (tid == 0) {
      s.bin = 0xFFFFFFFFu;
      s.count = 0;
    }
    __syncthreads();
    if (own > 0) {
      if (in > at) atomicMin(&s.bin, tid);
      atomicMax(&s.count, tid);
    }
    __syncthreads();
    const uint32_t who = s.bin != 0xFFFFFFFFu ? s.bin : s.count;
    if (warp != who / 32) return;
    at -= __shfl_sync(0xFFFFFFFFu, in - own, who % 32);
    const uint32_t f = __shfl_sync(0xFFFFFFFFu, first, who % 32), n = __shfl_sync(0xFFFFFFFFu, n_own, who % 32);
    double run = 0;
    uint32_t best = 0xFFFFFFFFu;
    double best_w = 0;
    for (uint32_t j0 = 0; j0 < n; j0 += 32) {  // the warp takes the thread's elements together
      const uint32_t j = j0 + lane;
      double w = 0;
      if (j < n && kept(x[f + j], id0 + f + j)) w = weight(x[f + j]);
      if (w < min_p) w = 0;
      double sum = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= (uint32_t)o) sum += y;
      }
      const uint32_t over = __ballot_sync(0xFFFFFFFFu, w > 0 && run + sum > at), some = __ballot_sync(0xFFFFFFFFu, w > 0);
      if (over || some) {
        const uint32_t l = over ? __ffs(over) - 1 : 31 - __clz(some);
        best = id0 + f + j0 + l;
        best_w = __shfl_sync(0xFFFFFFFFu, w, l);
      }
      if (over) break;
      run += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    if (lane == 0) answer(row, best, best_w / M);
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample_logits(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ Small s;
  const uint32_t ctas = p.ctas, row = blockIdx.x / ctas;
  Row w(p, s);
  w.tid = threadIdx.x;
  w.lane = w.tid & 31;
  w.warp = w.tid >> 5;
  w.rank = cluster_ctarank();
  w.ctas = ctas;
  w.list = reinterpret_cast<uint64_t *>(dsm);
  w.hist = reinterpret_cast<uint32_t *>(dsm);
  w.x = reinterpret_cast<float *>(dsm + kList * 8);
  const uint32_t slice = p.each * kThreads;
  w.id0 = w.rank * slice;
  w.first = w.tid * p.each;
  // the row's own settings; one that does not hold leaves it as it was (the same for all CTAs)
  const uint32_t at = p.rows ? p.rows[row] : row;
  if (at == FA_NO_TOKEN) return;
  const float t = p.temperature ? p.temperature[row] : 1.0f, u = p.u[row], pp = p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f;
  uint32_t k = p.top_k ? p.top_k[row] : 0;
  if (at >= p.n_logits || !(t == 0.0f || (t >= 1e-6f && t <= 1e6f)) || !(u >= 0.0f && u < 1.0f) || !(pp >= 0.0f) || !(mp >= 0.0f && mp <= 1.0f)) {
    if (p.err && w.rank == 0 && w.tid == 0) atomicOr(p.err, kFlagRange);
    return;
  }
  // the CTA's part of the row, in f32; behind its end nothing
  const uint32_t len = w.id0 < p.vocab ? min(slice, p.vocab - w.id0) : 0;
  w.n_own = w.first < len ? min(p.each, len - w.first) : 0;
  const T *src = reinterpret_cast<const T *>(p.logits) + (uint64_t)at * p.ld + w.id0;
  float mx = -INFINITY;
  constexpr uint32_t kV = 16 / sizeof(T);
  uint32_t i = 0;
  if (p.aligned) {
    const uint32_t whole = len / kV;
    constexpr uint32_t kAhead = 8;  // loads in flight
    for (uint32_t j0 = w.tid; j0 < whole; j0 += kAhead * kThreads) {
      Vec<T> v[kAhead];
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
        if (j0 + a * kThreads < whole) v[a] = *reinterpret_cast<const Vec<T> *>(src + (uint64_t)(j0 + a * kThreads) * kV);
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) {
        if (j0 + a * kThreads >= whole) break;
        float f[kV];
#pragma unroll
        for (uint32_t e = 0; e < kV; ++e) {
          f[e] = to_logit((float)v[a].v[e]);
          mx = fmaxf(mx, f[e]);
        }
#pragma unroll
        for (uint32_t e = 0; e < kV; e += 4)
          *reinterpret_cast<float4 *>(w.x + (j0 + a * kThreads) * kV + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      }
    }
    i = whole * kV;
  }
  for (uint32_t j = i + w.tid; j < len; j += kThreads) {
    const float f = to_logit((float)src[j]);
    w.x[j] = f;
    mx = fmaxf(mx, f);
  }
  uint32_t o0 = 0, o1 = 0, o2 = 0, key = float_key(mx);
  w.sums(o0, o1, o2, key);
  const Msg *all = w.share(Msg{0, 0, key, 0, 0, 0});
  for (uint32_t r = 0; r < ctas; ++r) key = max(key, all[r].c);
  w.mx = key_float(key);
  if (w.mx == -INFINITY) {  // no candidate at all
    if (w.rank == 0 && w.tid == 0) {
      p.ids[row] = FA_NO_TOKEN;
      if (p.logprobs) p.logprobs[row] = -INFINITY;
      if (p.err) atomicOr(p.err, kFlagRange);
    }
    return;
  }
  if (t == 0.0f) {  // the lowest id of the maximum
    uint32_t best = 0xFFFFFFFFu;
    for (uint32_t j = w.n_own; j-- > 0;)
      if (w.x[w.first + j] == w.mx) best = w.id0 + w.first + j;
    w.sums(o0, o1, best, o2);
    all = w.share(Msg{0, 0, best, 0, 0, 0});
    for (uint32_t r = 0; r < ctas; ++r) best = min(best, all[r].c);
    if (w.rank == 0 && w.tid == 0) w.answer(row, best, 1.0);
    return;
  }
  w.cd = 1.4426950408889634074 / (double)t;
  w.cf = (float)w.cd;
  w.mxd = (double)w.mx;
  if (k && k < p.vocab) {
    w.fill<false>(0);
    const double total = w.reduce_bins<false>();
    all = w.share(Msg{total, 0, 0, 0, 0, 0});
    double n = 0;
    for (uint32_t r = 0; r < ctas; ++r) n += all[r].a;
    if (n > (double)k) {
      const uint32_t b = w.find_bin(all, (double)k);
      cluster_sync();  // the sums over bins have been read
      if (w.cut<false>(row, b, b, (double)k, k, pp, -1.0, mp, u)) return;
    } else {
      cluster_sync();
    }
  }
  if (pp < 1.0f) {
    // all mass above z_most is less than half of what may be cut: the place is below it
    const float z_most = log2f((float)p.vocab) - log2f(1.0f - pp) + 1.0f;
    const double whole = w.fill<true>(z_most);
    const double total = w.reduce_bins<true>();
    all = w.share(Msg{total, whole, 0, 0, 0, 0});
    double W = 0;
    for (uint32_t r = 0; r < ctas; ++r) W += all[r].b;
    const double target = (double)pp * W;
    const uint32_t b0 = w.find_bin(all, target * (1.0 - 2 * kHistError)), b1 = w.find_bin(all, target * (1.0 + 2 * kHistError));
    cluster_sync();
    if (w.cut<true>(row, b0, b1, target, 0xFFFFFFFFu, pp, W, mp, u)) return;
  }
  w.draw(row, (double)mp, (double)u);
}

template <typename T>
int launch(const SampleParams &p, cudaStream_t st) {
  const uint32_t smem = kList * 8 + p.each * kThreads * 4;
  if (cudaFuncSetAttribute(k_sample_logits<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleMaxSmem) != cudaSuccess) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n * p.ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_sample_logits<T>, p) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_sample_logits(const SampleParams &in, cudaStream_t st) {
  SampleParams p = in;
  // the smallest cluster that leaves 17 elements or fewer a thread; eight CTAs at most
  p.ctas = 1;
  while (p.ctas < kMaxCtas && (p.vocab + p.ctas * kThreads - 1) / (p.ctas * kThreads) > 17) p.ctas *= 2;
  p.each = ((p.vocab + p.ctas * kThreads - 1) / (p.ctas * kThreads)) | 1;  // odd
  switch (p.dtype) {
    case FA_KV_F32: return launch<float>(p, st);
    case FA_KV_F16: return launch<__half>(p, st);
    default: return launch<__nv_bfloat16>(p, st);
  }
}

}  // namespace fa
