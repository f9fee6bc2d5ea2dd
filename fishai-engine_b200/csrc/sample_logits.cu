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

constexpr uint32_t kThreads = 512, kWarps = kThreads / 32, kBins = 2048, kList = 1024, kMaxCtas = 8;
constexpr float kOctaves = 64.0f, kPerOctave = kBins / kOctaves;
constexpr double kHistError = 1.0 / 32768;  // of a sum of the histogram's masses: each is rounded to 2^-15 of its bin's largest, and exponentials are f32
constexpr uint32_t kGroup = 4 * kThreads;   // elements of a CTA's group: four a thread, a warp's 128 in a row

struct Msg {  // what a CTA tells the others
  double a, b;
  uint32_t c, d, e, f;
};
struct Small {
  Msg msg[2][kMaxCtas];
  double red[kWarps];
  uint32_t redu[4][kWarps];
  uint32_t bin, count;
  double power[32];  // 2^(i / 32)
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

// A cluster's work on one row.  Element e of the thread in group g is number
// warp * 128 groups + 128 g + 4 lane + e of the CTA's part: a warp has consecutive ids.
struct Row {
  const SampleParams &p;
  Small &s;
  float *x;         // this CTA's part of the row; -inf behind its end
  uint32_t *hist;   // [kBins]
  double *binsum;   // [kBins / ctas] inclusive sums of this CTA's share of the cluster's bins
  uint64_t *list;   // [kList] (ordered value, ~id)
  uint32_t tid, lane, warp, rank, ctas, groups, mine;  // mine: the thread's first element
  uint32_t id0;     // id of the CTA's first element
  uint32_t turn = 0;
  float mx, cf;     // the maximum, log2(e) / T
  double mxd, c32;  // 32 log2(e) / T
  // kept so far: value above the key, or equal and id at most cut_id
  uint32_t cut_key = 0, cut_id = 0xFFFFFFFFu;

  __device__ Row(const SampleParams &p, Small &s) : p(p), s(s) {}

  __device__ float z(float v) const { return (mx - v) * cf; }
  // 2^-z in 64 bits, table-driven: 2^(n / 32) from a table, 2^(f / 32), |f| <= 1/2, from the series to
  // f^5 (the next term is below 2^-48.6).  For z <= 64, so the exponent stays in range.
  __device__ double weight(float v) const {
    const double d = (double)v - mxd, big = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the nearest whole number
    const double t = fma(d, c32, big);
    const int n = __double2loint(t);
    const double f = fma(d, c32, big - t);
    double y = 3.97370998454941613e-11;  // (ln 2 / 32)^k / k!
    y = fma(y, f, 9.17256270182464329e-9);
    y = fma(y, f, 1.69385097243718201e-6);
    y = fma(y, f, 0.000234596198202246789);
    y = fma(y, f, 0.0216608493924982909);
    y = fma(y, f, 1.0);
    y *= s.power[n & 31];
    return __hiloint2double(__double2hiint(y) + ((n >> 5) << 20), __double2loint(y));
  }
  template <bool CUT>
  __device__ bool kept(float v, uint32_t id) const {
    if (!(z(v) <= kOctaves)) return false;
    if (!CUT) return true;
    const uint32_t k = float_key(v);
    return k > cut_key || (k == cut_key && id <= cut_id);
  }
  // Four values at once, without a branch: their chains of dependent operations run side by side.  Where
  // use[j] is false, 0.
  __device__ void weights(const float (&v)[4], const bool (&use)[4], double (&w)[4]) const {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) w[j] = weight(v[j]);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
      if (!use[j]) w[j] = 0.0;
  }
  // f(values, which are kept, first id) of the thread's groups of four, in the order of ids
  template <bool CUT, typename F>
  __device__ void each4(F f) const {
    for (uint32_t g = 0; g < groups; ++g) {
      const float4 x4 = *reinterpret_cast<const float4 *>(x + mine + 128 * g);
      const uint32_t id = id0 + mine + 128 * g;
      const float v[4] = {x4.x, x4.y, x4.z, x4.w};
      bool use[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) use[j] = kept<CUT>(v[j], id + j);
      f(v, use, id);
    }
  }
  // f(value, id) of the thread's elements that are kept
  template <bool CUT, typename F>
  __device__ void each(F f) const {
    for (uint32_t g = 0; g < groups; ++g) {
      const float4 v = *reinterpret_cast<const float4 *>(x + mine + 128 * g);
      const uint32_t id = id0 + mine + 128 * g;
      if (kept<CUT>(v.x, id)) f(v.x, id);
      if (kept<CUT>(v.y, id + 1)) f(v.y, id + 1);
      if (kept<CUT>(v.z, id + 2)) f(v.z, id + 2);
      if (kept<CUT>(v.w, id + 3)) f(v.w, id + 3);
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

  // n more in bin b; those of one bin in a row are added at once
  struct Bin {
    uint32_t *hist, b = 0, n = 0;
    __device__ void add(uint32_t to, uint32_t by) {
      if (to != b) {
        flush();
        b = to;
        n = 0;
      }
      n += by;
    }
    __device__ void flush() {
      if (n) atomicAdd(hist + b, n);
    }
  };
  __device__ uint32_t bin_of(float zv) const { return min((uint32_t)(zv * kPerOctave), kBins - 1); }
  __device__ void clear() {
    for (uint32_t i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
  }
  // histogram of the kept elements' counts
  template <bool CUT>
  __device__ void fill_counts() {
    clear();
    Bin bin{hist};
    each<CUT>([&](float v, uint32_t) { bin.add(bin_of(z(v)), 1); });
    bin.flush();
  }
  // of their masses, where elements above z_most only count for the whole mass, which is returned
  template <bool CUT>
  __device__ double fill_masses(float z_most) {
    clear();
    double w = 0;
    Bin bin{hist};
    each4<CUT>([&](const float (&v)[4], const bool (&use)[4], uint32_t) {
      double e[4];
      weights(v, use, e);
      w += (e[0] + e[1]) + (e[2] + e[3]);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const float zv = z(v[j]);
        if (!use[j] || zv > z_most) continue;
        const uint32_t b = bin_of(zv);
        bin.add(b, __float2uint_rn(exp2f((float)b * (1.0f / kPerOctave) - zv) * 32768.0f));
      }
    });
    bin.flush();
    return sum(w);
  }
  // The cluster's sums over bins: each CTA takes a share of the bins.  Returns that share's total.
  template <bool MASS>
  __device__ double reduce_bins() {
    const uint32_t nb = kBins / ctas, per = nb > kThreads ? nb / kThreads : 1;  // at most 4 a thread
    double v[4] = {0, 0, 0, 0};
    cluster_sync();
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t i = tid * per + j;
      if (j >= per || i >= nb) continue;
      const uint32_t b = rank * nb + i;
      uint32_t h[kMaxCtas];
#pragma unroll
      for (uint32_t r = 0; r < kMaxCtas; ++r) h[r] = r < ctas ? ld_cluster32(dsmem_addr(hist + b, r)) : 0;
      uint64_t t = 0;
#pragma unroll
      for (uint32_t r = 0; r < kMaxCtas; ++r) t += h[r];
      v[j] = MASS ? (double)t * exp2(-(double)b / kPerOctave - 15.0) : (double)t;
    }
    double total;
    double in = scan((v[0] + v[1]) + (v[2] + v[3]), total) - ((v[0] + v[1]) + (v[2] + v[3]));
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      in += v[j];
      if (j < per && tid * per + j < nb) binsum[tid * per + j] = in;
    }
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
    for (uint32_t i = tid; i < nb; i += kThreads)
      if (before + __longlong_as_double((long long)ld_cluster64(dsmem_addr(binsum + i, r))) >= target) atomicMin(&s.bin, i);
    __syncthreads();
    const uint32_t b = r * nb + s.bin;
    __syncthreads();
    return b;
  }
  __device__ void note(uint32_t key, uint32_t id) {
    if (*reinterpret_cast<volatile uint32_t *>(&s.count) >= kList) return;  // a list that is full is of no use
    const uint32_t at = atomicAdd(&s.count, 1u);
    if (at < kList) list[at] = (uint64_t)key << 32 | (uint32_t)~id;
  }
  // Sorts list[0 .. n) in descending order, entries all different; behind them zeros to the next power of
  // two.  Up to 128 by counting the larger ones, four threads an entry: two barriers (a bitonic sort of 128: 28).
  __device__ void sort(uint32_t some) {
    if (some <= 128) {
      const uint32_t i = tid / 4;
      uint64_t e = 0;
      uint32_t place = 0;
      __syncthreads();
      if (i < some) {
        e = list[i];
        for (uint32_t j = tid % 4; j < some; j += 4) place += list[j] > e;
      }
      place += __shfl_xor_sync(0xFFFFFFFFu, place, 1);
      place += __shfl_xor_sync(0xFFFFFFFFu, place, 2);
      __syncthreads();
      if (tid < some) list[tid] = 0;
      __syncthreads();
      if (e && tid % 4 == 0) list[place] = e;
      __syncthreads();
      return;
    }
    uint32_t n = 2;
    while (n < some) n <<= 1;
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
    sort(n);
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
    sort(n);
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

  // What top-k needs, where k is small beside the threads: the elements down to the bin in which
  // the threads' k-th largest maximum lies, a few more than k.  True: the row is finished.
  __device__ bool few_largest(uint32_t row, float best, uint32_t k, double pp, double min_p, double u) {
    clear();
    if (tid == 0) s.count = 0;
    if (z(best) <= kOctaves) atomicAdd(hist + bin_of(z(best)), 1u);
    const Msg *all = share(Msg{reduce_bins<false>(), 0, 0, 0, 0, 0});
    double n = 0;
    for (uint32_t r = 0; r < ctas; ++r) n += all[r].a;
    if (n < (double)k) return false;
    const uint32_t b = find_bin(all, (double)k);
    uint32_t own = 0, o1 = 0, o2 = 0, o3 = 0;
    each<false>([&](float v, uint32_t id) {
      if (bin_of(z(v)) > b) return;
      note(float_key(v), id);
      ++own;
    });
    sums(own, o1, o2, o3);
    all = share(Msg{0, 0, own, 0, 0, 0});
    own = 0;
    for (uint32_t r = 0; r < ctas; ++r) own += all[r].c;
    if (own > kList) return false;
    uint32_t m;
    if (gather(all, m)) finish_list(row, m, k, pp, -1.0, min_p, u);
    return true;
  }

  // mass of the thread's elements above `upto`, where a cut has formed it
  double strict = 0;
  uint32_t upto = 0xFFFFFFFFu;

  // Finds the place of a cut whose bracket is the bins [b0, b1]: the shortest beginning with
  // the count or mass `target`, and takes it over into cut_key and cut_id.  CUT: there is one already.
  // True: the row is finished (its elements up to b1 were few).
  template <bool MASS, bool CUT>
  __device__ bool cut(uint32_t row, uint32_t b0, uint32_t b1, double target, uint32_t k, double pp, double whole, double min_p, double u) {
    if (tid == 0) s.count = 0;
    __syncthreads();
    double a = 0;
    uint32_t above = 0, m = 0, kmin = 0xFFFFFFFFu, kmax = 0;
    each4<CUT>([&](const float (&v)[4], const bool (&use)[4], uint32_t id) {
      bool over[4], any = false;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t b = bin_of(z(v[j]));
        over[j] = use[j] && b < b0;
        any |= over[j];
        above += over[j];
        if (use[j] && b >= b0 && b <= b1) {
          const uint32_t key = float_key(v[j]);
          note(key, id + j);
          ++m;
          kmin = min(kmin, key);
          kmax = max(kmax, key);
        }
      }
      if (MASS && any) {
        double w[4];
        weights(v, over, w);
        a += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          if (w[j] >= min_p) strict += w[j];
      }
    });
    sums(above, m, kmin, kmax);
    if (MASS) a = sum(a);
    const Msg *all = share(Msg{MASS ? a : (double)above, 0, above + m, m, kmin, kmax});
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
    if (total <= kList) {  // all of them to the list
      each<CUT>([&](float v, uint32_t id) {
        if (bin_of(z(v)) < b0) note(float_key(v), id);
      });
      __syncthreads();
      all = share(Msg{0, 0, s.count, 0, 0, 0});
      uint32_t n;
      if (gather(all, n)) finish_list(row, n, k, pp, whole, min_p, u);
      return true;
    }
    const bool listed = m <= kList;
    if (MASS) upto = kmax;
    // halve the range of values until the list holds it, or one value is left
    while (m > kList && kmin < kmax) {
      const uint32_t mid = kmin + (kmax - kmin + 1) / 2;
      double b = 0;
      uint32_t up = 0, o1 = 0, o2 = 0, o3 = 0;
      each<CUT>([&](float v, uint32_t) {
        const uint32_t key = float_key(v);
        if (key < mid || key > kmax) return;
        ++up;
        if (MASS) b += weight(v);
      });
      sums(up, o1, o2, o3);
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
      uint32_t own = 0, o1 = 0, o2 = 0, o3 = 0;
      each<CUT>([&](float v, uint32_t) { own += float_key(v) == kmin; });
      // by ids: CTAs, warps, groups of a warp, lanes
      const uint32_t of_warp = __reduce_add_sync(0xFFFFFFFFu, own);
      sums(own, o1, o2, o3);  // leaves the warps' sums of `own`
      all = share(Msg{0, 0, own, 0, 0, 0});
      uint32_t before = 0, found = 0xFFFFFFFFu;
      for (uint32_t r = 0; r < rank; ++r) before += all[r].c;
      for (uint32_t i = 0; i < warp; ++i) before += s.redu[0][i];
      if (before < need && need <= before + of_warp)
        for (uint32_t g = 0; g < groups; ++g) {
          const float4 v = *reinterpret_cast<const float4 *>(x + mine + 128 * g);
          const uint32_t id = id0 + mine + 128 * g;
          const float e[4] = {v.x, v.y, v.z, v.w};
          bool yes[4];
          uint32_t n = 0;
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) n += yes[j] = kept<CUT>(e[j], id + j) && float_key(e[j]) == kmin;
          uint32_t in = n;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, in, o);
            if (lane >= (uint32_t)o) in += y;
          }
          uint32_t at = before + in - n;
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j)
            if (yes[j] && ++at == need) found = id + j;
          before += __shfl_sync(0xFFFFFFFFu, in, 31);
        }
      o1 = o2 = o3 = 0;
      sums(o1, o2, found, o3);
      all = share(Msg{0, 0, found, 0, 0, 0});
      for (uint32_t r = 0; r < ctas; ++r) found = min(found, all[r].c);
      cut_key = kmin;
      cut_id = found;
      return false;
    }
    if (!listed) {
      if (tid == 0) s.count = 0;
      __syncthreads();
      each<CUT>([&](float v, uint32_t id) {
        const uint32_t key = float_key(v);
        if (key >= kmin && key <= kmax) note(key, id);
      });
    }
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
  template <bool CUT>
  __device__ void draw(uint32_t row, double min_p, double u) {
    double own = strict;
    each4<CUT>([&](const float (&v)[4], const bool (&use)[4], uint32_t) {
      bool add[4], any = false;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        add[j] = use[j] && !(CUT && float_key(v[j]) > upto);  // those above are counted
        any |= add[j];
      }
      if (CUT && !any) return;
      double w[4];
      weights(v, add, w);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (w[j] >= min_p) own += w[j];
    });
    double of_warp = own;
#pragma unroll
    for (int o = 16; o; o >>= 1) of_warp += __shfl_xor_sync(0xFFFFFFFFu, of_warp, o);
    __syncthreads();
    if (lane == 0) s.red[warp] = of_warp;
    __syncthreads();
    double total = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWarps; ++i) total += s.red[i];
    const Msg *all = share(Msg{total, 0, 0, 0, 0, 0});
    double M = 0, at, before = 0;
    for (uint32_t r = 0; r < ctas; ++r) M += all[r].a;
    at = u * M;
    // the CTA with the token, then its warp: the first whose sum is above, or (rounding) the last with any mass
    uint32_t r = 0, last = 0;
    for (uint32_t i = 0; i < ctas; ++i)
      if (all[i].a > 0) last = i;
    while (r < last && before + all[r].a <= at) before += all[r++].a;
    if (rank != r) return;
    at -= before;
    before = 0;
    uint32_t who = 0;
    for (uint32_t i = 0; i < kWarps; ++i)
      if (s.red[i] > 0) last = i;
    if (s.red[last] == 0) last = kWarps - 1;
    while (who < last && before + s.red[who] <= at) before += s.red[who++];
    // that warp's groups, one to each warp
    at -= before;
    const uint32_t chunk = who * 128 * groups + 4 * lane;
    auto group = [&](uint32_t g, float (&v)[4], double (&w)[4]) {
      const float4 x4 = *reinterpret_cast<const float4 *>(x + chunk + 128 * g);
      const uint32_t id = id0 + chunk + 128 * g;
      v[0] = x4.x, v[1] = x4.y, v[2] = x4.z, v[3] = x4.w;
      bool use[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) use[j] = kept<CUT>(v[j], id + j);
      weights(v, use, w);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (w[j] < min_p) w[j] = 0.0;
    };
    double *of_group = reinterpret_cast<double *>(list);
    float v[4];
    double w[4];
    for (uint32_t g = warp; g < groups; g += kWarps) {
      group(g, v, w);
      double t = (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
      for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
      if (lane == 0) of_group[g] = t;
    }
    __syncthreads();
    uint32_t g = 0;
    before = 0;
    last = 0;
    for (uint32_t i = 0; i < groups; ++i)
      if (of_group[i] > 0) last = i;
    while (g < last && before + of_group[g] <= at) before += of_group[g++];
    if (g % kWarps != warp) return;
    at -= before;
    group(g, v, w);
    const double four = (w[0] + w[1]) + (w[2] + w[3]);
    double in = four;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xFFFFFFFFu, in, o);
      if (lane >= (uint32_t)o) in += y;
    }
    const uint32_t over = __ballot_sync(0xFFFFFFFFu, four > 0 && in > at), some = __ballot_sync(0xFFFFFFFFu, four > 0);
    if (lane != (over ? __ffs(over) - 1 : 31 - __clz(some))) return;
    double sum = in - four, best_w = 0;
    uint32_t best = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      if (w[j] > 0 && !(best_w > 0 && sum > at)) {
        best = id0 + chunk + 128 * g + j;
        best_w = w[j];
      }
      sum += w[j];
    }
    answer(row, best, best_w / M);
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
  w.groups = p.groups;
  w.list = reinterpret_cast<uint64_t *>(dsm);
  w.hist = reinterpret_cast<uint32_t *>(dsm + kList * 8);
  w.binsum = reinterpret_cast<double *>(dsm + kList * 8 + kBins * 4);
  w.x = reinterpret_cast<float *>(dsm + kList * 8 + kBins * 4 + kBins / ctas * 8);
  const uint32_t slice = p.groups * kGroup;
  w.id0 = w.rank * slice;
  w.mine = w.warp * 128 * p.groups + 4 * w.lane;
  if (w.tid < 32) s.power[w.tid] = exp2((double)w.tid / 32.0);
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
  for (uint32_t j = i + w.tid; j < slice; j += kThreads) {
    const float f = j < len ? to_logit((float)src[j]) : -INFINITY;
    w.x[j] = f;
    mx = fmaxf(mx, f);
  }
  const float own_max = mx;
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
    for (uint32_t j = w.tid; j < len; j += kThreads)
      if (w.x[j] == w.mx) best = min(best, w.id0 + j);
    w.sums(o0, o1, best, o2);
    all = w.share(Msg{0, 0, best, 0, 0, 0});
    for (uint32_t r = 0; r < ctas; ++r) best = min(best, all[r].c);
    if (w.rank == 0 && w.tid == 0) w.answer(row, best, 1.0);
    return;
  }
  const double c = 1.4426950408889634074 / (double)t;
  w.cf = (float)c;
  w.c32 = 32.0 * c;
  w.mxd = (double)w.mx;
  bool has_cut = false;
  if (k && k < p.vocab) {
    // a quarter of the threads: beyond it the maxima stand for more and more elements
    if (k <= ctas * kThreads / 4 && w.few_largest(row, own_max, k, pp, mp, u)) return;
    w.fill_counts<false>();
    all = w.share(Msg{w.reduce_bins<false>(), 0, 0, 0, 0, 0});
    double n = 0;
    for (uint32_t r = 0; r < ctas; ++r) n += all[r].a;
    if (n > (double)k) {
      const uint32_t b = w.find_bin(all, (double)k);
      if (w.cut<false, false>(row, b, b, (double)k, k, pp, -1.0, mp, u)) return;
      has_cut = true;
    }
  }
  if (pp < 1.0f) {
    // all mass above z_most is less than half of what may be cut: the place is below it
    const float z_most = log2f((float)p.vocab) - log2f(1.0f - pp) + 1.0f;
    const double whole = has_cut ? w.fill_masses<true>(z_most) : w.fill_masses<false>(z_most);
    const double total = w.reduce_bins<true>();
    all = w.share(Msg{total, whole, 0, 0, 0, 0});
    double W = 0;
    for (uint32_t r = 0; r < ctas; ++r) W += all[r].b;
    const double target = (double)pp * W;
    const uint32_t b0 = w.find_bin(all, target * (1.0 - 2 * kHistError)), b1 = w.find_bin(all, target * (1.0 + 2 * kHistError));
    if (has_cut ? w.cut<true, true>(row, b0, b1, target, 0xFFFFFFFFu, pp, W, mp, u) : w.cut<true, false>(row, b0, b1, target, 0xFFFFFFFFu, pp, W, mp, u))
      return;
    has_cut = true;
  }
  if (has_cut) w.draw<true>(row, (double)mp, (double)u);
  else w.draw<false>(row, (double)mp, (double)u);
}

template <typename T>
int launch(const SampleParams &p, cudaStream_t st) {
  const uint32_t smem = kList * 8 + kBins * 4 + kBins / p.ctas * 8 + p.groups * kGroup * 4;
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
  // the smallest cluster that leaves four groups or fewer; eight CTAs at most
  auto groups = [&](uint32_t ctas) { return (p.vocab + ctas * kGroup - 1) / (ctas * kGroup); };
  p.ctas = 1;
  while (p.ctas < kMaxCtas && groups(p.ctas) > 4) p.ctas *= 2;
  p.groups = groups(p.ctas);
  static_assert(kSampleMaxVocab == kMaxCtas * kGroup * 25 && kList * 8 + kBins * 4 + kBins / kMaxCtas * 8 + 25 * kGroup * 4 <= kSampleMaxSmem,
                "shared memory of the largest vocabulary");
  switch (p.dtype) {
    case FA_KV_F32: return launch<float>(p, st);
    case FA_KV_F16: return launch<__half>(p, st);
    default: return launch<__nv_bfloat16>(p, st);
  }
}

}  // namespace fa
