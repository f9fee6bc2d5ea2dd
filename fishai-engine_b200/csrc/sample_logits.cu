// Draws a token from each row of logits, with cuts of the row's own:
//   w_v = 2^(-z_v),  z_v = (max x - x_v) log2(e) / T       (0 where z_v > 64)
//   order: x descending, equal ones by id;  top-k: the first k;
//   top-p: the shortest beginning of those whose mass is at least p of theirs;
//   min-p: those with w >= min_p;
//   the token: the first by id at which the mass of the kept ones exceeds u times all of it.
// Every cut keeps a beginning of the same order, so a row's cuts are one place in it.
//
// Each row is read once: a cluster of up to eight CTAs holds it in shared memory and
// exchanges sums over distributed shared memory.  Masses are 64-bit sums of
// 64-bit exponentials in a fixed order: which token is drawn from a flat row of 10^5
// tokens depends on 17 bits more than f32 has.
//
// Rows are not sorted.  A small top-k: each CTA notes its elements from the k-th largest
// of its threads' maxima on, a few more than k, and CTA 0 picks from those.  Other cuts: a histogram
// over z (of counts, or of masses to 2^-15, which bracket the place of the cut) leads to
// the elements of the bins around the place, which CTA 0 sorts.  Where more are in the bracket
// than it sorts, its range of values is halved until it does, or one value is left and the place is an id:
// flat rows, equal logits, and a top-p near to 1, since the bracket is 3 2^-15 of the mass to either side, in whole
// bins (of 128256 normal logits with a few peaks, at temperature 1, it holds some 200 at 0.9, 650 at 0.99, 2200 at
// 0.999, 9000 at 0.9999, which is two to five halvings, each a pass and an exchange).
//
// A row alone waits for its exchanges (1 us each) and three passes of 2 to 5 us: of 128256 in f32
// 10 us without cuts, 12 with top-k, 26 with top-p, 34 at 0.999 and 48 at 0.9999.  Many rows are bound by issue slots
// and the rows that have most to do: 64 without cuts 27 us, with top-k 32, with cuts of all kinds 35 to 38, with
// top-p on every row 68, at 0.999 103 and at 0.9999 183; 200 of 32000 in bf16 19, with top-p 69.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "fa_device.cuh"
#include "paged_ops.hpp"

namespace fa {
namespace {

constexpr uint32_t kThreads = 512, kWarps = kThreads / 32, kMaxCtas = 8;
constexpr uint32_t kList = 2048, kSort = 1024;  // noted elements of a CTA (and of a cluster); most that are sorted
constexpr uint32_t kCtaBins = 512;              // bins for each CTA of the cluster: finer for longer rows
constexpr uint32_t kFewK = 128;                 // the top-k that goes by the threads' maxima
constexpr float kOctaves = 64.0f;
constexpr double kHistError = 1.0 / 32768;      // of a sum of the histogram's masses: each is rounded to 2^-15 of its bin's largest, and exponentials are f32
constexpr uint32_t kGroup = 4 * kThreads;       // elements of a CTA's group: four a thread, a warp's 128 in a row

constexpr uint32_t kMostGroups = 32;            // of a CTA: a lane looks at each

struct alignas(16) Msg {  // what a CTA tells the others
  double a, b;
  uint32_t c, d, e, f;
};
struct Small {
  Msg msg[2][kMaxCtas];
  double red[kWarps], red2[kWarps];
  double group[kMostGroups];  // of a warp's groups
  uint32_t redu[4][kWarps];
  uint32_t bin, count, bins[2];
  double power[512];  // 2^(i / 512)
};

// the larger of both, NaN beside a number left out
__device__ __forceinline__ __half2 larger(__half2 a, __half2 b) { return __hmax2(a, b); }
__device__ __forceinline__ __nv_bfloat162 larger(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2(a, b); }
__device__ __forceinline__ uint32_t key_of(float v) { return float_key(v + 0.0f); }  // -0 as +0
__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// how the maximum is kept while a row is read: in pairs for 16-bit types
template <typename T>
struct Pair {
  using type = float;
  __device__ static float none() { return -INFINITY; }
  __device__ static float top(float x) { return x; }
};
template <>
struct Pair<__half> {
  using type = __half2;
  __device__ static __half2 none() { return __float2half2_rn(-INFINITY); }
  __device__ static float top(__half2 x) { return fmaxf(__low2float(x), __high2float(x)); }
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  __device__ static __nv_bfloat162 none() { return __float2bfloat162_rn(-INFINITY); }
  __device__ static float top(__nv_bfloat162 x) { return fmaxf(__low2float(x), __high2float(x)); }
};
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }

__device__ __forceinline__ void st_cluster(uint32_t addr, const Msg &m) {
  const uint64_t a = __double_as_longlong(m.a), b = __double_as_longlong(m.b), c = (uint64_t)m.d << 32 | m.c, d = (uint64_t)m.f << 32 | m.e;
  asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(addr), "l"(a), "l"(b) : "memory");
  asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(addr + 16), "l"(c), "l"(d) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t ld_cluster64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
// Dynamic shared memory: the list of noted elements, over it the cluster's bins; sums over this CTA's
// share of the bins; the CTA's part of the row.  (Reached by the array's name, which lets the compiler
// see that it is shared memory.)
__device__ __forceinline__ uint8_t *space() {
  extern __shared__ __align__(16) uint8_t sample_sm[];
  return sample_sm;
}
__host__ __device__ constexpr uint32_t region(uint32_t ctas) { return kList * 8 > kCtaBins * 4 * ctas ? kList * 8 : kCtaBins * 4 * ctas; }

template <bool CUTS>
__host__ __device__ constexpr uint32_t row_at(uint32_t ctas) {
  return CUTS ? region(ctas) + kCtaBins * 8 : 0;
}

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

// A cluster's work on one row.  Element e of the thread in group g is number
// warp * 128 groups + 128 g + 4 lane + e of the CTA's part: a warp has consecutive ids.
template <typename T>
struct Row {
  const SampleParams &p;
  Small &s;
  uint32_t x_at;    // where the row is
  uint32_t tid, lane, warp, rank, ctas, bins, groups, mine;  // mine: the thread's first element
  uint32_t id0;     // id of the CTA's first element
  uint32_t turn = 0;
  float mx, cb, low;   // the maximum; bins a unit of x; where z = 64 (to f32's rounding): below it and NaN is no candidate
  double mxd, c512;    // 512 log2(e) / T
  // kept so far: value above cut_at, or equal and id at most cut_id
  float cut_at = -INFINITY;
  uint32_t cut_id = 0xFFFFFFFFu;

  __device__ Row(const SampleParams &p, Small &s) : p(p), s(s) {}

  __device__ void scale(float top, float t) {
    const double c = 1.4426950408889634074 / (double)t;
    mx = top;
    mxd = (double)top;
    c512 = 512.0 * c;
    bins = kCtaBins * ctas;
    cb = (float)(c * (bins / kOctaves));
    low = __double2float_ru(mxd - (double)kOctaves / c);  // upwards: weight() needs z <= 64
  }
  __device__ float z(float v) const { return (mx - v) * cb; }  // in bins
  __device__ T *x() const { return reinterpret_cast<T *>(space() + x_at); }                    // -inf behind its end
  __device__ uint64_t *list() const { return reinterpret_cast<uint64_t *>(space()); }            // [kList] (ordered value, ~id)
  __device__ uint32_t *hist() const { return reinterpret_cast<uint32_t *>(space()); }            // [bins]
  __device__ double *binsum() const { return reinterpret_cast<double *>(space() + x_at) - kCtaBins; }  // [kCtaBins], inclusive

  // 2^-z in 64 bits, table-driven: 2^(n / 512) from a table, 2^(f / 512), |f| <= 1/2, from the series to
  // f^3 (the next term is below 2^-46.7).  For z <= 64, so the exponent stays in range.  The 64-bit
  // pipe has 64 lanes a clock and SM: a longer table for two terms less (a table of 32 needs the series to f^5).
  __device__ double weight(float v) const {
    const double d = (double)v - mxd, big = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the nearest whole number
    const double t = fma(d, c512, big);
    const int n = __double2loint(t);
    const double f = fma(d, c512, big - t);
    double y = 4.13537835067671388e-10;  // (ln 2 / 512)^k / k!
    y = fma(y, f, 9.16391399227526521e-7);
    y = fma(y, f, 0.00135380308703114318);
    y = fma(y, f, 1.0) * s.power[n & 511];
    return __hiloint2double(__double2hiint(y) + ((n >> 9) << 20), __double2loint(y));
  }
  template <bool CUT>
  __device__ bool kept(float v, uint32_t id) const {
    return v >= low && (!CUT || v > cut_at || (v == cut_at && id <= cut_id));
  }
  // Four values at once, without a branch: their chains of dependent operations run side by side.
  __device__ void weights(const float (&v)[4], double (&w)[4]) const {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) w[j] = weight(v[j]);
  }
  __device__ void load(uint32_t at, float (&v)[4]) const {
    const Four<T> f = *reinterpret_cast<const Four<T> *>(x() + at);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) v[j] = (float)f.v[j];
  }
  // f(values, which are kept, first id) of the thread's groups of four, in the order of ids
  template <bool CUT, typename F>
  __device__ void each4(F f) const {
    for (uint32_t g = 0; g < groups; ++g) {
      float v[4];
      load(mine + 128 * g, v);
      const uint32_t id = id0 + mine + 128 * g;
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
      float v[4];
      load(mine + 128 * g, v);
      const uint32_t id = id0 + mine + 128 * g;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (kept<CUT>(v[j], id + j)) f(v[j], id + j);
    }
  }

  // Whether row i goes by a histogram, which takes twice as long as all else.
  __device__ bool lengthy(uint32_t i) const {
    if (i >= p.n || (p.temperature && p.temperature[i] == 0.0f)) return false;
    const uint32_t k = p.top_k && p.top_k[i] < p.vocab ? p.top_k[i] : 0;
    return k ? k > kFewK : p.top_p && p.top_p[i] < 1.0f;
  }
  // The row that a call of at most a row a thread takes in place of row c: the lengthy ones first, which are else
  // what the GPU ends with alone (64 rows of 128256, nine of them lengthy: 40 us as they are given, 42 with those
  // last, 31 so; 64 lengthy ones 63.5, without the order 62).  In a kernel of its own: the choice at run time cost a row alone
  // half a us.
  __device__ uint32_t long_first(uint32_t c, bool lengthy) {
    const uint32_t mask = __ballot_sync(0xFFFFFFFFu, lengthy);
    if (lane == 0) s.redu[0][warp] = __popc(mask);
    __syncthreads();
    const uint32_t of = lane < kWarps ? s.redu[0][lane] : 0, all = __reduce_add_sync(0xFFFFFFFFu, of);
    const uint32_t before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? of : 0) + __popc(mask & ((1u << lane) - 1));
    if (tid < p.n && (lengthy ? before : all + tid - before) == c) s.bin = tid;
    __syncthreads();
    return s.bin;
  }

  // what every CTA says, the same m in all its threads; valid until the call after the next
  __device__ const Msg *share(const Msg &m) {
    const uint32_t t = turn;
    turn ^= 1;
    if (tid < ctas) st_cluster(dsmem_addr(&s.msg[t][rank], tid), m);
    cluster_sync();
    return s.msg[t];
  }
  // sum of all CTAs' a, or b: in the order of a butterfly, the same everywhere
  __device__ double all_a(const Msg *all) const { return lanes_sum(lane < ctas ? all[lane].a : 0.0); }
  __device__ double all_b(const Msg *all) const { return lanes_sum(lane < ctas ? all[lane].b : 0.0); }
  __device__ uint32_t all_c(const Msg *all) const { return __reduce_add_sync(0xFFFFFFFFu, lane < ctas ? all[lane].c : 0); }
  // sums over the CTA, the same for all threads
  __device__ double sum(double v) {
    v = lanes_sum(v);
    __syncthreads();
    if (lane == 0) s.red[warp] = v;
    __syncthreads();
    return lanes_sum(lane < kWarps ? s.red[lane] : 0.0);
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
    read_sums(a, b, c, d);
  }
  __device__ void read_sums(uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) const {
    const uint32_t l = lane % kWarps;
    a = __reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? s.redu[0][l] : 0);
    b = __reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? s.redu[1][l] : 0);
    c = __reduce_min_sync(0xFFFFFFFFu, s.redu[2][l]);
    d = __reduce_max_sync(0xFFFFFFFFu, s.redu[3][l]);
  }
  // the same with the sums of x and y, in one exchange
  __device__ void sums(double &x, double &y, uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) {
    x = lanes_sum(x);
    y = lanes_sum(y);
    a = __reduce_add_sync(0xFFFFFFFFu, a);
    b = __reduce_add_sync(0xFFFFFFFFu, b);
    c = __reduce_min_sync(0xFFFFFFFFu, c);
    d = __reduce_max_sync(0xFFFFFFFFu, d);
    __syncthreads();
    if (lane == 0) {
      s.red[warp] = x;
      s.red2[warp] = y;
      s.redu[0][warp] = a;
      s.redu[1][warp] = b;
      s.redu[2][warp] = c;
      s.redu[3][warp] = d;
    }
    __syncthreads();
    x = lanes_sum(lane < kWarps ? s.red[lane] : 0.0);
    y = lanes_sum(lane < kWarps ? s.red2[lane] : 0.0);
    read_sums(a, b, c, d);
  }
  // inclusive sums over a warp's lanes
  __device__ double lanes_scan(double v) const {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= (uint32_t)o) v += y;
    }
    return v;
  }
  // inclusive sum over the CTA's threads, and the total
  __device__ double scan(double v, double &total) {
    v = lanes_scan(v);
    __syncthreads();
    if (lane == 31) s.red[warp] = v;
    __syncthreads();
    const double in = lanes_scan(lane < kWarps ? s.red[lane] : 0.0);
    total = __shfl_sync(0xFFFFFFFFu, in, kWarps - 1);
    const double before = __shfl_sync(0xFFFFFFFFu, in, (warp + 31) % 32);
    return warp ? before + v : v;
  }

  __device__ uint32_t bin_of(float zv) const { return min((uint32_t)zv, bins - 1); }  // (low may be a rounding beyond the last)
  __device__ void clear() {
    for (uint32_t i = tid; i < bins; i += kThreads) hist()[i] = 0;
    __syncthreads();
  }
  // histogram of the elements' counts
  __device__ void fill_counts() {
    clear();
    each<false>([&](float v, uint32_t) { atomicAdd(hist() + bin_of(z(v)), 1u); });
  }
  // of the masses of those kept, in f32 and without those beyond z_most, whose mass is returned
  template <bool CUT>
  __device__ double fill_masses(float z_most) {
    clear();
    const float unit = kOctaves / bins;
    float rest = 0.0f;
    each<CUT>([&](float v, uint32_t) {
      const float zv = z(v);
      if (zv > z_most) {
        rest += ex2(-zv * unit);
        return;
      }
      const uint32_t b = bin_of(zv);
      atomicAdd(hist() + b, __float2uint_rn(ex2(fmaf((float)b - zv, unit, 15.0f))));
    });
    return sum((double)rest);
  }
  // The cluster's sums over bins: each CTA takes a share of the bins, one a thread.  Returns that share's total.
  template <bool MASS>
  __device__ double reduce_bins() {
    static_assert(kCtaBins == kThreads, "a bin a thread");
    cluster_sync();
    const uint32_t b = rank * kCtaBins + tid;
    uint32_t h[kMaxCtas];
#pragma unroll
    for (uint32_t r = 0; r < kMaxCtas; ++r) h[r] = r < ctas ? ld_cluster32(dsmem_addr(hist() + b, r)) : 0;
    uint64_t t = 0;
#pragma unroll
    for (uint32_t r = 0; r < kMaxCtas; ++r) t += h[r];
    double v = (double)t, total;
    if (MASS) v *= exp2((double)b * (-(double)kOctaves / bins) - 15.0);  // counted in 2^-15 of the bin's largest weight
    binsum()[tid] = scan(v, total);
    return total;
  }
  // The first bins whose inclusive sums reach two targets (the last bin where none does): the CTA by what all
  // have said, then its warp and that one's lane, read from there by a warp for each target.  (Read whole
  // by every CTA, the 4 KB of that one CTA took 3 us.)
  __device__ void find_bins(const Msg *all, const double (&target)[2], uint32_t (&b)[2]) {
    if (warp < 2) {
      const double to = target[warp], of_cta = lane < ctas ? all[lane].a : 0.0, in = lanes_scan(of_cta);
      const uint32_t r = min((uint32_t)__popc(__ballot_sync(0xFFFFFFFFu, lane < ctas && in < to)), ctas - 1);
      const double before = __shfl_sync(0xFFFFFFFFu, in - of_cta, r);
      const double *far = binsum();
      auto at = [&](uint32_t i) { return before + __longlong_as_double((long long)ld_cluster64(dsmem_addr(far + i, r))); };
      const double ends = at(min(lane, kWarps - 1) * 32 + 31);
      const uint32_t w = min((uint32_t)__popc(__ballot_sync(0xFFFFFFFFu, lane < kWarps && ends < to)), kWarps - 1);
      const uint32_t l = min((uint32_t)__popc(__ballot_sync(0xFFFFFFFFu, at(w * 32 + lane) < to)), 31u);
      if (lane == 0) s.bins[warp] = r * kCtaBins + w * 32 + l;
    }
    __syncthreads();
    b[0] = s.bins[0];
    b[1] = s.bins[1];
    __syncthreads();
  }
  __device__ void note(uint32_t key, uint32_t id) {
    if (*reinterpret_cast<volatile uint32_t *>(&s.count) >= kList) return;  // a list that is full is of no use
    const uint32_t at = atomicAdd(&s.count, 1u);
    if (at < kList) list()[at] = (uint64_t)key << 32 | (uint32_t)~id;
  }
  // Sorts list[0 .. n) in descending order, entries all different but for zeros, which come last.  By buckets:
  // the high words' range is cut into 1024 parts, entries are placed by the sums over those, and within a
  // bucket by counting the larger ones; ten barriers.  Where a bucket is large (values that are equal, or nearly)
  // by the bitonic network, 55 steps for 1024.
  __device__ void sort(uint32_t n) {
    uint32_t *count = reinterpret_cast<uint32_t *>(binsum());  // [1024], of no other use by now
    static_assert(kCtaBins * 8 >= kSort * 4 && kSort == 2 * kThreads && kList >= 2 * kSort, "room to sort in");
    uint64_t e[2];
    uint32_t lo = 0xFFFFFFFFu, hi = 0, some = 0, o = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t i = tid + j * kThreads;
      e[j] = i < n ? list()[i] : 0;
      count[i] = 0;
      if (!e[j]) continue;
      ++some;
      lo = min(lo, (uint32_t)(e[j] >> 32));
      hi = max(hi, (uint32_t)(e[j] >> 32));
    }
    sums(some, o, lo, hi);
    const uint32_t shift = hi - lo < kSort ? 0 : 22 - __clz(hi - lo);  // (hi - lo) >> shift < 1024
    uint32_t at[2] = {0, 0}, order[2] = {0, 0}, most = 0;
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j)
      if (e[j]) order[j] = atomicAdd(count + (at[j] = (hi - (uint32_t)(e[j] >> 32)) >> shift), 1u);
    __syncthreads();
    const uint2 c = reinterpret_cast<const uint2 *>(count)[tid];
    most = __reduce_max_sync(0xFFFFFFFFu, max(c.x, c.y));
    uint32_t in = c.x + c.y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, in, d);
      if (lane >= (uint32_t)d) in += y;
    }
    if (lane == 31) {
      s.redu[0][warp] = in;
      s.redu[1][warp] = most;
    }
    __syncthreads();
    const uint32_t before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? s.redu[0][lane % kWarps] : 0);
    most = __reduce_max_sync(0xFFFFFFFFu, s.redu[1][lane % kWarps]);
    if (most <= 16) {
      in += before;
      reinterpret_cast<uint2 *>(count)[tid] = make_uint2(in - c.x - c.y, in - c.y);  // exclusive
      __syncthreads();
      uint64_t *part = list() + kSort;
      uint32_t first[2], end[2];
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) {
        first[j] = e[j] ? count[at[j]] : 0;
        end[j] = e[j] ? at[j] + 1 < kSort ? count[at[j] + 1] : some : 0;
        if (e[j]) part[first[j] + order[j]] = e[j];
        if (tid + j * kThreads < n) list()[tid + j * kThreads] = 0;
      }
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) {
        uint32_t place = first[j];
        for (uint32_t i = first[j]; i < end[j]; ++i) place += part[i] > e[j];
        if (e[j]) list()[place] = e[j];
      }
      __syncthreads();
      return;
    }
    uint32_t n2 = 2;
    while (n2 < n) n2 <<= 1;
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j)
      if (tid + j * kThreads < n2) list()[tid + j * kThreads] = e[j];  // zeros behind the last
    for (uint32_t k = 2; k <= n2; k <<= 1)
      for (uint32_t j = k >> 1; j; j >>= 1) {
        __syncthreads();
        if (tid < n2 / 2) {
          const uint32_t i = (tid / j) * 2 * j + tid % j;
          const uint64_t a = list()[i], b = list()[i + j];
          if ((a < b) == ((i & k) == 0)) {
            list()[i] = b;
            list()[i + j] = a;
          }
        }
      }
    __syncthreads();
  }
  // CTA 0 brings all CTAs' lists together in its own, sorted; true there.  After it
  // no CTA reads another's memory.  noted: of the lane's CTA.
  __device__ bool gather(uint32_t noted, uint32_t &n) {
    uint64_t mine[2] = {0, 0};
    if (lane >= ctas) noted = 0;
    n = __reduce_add_sync(0xFFFFFFFFu, noted);
    if (rank == 0) {
      uint32_t c[kMaxCtas];
#pragma unroll
      for (uint32_t r = 0; r < kMaxCtas; ++r) c[r] = __shfl_sync(0xFFFFFFFFu, noted, r);
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e) {
        uint32_t i = tid + e * kThreads, r = 0;
        if (i >= n) continue;
#pragma unroll
        for (uint32_t k = 0; k + 1 < kMaxCtas; ++k)
          if (r == k && i >= c[k]) i -= c[k], ++r;
        mine[e] = ld_cluster64(dsmem_addr(list() + i, r));
      }
    }
    cluster_sync();
    if (rank) return false;
    list()[tid] = mine[0];
    list()[tid + kThreads] = mine[1];
    sort(n);
    return true;
  }
  __device__ double list_weight(uint64_t e) const {
    const float v = key_float((uint32_t)(e >> 32));
    return e && v >= low ? weight(v) : 0.0;
  }

  __device__ void answer(uint32_t row, uint32_t id, double prob) {
    p.ids[row] = id;
    if (p.logprobs) p.logprobs[row] = (float)log(prob);
  }
  // The rest of a row whose candidates are all in CTA 0's sorted list: the first k of
  // them, of those the beginning with the mass p * whole (whole < 0: their own), min-p, the draw.
  __device__ void finish_list(uint32_t row, uint32_t n, uint32_t k, double pp, double whole, double min_p, double u) {
    const uint64_t e[2] = {list()[2 * tid], list()[2 * tid + 1]};
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
      const bool stay = i < min(n, k) && (i == 0 || pp >= 1.0 || before < target) && w[j] >= min_p && w[j] > 0;
      list()[i] = stay ? (e[j] & 0xFFFFFFFFull) << 32 | (uint32_t)(e[j] >> 32) : 0;  // (~id, value): by id
    }
    sort(n);
    const uint64_t f[2] = {list()[2 * tid], list()[2 * tid + 1]};
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

  // Notes this CTA's elements from the k-th largest of its threads' maxima on: what the row's first k are among.
  __device__ void note_largest(float best, uint32_t k) {
    const uint32_t key = key_of(best);
    const bool some = best > -INFINITY;
    uint32_t o1 = 0, have = some, lo = some ? key : 0xFFFFFFFFu, hi = key;
    sums(have, o1, lo, hi);
    if (have < k) lo = hi = 0;  // all there are
    while (lo < hi) {  // at least k maxima are not below lo
      const uint32_t mid = lo + (hi - lo + 1) / 2, n = __syncthreads_count(key >= mid);
      if (n >= k) lo = mid;
      else hi = mid - 1;
      if (n >= k && n <= k + k / 4 + 2) break;
    }
    const float from = lo ? key_float(lo) : -3.402823466e38f;
    if (tid == 0) s.count = 0;
    __syncthreads();
    for (uint32_t g = 0; g < groups; ++g) {
      float v[4];
      load(mine + 128 * g, v);
      if (fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) < from) continue;
      const uint32_t id = id0 + mine + 128 * g;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (v[j] >= from) note(key_of(v[j]), id + j);
    }
    __syncthreads();
  }
  // The row from what all CTAs noted, n together.
  __device__ void pick_largest(uint32_t row, const Msg *all, uint32_t n, uint32_t k, double pp, double min_p, double u) {
    constexpr uint32_t kPer = kList / kThreads;
    uint64_t e[kPer];
    if (rank == 0)
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j) {
        uint32_t i = tid + j * kThreads, r = 0;
        e[j] = 0;
        if (i >= n) continue;
        while (i >= all[r].d) i -= all[r++].d;
        e[j] = ld_cluster64(dsmem_addr(list() + i, r));
      }
    cluster_sync();
    if (rank) return;
    // a value that at least k are not below, and few more
    uint32_t lo = 0xFFFFFFFFu, hi = 0, o0 = 0, o1 = 0;
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j)
      if (e[j]) {
        lo = min(lo, (uint32_t)(e[j] >> 32));
        hi = max(hi, (uint32_t)(e[j] >> 32));
      }
    sums(o0, o1, lo, hi);
    while (n > 256 && lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      uint32_t c = 0;
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j)
        if (j * kThreads < n) c += __syncthreads_count((uint32_t)(e[j] >> 32) >= mid);
      if (c >= k) lo = mid;
      else hi = mid - 1;
      if (c >= k && c <= 256) break;
    }
    if (tid == 0) s.count = 0;
    for (uint32_t i = tid; i < kSort; i += kThreads) list()[i] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j)
      if (e[j] && (uint32_t)(e[j] >> 32) >= lo) {
        const uint32_t at = atomicAdd(&s.count, 1u);
        if (at < kSort) list()[at] = e[j];
      }
    __syncthreads();
    uint32_t m = s.count;
    __syncthreads();
    if (m > kSort) {  // equal values at the place: of those the lowest ids, the k largest entries
      uint64_t a = (uint64_t)lo << 32, b = (uint64_t)hi << 32 | 0xFFFFFFFFu;
      while (a < b) {
        const uint64_t mid = a + (b - a + 1) / 2;
        uint32_t c = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) c += __syncthreads_count(e[j] >= mid);
        if (c >= k) a = mid;
        else b = mid - 1;
        if (c == k) break;
      }
      if (tid == 0) s.count = 0;
      for (uint32_t i = tid; i < kSort; i += kThreads) list()[i] = 0;
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j)
        if (e[j] && e[j] >= a) list()[atomicAdd(&s.count, 1u)] = e[j];
      __syncthreads();
      m = s.count;
      __syncthreads();
    }
    sort(m);
    finish_list(row, m, k, pp, -1.0, min_p, u);
  }

  // mass of the thread's elements above `upto`, where a cut has formed it, and which of its elements were in the
  // cut's bracket (4 g + e of group g), where the groups are few enough
  double strict = 0;
  float upto = INFINITY;
  uint64_t marks = 0;
  __device__ bool marked() const { return groups <= 16; }

  // Finds the place of a cut whose bracket is the bins [b0, b1], the shortest beginning with a count of k or
  // (MASS) a mass of pp of the whole, and takes it over into cut_at and cut_id.  CUT: there is one already.
  // True: the row is finished (its elements up to b1 were few).
  template <bool MASS, bool CUT>
  __device__ bool cut(uint32_t row, uint32_t b0, uint32_t b1, uint32_t k, double pp, double min_p, double u) {
    if (tid == 0) s.count = 0;
    __syncthreads();
    // the bins b0 to b1 are z0 <= z < z1; the last one has all that is left
    const float z0 = (float)b0, z1 = b1 + 1 == bins ? INFINITY : (float)(b1 + 1);
    double a = 0, whole = -1.0, target = (double)k, every = 0;
    uint32_t above = 0, m = 0, kmin = 0xFFFFFFFFu, kmax = 0;
    uint64_t bit = 1;  // of the group's first element
    each4<CUT>([&](const float (&v)[4], const bool (&use)[4], uint32_t id) {
      double w[4];
      if (MASS) weights(v, w);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const float zv = z(v[j]);
        const bool over = use[j] && zv < z0;
        above += over;
        if (MASS) {
          if (use[j]) every += w[j];
          if (over) a += w[j];
          if (over && w[j] >= min_p) strict += w[j];
        }
        if (use[j] && !over && zv < z1) {
          const uint32_t key = key_of(v[j]);
          note(key, id + j);
          ++m;
          kmin = min(kmin, key);
          kmax = max(kmax, key);
          if (MASS) marks |= bit << j;
        }
      }
      bit <<= 4;
    });
    if (MASS) sums(a, every, above, m, kmin, kmax);
    else sums(above, m, kmin, kmax);
    const Msg *all = share(Msg{MASS ? a : (double)above, every, above + m, m, kmin, kmax});
    double A = all_a(all);
    if (MASS) {
      whole = all_b(all);
      target = pp * whole;
    }
    const uint32_t total = all_c(all), l = lane % ctas;
    m = __reduce_add_sync(0xFFFFFFFFu, lane < ctas ? all[lane].d : 0);
    kmin = __reduce_min_sync(0xFFFFFFFFu, all[l].e);
    kmax = __reduce_max_sync(0xFFFFFFFFu, all[l].f);
    if (total <= kSort) {  // all of them to the list
      each<CUT>([&](float v, uint32_t id) {
        if (z(v) < z0) note(key_of(v), id);
      });
      __syncthreads();
      all = share(Msg{0, 0, s.count, 0, 0, 0});
      uint32_t n;
      if (gather(all[l].c, n)) finish_list(row, n, MASS ? 0xFFFFFFFFu : k, pp, whole, min_p, u);
      return true;
    }
    const bool listed = m <= kSort;
    if (MASS) upto = key_float(kmax);
    // halve the range of values until the list holds it, or one value is left
    while (m > kSort && kmin < kmax) {
      const uint32_t mid = kmin + (kmax - kmin + 1) / 2;
      double b = 0;
      uint32_t up = 0, o1 = 0, o2 = 0, o3 = 0;
      each<CUT>([&](float v, uint32_t) {
        const uint32_t key = key_of(v);
        if (key < mid || key > kmax) return;
        ++up;
        if (MASS) b += weight(v);
      });
      sums(up, o1, o2, o3);
      if (MASS) b = sum(b);
      all = share(Msg{MASS ? b : (double)up, 0, up, 0, 0, 0});
      const double B = all_a(all);
      const uint32_t n = all_c(all);
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
      each<CUT>([&](float v, uint32_t) { own += key_of(v) == kmin; });
      // by ids: CTAs, warps, groups of a warp, lanes
      const uint32_t of_warp = __reduce_add_sync(0xFFFFFFFFu, own);
      sums(own, o1, o2, o3);  // leaves the warps' sums of `own`
      all = share(Msg{0, 0, own, 0, 0, 0});
      uint32_t before = 0, found = 0xFFFFFFFFu;
      for (uint32_t r = 0; r < rank; ++r) before += all[r].c;
      for (uint32_t i = 0; i < warp; ++i) before += s.redu[0][i];
      if (before < need && need <= before + of_warp)
        for (uint32_t g = 0; g < groups; ++g) {
          float e[4];
          load(mine + 128 * g, e);
          const uint32_t id = id0 + mine + 128 * g;
          bool yes[4];
          uint32_t n = 0;
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) n += yes[j] = kept<CUT>(e[j], id + j) && key_of(e[j]) == kmin;
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
      cut_at = key_float(kmin);
      cut_id = found;
      return false;
    }
    if (!listed) {
      if (tid == 0) s.count = 0;
      __syncthreads();
      each<CUT>([&](float v, uint32_t id) {
        const uint32_t key = key_of(v);
        if (key >= kmin && key <= kmax) note(key, id);
      });
      __syncthreads();
      all = share(Msg{0, 0, 0, s.count, 0, 0});
    }
    uint32_t n;
    Msg place{};
    if (gather(all[l].d, n)) {
      const uint64_t e[2] = {list()[2 * tid], list()[2 * tid + 1]};
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
      const uint64_t at = list()[s.bin];
      place.c = (uint32_t)(at >> 32);
      place.d = ~(uint32_t)at;
    }
    all = share(place);
    cut_at = key_float(all[0].c);
    cut_id = all[0].d;
    return false;
  }

  // The first lane up to which the sums of v exceed `at`, or (rounding) the last with any; `at` becomes
  // what is left of it there.  The same in all warps.
  __device__ uint32_t find_sum(double v, double &at) const {
    const double in = lanes_scan(v);
    const uint32_t over = __ballot_sync(0xFFFFFFFFu, v > 0 && in > at), some = __ballot_sync(0xFFFFFFFFu, v > 0);
    const uint32_t l = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : 0;
    at -= __shfl_sync(0xFFFFFFFFu, in - v, l);
    return l;
  }
  // the draw from what is kept, by id
  template <bool CUT>
  __device__ void draw(uint32_t row, double min_p, double u) {
    double own = strict;
    if (CUT && marked() && upto < INFINITY) {  // only what was in the bracket is left to look at
      for (uint64_t m = marks; m; m &= m - 1) {
        const uint32_t i = __ffsll((long long)m) - 1, at = mine + 128 * (i / 4) + i % 4;
        const float v = (float)x()[at];
        if (!kept<CUT>(v, id0 + at)) continue;
        const double w = weight(v);
        if (w >= min_p) own += w;
      }
    } else {
      each4<CUT>([&](const float (&v)[4], const bool (&use)[4], uint32_t) {
        bool add[4], any = false;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          add[j] = use[j] && !(CUT && v[j] > upto);  // those above are counted
          any |= add[j];
        }
        if (CUT && !any) return;
        double w[4];
        weights(v, w);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          if (add[j] && w[j] >= min_p) own += w[j];
      });
    }
    const Msg *all = share(Msg{sum(own), 0, 0, 0, 0, 0});  // the warps' sums stay in s.red
    const double M = all_a(all);
    double at = u * M;
    // the CTA with the token, then its warp
    if (rank != find_sum(lane < ctas ? all[lane].a : 0.0, at)) return;
    const uint32_t who = find_sum(lane < kWarps ? s.red[lane] : 0.0, at);
    // that warp's groups, one to each warp
    const uint32_t chunk = who * 128 * groups + 4 * lane;
    auto group = [&](uint32_t g, float (&v)[4], double (&w)[4]) {
      load(chunk + 128 * g, v);
      const uint32_t id = id0 + chunk + 128 * g;
      bool use[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) use[j] = kept<CUT>(v[j], id + j);
      weights(v, w);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (!use[j] || w[j] < min_p) w[j] = 0.0;
    };
    float v[4];
    double w[4];
    for (uint32_t g = warp; g < groups; g += kWarps) {
      group(g, v, w);
      const double t = lanes_sum((w[0] + w[1]) + (w[2] + w[3]));
      if (lane == 0) s.group[g] = t;
    }
    __syncthreads();
    const uint32_t g = find_sum(lane < groups ? s.group[lane] : 0.0, at);
    if (g % kWarps != warp) return;
    group(g, v, w);
    const double four = (w[0] + w[1]) + (w[2] + w[3]);
    const double in = lanes_scan(four);
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

// CTAs that fit on an SM.  Without top-k and top-p (CUTS) a row needs no lists, and in 16 bits 40 registers are
// enough for three (200 rows of 32000 in bf16: 18.4 us, with two 20.5); f32 rows, whose loads hold more, would spill
// (in a graph of calls 64 rows of 128256: 31.7 us with three, 25.0 with two; 200 of 32000: 22.2 and 19.8).
__host__ __device__ constexpr uint32_t ctas_an_sm(bool cuts, uint32_t elem_bytes) { return cuts || elem_bytes == 4 ? 2 : 3; }

// CUTS: top-k or top-p may be asked for.  LONG_FIRST: rows in another order than given.
template <typename T, bool CUTS, bool LONG_FIRST>
__global__ void __launch_bounds__(kThreads, ctas_an_sm(CUTS, sizeof(T))) k_sample_logits(const SampleParams p) {
  __shared__ Small s;
  const uint32_t ctas = p.ctas;
  Row<T> w(p, s);
  w.tid = threadIdx.x;
  w.lane = w.tid & 31;
  w.warp = w.tid >> 5;
  w.rank = cluster_ctarank();
  w.ctas = ctas;
  w.groups = p.groups;
  w.x_at = row_at<CUTS>(ctas);
  w.id0 = w.rank * p.slice;
  w.mine = w.warp * 128 * p.groups + 4 * w.lane;
  // the others' shared memory may be written once all have begun: waited for before the first time
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const bool lengthy = LONG_FIRST && w.lengthy(w.tid);
  s.power[w.tid] = exp2((double)w.tid / 512.0);
  const uint32_t row = LONG_FIRST ? w.long_first(blockIdx.x / ctas, lengthy) : blockIdx.x / ctas;
  const uint32_t at = p.rows ? p.rows[row] : row;
  if (at == FA_NO_TOKEN) return;
  // the row's own settings: on their way while the logits are read
  const float t = p.temperature ? p.temperature[row] : 1.0f, u = p.u[row], pp = CUTS && p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f;
  const uint32_t k = CUTS && p.top_k ? p.top_k[row] : 0;
  // the CTA's part of the row; behind its end -inf
  const uint32_t len = at < p.n_logits && w.id0 < p.vocab ? min(p.slice, p.vocab - w.id0) : 0, room = p.groups * kGroup;
  const T *src = reinterpret_cast<const T *>(p.logits) + (uint64_t)at * p.ld + w.id0;
  float mx = -INFINITY;
  constexpr uint32_t kV = 16 / sizeof(T);
  uint32_t i = 0;
  if (p.aligned) {
    const uint32_t whole = len / kV;
    constexpr uint32_t kAhead = sizeof(T) == 4 ? 8 : 4;  // loads in flight
    using T2 = typename Pair<T>::type;
    union Piece {
      uint4 u;
      T2 p[16 / sizeof(T2)];
    };
    T2 most = Pair<T>::none();
    for (uint32_t j0 = w.tid; j0 < whole; j0 += kAhead * kThreads) {
      Piece v[kAhead];
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
        if (j0 + a * kThreads < whole) v[a].u = *reinterpret_cast<const uint4 *>(src + (uint64_t)(j0 + a * kThreads) * kV);
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) {
        if (j0 + a * kThreads >= whole) break;
#pragma unroll
        for (uint32_t e = 0; e < 16 / sizeof(T2); ++e) most = larger(most, v[a].p[e]);
        *reinterpret_cast<uint4 *>(w.x() + (j0 + a * kThreads) * kV) = v[a].u;
      }
    }
    mx = Pair<T>::top(most);
    i = whole * kV;
  }
  for (uint32_t j = i + w.tid; j < room; j += kThreads) {
    const T f = j < len ? src[j] : (T)(-INFINITY);
    w.x()[j] = f;
    mx = fmaxf(mx, (float)f);
  }
  // a setting that does not hold leaves the row as it was (the same for all CTAs)
  if (at >= p.n_logits || !(t == 0.0f || (t >= 1e-6f && t <= 1e6f)) || !(u >= 0.0f && u < 1.0f) || !(pp >= 0.0f) || !(mp >= 0.0f && mp <= 1.0f)) {
    if (p.err && w.rank == 0 && w.tid == 0) atomicOr(p.err, kFlagRange);
    return;
  }
  bool few = CUTS && t > 0 && k && k < p.vocab && k <= kFewK;
  if (CUTS && few) {
    __syncthreads();
    w.note_largest(mx, k);
  }
  uint32_t o0 = 0, o1 = 0, o2 = 0, key = key_of(mx);
  w.sums(o0, o1, o2, key);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const Msg *all = w.share(Msg{0, 0, key, few ? s.count : 0, 0, 0});
  key = __reduce_max_sync(0xFFFFFFFFu, all[w.lane % ctas].c);
  const uint32_t noted = __reduce_add_sync(0xFFFFFFFFu, w.lane < ctas ? all[w.lane].d : 0);
  float top = key_float(key);
  if (top == -INFINITY) {  // no candidate at all
    if (w.rank == 0 && w.tid == 0) {
      p.ids[row] = FA_NO_TOKEN;
      if (p.logprobs) p.logprobs[row] = -INFINITY;
      if (p.err) atomicOr(p.err, kFlagRange);
    }
    return;
  }
  if (top == INFINITY) {  // counts as the largest f32: beside it nothing in 16 bits is a candidate
    few = false;
    for (uint32_t j = w.tid; j < room; j += kThreads) {
      const float f = (float)w.x()[j];
      if (sizeof(T) == 4) w.x()[j] = (T)(f == INFINITY ? 3.402823466e38f : f);
      else w.x()[j] = (T)(f == INFINITY ? 0.0f : -INFINITY);
    }
    top = sizeof(T) == 4 ? 3.402823466e38f : 0.0f;
    __syncthreads();
  }
  if (t == 0.0f) {  // the lowest id of the maximum
    uint32_t best = 0xFFFFFFFFu;
    for (uint32_t g = w.groups; g-- > 0;) {
      float v[4];
      w.load(w.mine + 128 * g, v);
#pragma unroll
      for (int j = 3; j >= 0; --j)
        if (v[j] == top) best = w.id0 + w.mine + 128 * g + j;
    }
    w.sums(o0, o1, best, o2);
    all = w.share(Msg{0, 0, best, 0, 0, 0});
    for (uint32_t r = 0; r < ctas; ++r) best = min(best, all[r].c);
    if (w.rank == 0 && w.tid == 0) w.answer(row, best, 1.0);
    return;
  }
  w.scale(top, t);
  if constexpr (CUTS) {
    if (few && noted < kList) {  // a CTA whose list ran over has at least kList
      w.pick_largest(row, all, noted, k, pp, mp, u);
      return;
    }
    bool has_cut = false;
    uint32_t b[2];
    if (k && k < p.vocab) {
      w.fill_counts();
      all = w.share(Msg{w.template reduce_bins<false>(), 0, 0, 0, 0, 0});
      if (w.all_a(all) > (double)k) {
        const double target[2] = {(double)k, (double)k};
        w.find_bins(all, target, b);
        if (w.template cut<false, false>(row, b[0], b[1], k, pp, mp, u)) return;
        has_cut = true;
      }
    }
    if (pp < 1.0f) {
      // all mass above z_most is less than half of what may be cut: the place is below it
      const float z_most = (log2f((float)p.vocab) - log2f(1.0f - pp) + 1.0f) * (w.bins / kOctaves);
      const double rest = has_cut ? w.template fill_masses<true>(z_most) : w.template fill_masses<false>(z_most);
      const double total = w.template reduce_bins<true>();
      all = w.share(Msg{total, rest, 0, 0, 0, 0});
      const double about = (double)pp * (w.all_a(all) + w.all_b(all));
      const double around[2] = {about * (1.0 - 3 * kHistError), about * (1.0 + 3 * kHistError)};
      w.find_bins(all, around, b);
      if (has_cut ? w.template cut<true, true>(row, b[0], b[1], 0, pp, mp, u) : w.template cut<true, false>(row, b[0], b[1], 0, pp, mp, u)) return;
      has_cut = true;
    }
    if (has_cut) {
      w.template draw<true>(row, (double)mp, (double)u);
      return;
    }
  }
  w.template draw<false>(row, (double)mp, (double)u);
}

template <typename T, bool CUTS, bool LONG_FIRST = false>
int launch(const SampleParams &p, cudaStream_t st) {
  const uint32_t smem = row_at<CUTS>(p.ctas) + p.groups * kGroup * (uint32_t)sizeof(T);
  if (cudaFuncSetAttribute(k_sample_logits<T, CUTS, LONG_FIRST>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleMaxSmem) != cudaSuccess) return -1;
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
  return cudaLaunchKernelEx(&cfg, k_sample_logits<T, CUTS, LONG_FIRST>, p) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_sample_logits(const SampleParams &in, uint32_t n_sm, cudaStream_t st) {
  SampleParams p = in;
  const uint32_t es = elem_size(p.dtype);
  auto groups = [&](uint32_t ctas) { return (p.vocab + ctas * kGroup - 1) / (ctas * kGroup); };
  // (in 16 bits more than kMostGroups of them go into shared memory)
  auto fits = [&](uint32_t ctas) { return groups(ctas) <= kMostGroups && region(ctas) + kCtaBins * 8 + groups(ctas) * kGroup * es <= kSampleMaxSmem; };
  p.ctas = 1;
  while (!fits(p.ctas)) p.ctas *= 2;
  // More CTAs to a row are shorter passes, but more barriers of clusters.  Rows whose times differ little (no cuts;
  // top-k, which mostly is small) take as many as run at once, where that goes: 64 rows of 128256 in bf16 without
  // cuts 20.5 us with 4 CTAs, 24.6 with 8; 200 of 32000 18.4 with 2, 20.1 with 1, 22.6 with 4; with top-k 17.5 with 1,
  // 26.7 with 2, 35.9 with 4.  Else as many as keep four an SM: 128 rows of 128256 in bf16 without cuts 33 with 4, 37
  // with 2; 64 in f32, cuts of all kinds, 31 with 8, 45 with 4; 200 of 32000 in bf16 35 with 2, 55 with 1, 41 with 4.
  const bool cuts = p.top_k || p.top_p;
  auto at_once = [&](uint32_t ctas) {
    const uint32_t smem = (cuts ? row_at<true>(ctas) : row_at<false>(ctas)) + groups(ctas) * kGroup * es + (uint32_t)sizeof(Small) + 1024;
    return std::min<uint32_t>(ctas_an_sm(cuts, es), 227 * 1024 / smem) * n_sm;
  };
  const uint32_t fewest = p.ctas;
  if (!p.top_p)
    for (uint32_t c = kMaxCtas; c >= fewest && p.ctas == fewest; c /= 2)
      if (p.n * c <= at_once(c) && (c == 1 || groups(c / 2) > 1)) p.ctas = c;
  if (p.top_p || p.n * p.ctas > at_once(p.ctas))
    while (p.ctas < kMaxCtas && groups(p.ctas) > 1 && p.n * p.ctas * 2 <= 4 * n_sm) p.ctas *= 2;
  p.groups = groups(p.ctas);
  p.slice = ((p.vocab + p.ctas - 1) / p.ctas + 15) / 16 * 16;
  static_assert(region(kMaxCtas) + kCtaBins * 8 + kSampleMaxVocab / kMaxCtas * 4 <= kSampleMaxSmem && kSampleMaxVocab % (kMaxCtas * kGroup) == 0 &&
                    kSampleMaxVocab / (kMaxCtas * kGroup) <= kMostGroups,
                "shared memory of the largest vocabulary");
  // Where not all rows run at once the lengthy ones are taken first; not where a row's answer is written over
  // settings that others have yet to look at.
  auto apart = [&](const void *out, const void *in) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(in), bytes = 4ull * p.n;
    return !out || !in || a + bytes <= b || b + bytes <= a;
  };
  bool clear = true;
  for (const void *out : {(const void *)p.ids, (const void *)p.logprobs, (const void *)p.err})
    for (const void *in : {(const void *)p.temperature, (const void *)p.top_k, (const void *)p.top_p}) clear = clear && apart(out, in);
  const bool first = cuts && clear && p.n <= kThreads && (uint64_t)p.n * p.ctas > 2 * n_sm;
  auto run = [&](auto x) {
    using T = decltype(x);
    return first ? launch<T, true, true>(p, st) : cuts ? launch<T, true>(p, st) : launch<T, false>(p, st);
  };
  return p.dtype == FA_KV_F32 ? run(0.0f) : p.dtype == FA_KV_F16 ? run(__half()) : run(__nv_bfloat16());
}

}  // namespace fa
