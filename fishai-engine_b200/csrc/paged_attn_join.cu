// Joins the pieces of attention items that were split between CTAs, and chooses
// the kernels of a call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>

#include "paged_tma.cuh"

namespace fa {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static std::mutex mu;
  static PFN_cuTensorMapEncodeTiled_v12000 f = nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (!f) {
    cudaDriverEntryPointQueryResult q;
    void *fn = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return nullptr;
    f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }
  return f;
}

__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// CTA x takes the item that CTA x of the launch before began and others
// finished.  A row's pieces (m_i, l_i, o_i) give
//   o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m),  m = max m_i,
// added in the order of the positions, four loads in flight.  Items of many
// rows, or of few pieces: a warp a row.  Few rows of many pieces (one long
// cache): the eight warps take the pieces in turn and their sums are added in
// order; with a warp to a whole row the 60 pieces of one 8192-position cache
// were one chain of loads: 44 us for 8 kv heads x 4 rows, against 6 us so.
constexpr uint32_t kJoinWarps = 8, kJoinFew = 8;

template <uint32_t kPer>
struct Sum {
  float m, l, acc[kPer];
};
// adds the pieces i0, i0 + step, .. i0 + 3 step of row r
template <uint32_t kPer, typename P>
__device__ __forceinline__ void add4(Sum<kPer> &s, P piece, uint32_t i0, uint32_t step, uint32_t n, uint32_t R, uint32_t r, uint32_t hd,
                                     uint32_t lane) {
  float2 ml[4];
  float x[4][kPer];
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const uint32_t i = i0 + k * step;
    const float *q = piece(i < n ? i : 0);
    ml[k] = i < n ? __ldcg(reinterpret_cast<const float2 *>(q + R * hd + 2 * r)) : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) x[k][j] = i < n && lane + 32 * j < hd ? __ldcg(q + r * hd + lane + 32 * j) : 0.0f;
  }
  const float mn = fmaxf(fmaxf(fmaxf(s.m, ml[0].x), fmaxf(ml[1].x, ml[2].x)), ml[3].x), ms = mn == -INFINITY ? 0.0f : mn;
  const float f = exp2f(s.m - ms);
  s.l *= f;
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) s.acc[j] *= f;
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const float e = exp2f(ml[k].x - ms);
    s.l = fmaf(ml[k].y, e, s.l);
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) s.acc[j] = fmaf(x[k][j], e, s.acc[j]);
  }
  s.m = mn;
}

// kPer: head elements of a lane (hd <= 32 kPer)
// An item of the launch for many rows: a thread has 16 elements of a row, as
// they lie in the slots (tc_part), and writes them as 32 bytes.
template <typename T>
__device__ __forceinline__ void join_tc(const AttnChunksParams &p, const float *part, const uint4 &d, uint32_t cta, uint32_t at, uint32_t R) {
  const uint32_t hd = p.pg.head_dim, head = d.z & 0xFFFF, rows = d.z >> 16;
  const uint32_t block = at * kJoinWarps + threadIdx.x / 32;  // (32 rows, 16 elements)
  const uint32_t r = block / (hd / 16) * 32 + threadIdx.x % 32, e0 = block % (hd / 16) * 16;
  if (r >= rows) return;
  const uint64_t slot = (uint64_t)R * (hd + 2);
  const float *first = part + ((uint64_t)cta * 2 + 1) * slot;
  float m = -INFINITY, l = 0.0f, acc[16] = {};
  // four pieces' loads in flight (one at a time took 19 us for the 17 pieces of
  // 128 rows over 8192 positions)
  for (uint32_t i0 = 0; i0 < d.w; i0 += 4) {
    float2 ml[4];
    float4 x[4][4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t i = min(i0 + k, d.w - 1);
      const float *q = i ? first + (2 * (uint64_t)i - 1) * slot : first;  // slot 1 of the CTA, then slot 0 of the next ones
      ml[k] = __ldcg(reinterpret_cast<const float2 *>(q + R * hd + 2 * r));
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) x[k][j] = __ldcg(reinterpret_cast<const float4 *>(q + tc_part(r, e0 + 4 * j, hd)));
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      if (i0 + k >= d.w) break;
      const float mn = fmaxf(m, ml[k].x), ms = mn == -INFINITY ? 0.0f : mn, f = exp2f(m - ms), e = exp2f(ml[k].x - ms);
      l = fmaf(l, f, ml[k].y * e);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        acc[4 * j] = fmaf(acc[4 * j], f, x[k][j].x * e);
        acc[4 * j + 1] = fmaf(acc[4 * j + 1], f, x[k][j].y * e);
        acc[4 * j + 2] = fmaf(acc[4 * j + 2], f, x[k][j].z * e);
        acc[4 * j + 3] = fmaf(acc[4 * j + 3], f, x[k][j].w * e);
      }
      m = mn;
    }
  }
  const uint32_t row = d.y + r;
  T *out = reinterpret_cast<T *>(p.out) + (uint64_t)(d.x + row / p.rep) * p.os + (head * p.rep + row % p.rep) * hd + e0;
  struct alignas(16) Out {
    T v[8];
  } o[2];
#pragma unroll
  for (uint32_t j = 0; j < 16; ++j) put(&o[j / 8].v[j % 8], l == 0.0f ? 0.0f : acc[j] / l);
  if (p.aligned) {
    reinterpret_cast<Out *>(out)[0] = o[0];
    reinterpret_cast<Out *>(out)[1] = o[1];
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) out[j] = o[j / 8].v[j % 8];
  }
}

template <typename T, uint32_t kPer>
__global__ void __launch_bounds__(kJoinWarps * 32) k_attn_join(const AttnChunksParams p, JoinSet a, JoinSet b) {
  __shared__ float part[kJoinWarps][32 * kPer];
  __shared__ float wm[kJoinWarps], wl[kJoinWarps];
  pdl_wait();
  const bool second = blockIdx.x >= a.ctas * a.parts;
  const uint32_t parts = second ? b.parts : a.parts, at = second ? blockIdx.x - a.ctas * a.parts : blockIdx.x;
  const uint32_t cta = at / parts, y = at % parts, R = a.R;
  const uint4 d = second ? b.desc[cta] : a.desc[cta];
  if (!d.w) return;
  if constexpr (sizeof(T) == 2 && kPer == 4) {
    if (second) {
      join_tc<T>(p, b.part, d, cta, y, b.R);
      return;
    }
  }
  const uint32_t hd = p.pg.head_dim, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = d.z & 0xFFFF, rows = d.z >> 16;
  const uint64_t slot = (uint64_t)R * (hd + 2);
  const float *first = a.part + ((uint64_t)cta * 2 + 1) * slot;
  // piece i: slot 1 of the CTA, then slot 0 of the next ones
  auto piece = [&](uint32_t i) { return i ? first + (2 * (uint64_t)i - 1) * slot : first; };
  auto out = [&](uint32_t r) {
    const uint32_t row = d.y + r;
    return reinterpret_cast<T *>(p.out) + (uint64_t)(d.x + row / p.rep) * p.os + (head * p.rep + row % p.rep) * hd;
  };
  if (d.w <= kJoinFew || rows > 16) {
    for (uint32_t r = y * kJoinWarps + warp; r < rows; r += parts * kJoinWarps) {
      Sum<kPer> s{-INFINITY, 0.0f, {}};
      for (uint32_t i = 0; i < d.w; i += 4) add4(s, piece, i, 1, d.w, R, r, hd, lane);
      T *o = out(r);
#pragma unroll
      for (uint32_t j = 0; j < kPer; ++j)
        if (lane + 32 * j < hd) put(o + lane + 32 * j, s.l == 0.0f ? 0.0f : s.acc[j] / s.l);
    }
    return;
  }
  for (uint32_t r = y; r < rows; r += parts) {
    Sum<kPer> s{-INFINITY, 0.0f, {}};
    for (uint32_t i = warp; i < d.w; i += 4 * kJoinWarps) add4(s, piece, i, kJoinWarps, d.w, R, r, hd, lane);
    __syncthreads();  // the row before has been read
    if (lane == 0) {
      wm[warp] = s.m;
      wl[warp] = s.l;
    }
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j)
      if (lane + 32 * j < hd) part[warp][lane + 32 * j] = s.acc[j];
    __syncthreads();
    float M = wm[0], L = 0.0f, e[kJoinWarps];
#pragma unroll
    for (uint32_t w = 1; w < kJoinWarps; ++w) M = fmaxf(M, wm[w]);
    const float Ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (uint32_t w = 0; w < kJoinWarps; ++w) {
      e[w] = exp2f(wm[w] - Ms);
      L = fmaf(wl[w], e[w], L);
    }
    T *o = out(r);
    for (uint32_t x = threadIdx.x; x < hd; x += kJoinWarps * 32) {
      float y = 0.0f;
#pragma unroll
      for (uint32_t w = 0; w < kJoinWarps; ++w) y = fmaf(part[w][x], e[w], y);
      put(o + x, L == 0.0f ? 0.0f : y / L);
    }
  }
}

template <typename T>
int launch_join(const AttnChunksParams &p, const JoinSet &a, const JoinSet &b, cudaStream_t st) {
  const dim3 grid(a.ctas * a.parts + b.ctas * b.parts), block(kJoinWarps * 32);
  return p.pg.head_dim <= 128 ? launch_pdl(k_attn_join<T, 4>, grid, block, 0, st, p, a, b)
                              : launch_pdl(k_attn_join<T, 8>, grid, block, 0, st, p, a, b);
}

constexpr size_t kSmallSlots = (size_t)2 * kAttnMaxCtas * kAttnMaxRows, kTcSlots = (size_t)2 * kTcMaxCtas * kTcRows;

}  // namespace

bool page_map(const AttnChunksParams &p, uint32_t rows, CUtensorMap *map) {
  const PFN_cuTensorMapEncodeTiled_v12000 encode = encoder();
  if (!encode) return false;
  const uint32_t es = elem_size(p.pg.dtype);
  const cuuint64_t dims[2] = {p.pg.head_dim, (cuuint64_t)p.pg.n_pages * 2 * p.pg.n_kv_heads * kPageLen}, strides[1] = {(cuuint64_t)p.pg.head_dim * es};
  const cuuint32_t box[2] = {64, rows}, one[2] = {1, 1};
  void *base = static_cast<char *>(p.pg.base) + (uint64_t)p.layer * p.pg.layer_stride * es;
  return encode(map, p.pg.dtype == FA_KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box,
                one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static std::atomic<uint32_t> g_withhold{0};
void attn_withhold(uint32_t copy) { g_withhold.store(copy, std::memory_order_relaxed); }

// slots of the launch for few rows, of the one for many, descriptors
size_t attn_chunks_ws(uint32_t head_dim) {
  return (kSmallSlots + kTcSlots) * (head_dim + 2) * 4 + (kAttnMaxCtas + 2 * kTcMaxCtas) * sizeof(uint4);
}

int launch_attn_chunks(const AttnChunksParams &p, void *ws, uint32_t n_sm, cudaStream_t st) {
  AttnChunksParams a = p, b = p;
  b.withhold = g_withhold.load(std::memory_order_relaxed);
  a.part = static_cast<float *>(ws);
  b.part = a.part + kSmallSlots * (p.pg.head_dim + 2);
  a.desc = reinterpret_cast<uint4 *>(b.part + kTcSlots * (p.pg.head_dim + 2));
  b.desc = a.desc + kAttnMaxCtas;
  a.rows_min = 1;
  a.rows_max = 0xFFFFFFFFu;
  JoinSet ja{a.part, a.desc, 0, 0, 0}, jb{b.part, b.desc, 0, 0, 0};
  const bool mma = attn_mma_takes(p), few = (uint64_t)p.max_q * p.rep <= 16;
  const int one = mma ? few ? launch_one_mma(a, st) : launch_short_mma(a, n_sm, st) : few ? launch_one_few(a, st) : launch_one_any(a, st);
  if (one <= 0) return one;
  if (mma) {
    // (Short calls have gone to launch_short_mma.)  Up to 16 rows mma.sync keeps up with the copies of K and V; above, the
    // items of tcgen05, also where they are mostly empty: 64 sequences of 4096
    // positions with 32 and 64 rows take 200 and 208 us, and took 264 and 316
    // with mma.sync and a warp for each 16 rows (which was the faster one over
    // short caches: 300 of 300 positions with 20 rows 129 us against 139).
    // Chunks of both kinds: both kernels, each leaving out the other's.  Where
    // all chunks are as long as the longest the second kernel takes them alone,
    // whatever their rows.
    const bool many = (uint64_t)p.max_q * p.rep > kMmaRows, alike = p.n_tokens == (uint64_t)p.n_chunks * p.max_q;
    if (many) a.rows_max = kMmaRows;
    if (!many || !alike) {
      ja.R = kMmaRows;
      if (!(ja.ctas = launch_attn_mma(a, n_sm, st))) return -1;
    }
    if (many) {
      b.rows_min = alike ? 1 : kMmaRows + 1;
      b.rows_max = 0xFFFFFFFFu;
      if (!(jb.ctas = launch_attn_tc(b, n_sm, !alike, st, &jb.R))) return -1;
      jb.parts = jb.R / 32 * (p.pg.head_dim / 16) / kJoinWarps;  // a thread 16 elements of a row
    }
  } else if (!(ja.ctas = few ? launch_attn_few(a, n_sm, st, &ja.R) : launch_attn_any(a, n_sm, st, &ja.R))) {
    return -1;
  }
  // CTAs to an item: a row each, for the few rows of one long cache
  const uint64_t rows = (uint64_t)p.max_q * p.rep;
  ja.parts = jb.ctas ? 2 : rows < 8 ? (uint32_t)rows : 8;
  switch (p.pg.dtype) {
    case FA_KV_F32: return launch_join<float>(p, ja, jb, st);
    case FA_KV_F16: return launch_join<__half>(p, ja, jb, st);
    default: return launch_join<__nv_bfloat16>(p, ja, jb, st);
  }
}

}  // namespace fa
