// Attention of chunks over paged f16 / bf16 K/V with many rows per kv head, on
// tcgen05 (head sizes 64 and 128).  Same mathematics as paged_attn_any.cu:
//   S = Q K^T,  P = 2^(scale S - m),  O += P V,  l += row sums of P,  O / l.
//
// The tensor pipe bounds it, and beside it the 16 exponentials a clock and SM:
// 128 x 128 scores take 512 clocks of MMA for S, 512 for P V (head size 128)
// and 1024 of exponentials.  So an item is 256 rows, two Q tiles of 128, and
// the tiles take turns: while one's scores are turned into weights, the tensor
// pipe works on the other's.  Rows are (token, query head of the kv head)
// pairs, so all query heads of a kv head share its K and V.
//
// (Chunks of up to 128 rows: one Q tile an item, softmax warps 0-3, the others
// from 4 on, two CTAs an SM.)
//   warps 0-3, 4-7   softmax of Q tile 0, 1: a thread a row.  Scores come from
//                    tensor memory, weights go back over them (16 bits, as V
//                    was rounded), read by the second MMA as its A operand.
//   warp 8           issues the MMAs (an elected lane); owns the tensor memory
//   warp 9           TMA: K and V tiles of 128 positions, a box per page of 16
//                    (pages that the item does not see start past the end of the
//                    tensor and arrive as zeros), 128-byte swizzle, a ring
//   warps 10, 11     copy the next item's Q rows (a row is a token and a head,
//                    so they are gathered) as soon as the last scores of the
//                    item before are formed
// Order of the MMAs per tile: P0 V, S0 of the next tile, P1 V, S1 of the next.
// They run in the order of issue, so S0 may overwrite P0 without a wait.
// 2048 tokens over 8192 positions, 32/8 heads x 128 f16: 367 thousand clocks, 222
// us at 1.63 GHz, the clock it was captured at (1.08 PFLOP/s; tensor pipe 56%,
// special-function pipe 56%), and 14 us for the join.
// The reference point m of a row only moves when a maximum exceeds it by 2^8:
// weights stay below 2^8 and sums in f32 are exact to the same relative error,
// and the output in tensor memory is rescaled only then (by the softmax warps,
// after the P V before it is done).  In f16 the weights and their sums are 2^7
// times that, up to 2^15: they keep their full precision down to 2^-21 of the
// largest (paged_attn_mma.cu).
// Waits are bounded; one that runs out sets an abort flag that the others see,
// and the kernel drains its copies and MMAs, frees the tensor memory and sets
// FA_FLAG_TIMEOUT.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_tma.cuh"

namespace fa {
namespace {

constexpr uint32_t kTcPos = 128;

// G Q tiles to an item
template <uint32_t HD, uint32_t G>
struct TcCfg {
  static constexpr uint32_t kThreads = 128 * G + 128, kRows = 128 * G;
  static constexpr uint32_t kHalf = kTcPos * 128;           // 128 positions (or rows) x 64 elements
  static constexpr uint32_t kTile = kHalf * (HD / 64);      // one of K, V, or a Q tile
  static constexpr uint32_t kStages = HD == 128 ? (G == 2 ? 5 : 2) : (G == 2 ? 8 : 5);
  static constexpr uint32_t kBarOff = G * kTile + kStages * kTile;
  static constexpr uint32_t kSmem = 1024 + kBarOff + 512;   // alignment, barriers
  static_assert(kSmem <= (G == 2 ? 227 : 113) * 1024, "shared memory of a CTA");
  static constexpr uint32_t kTmem = 256 * G;
};
template <uint32_t G>
using TcWalk = Walk<128 * G, kTcPos, 3, 128 * G + 128>;  // an item costs some 5 us beside its tiles of 1.9
struct TcBars {
  uint64_t full[8], empty[8], q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], o_full[2], done;
  uint64_t red[384 / 32 + 2];
  uint32_t tmem, abort, fills;
};
static_assert(sizeof(TcBars) <= 512, "barrier space");

// tensor memory columns: scores (and weights over them) of tile i, outputs
template <uint32_t G>
__device__ __forceinline__ uint32_t s_col(uint32_t i) { return 128 * i; }
template <uint32_t G>
__device__ __forceinline__ uint32_t o_col(uint32_t i) { return 128 * (G + i); }

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Descriptor of a shared-memory operand with 128-byte swizzle: 8-row groups
// 1024 bytes apart, `lead` bytes between blocks of 64 elements (rows-contiguous
// operand V) or unused (K, Q).  The address is in the low word, so a tile's
// descriptors differ by an addition there.
__device__ __forceinline__ uint32_t sdesc_lo(uint32_t addr, uint32_t lead) { return ((addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16); }
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t sdesc(uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(kDescHi));
  return d;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void ld32(uint32_t addr, float *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
        "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
        "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
      "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
               "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp; below 2^-126: 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (__is_same(T, __half)) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}

// two f32 in a register pair
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Weights 2^(scale x - m) of 32 scores: 16 packed pairs, their sums added to
// `sum`.  (A polynomial on the FMA pipes for 3 of 8 pairs, to unburden the
// special-function unit, was slower: 2048 rows over 16384 positions 495 us
// against 472; the chain of instructions of a row counts for more.)
template <typename T>
__device__ __forceinline__ void weights32(const float *x, uint64_t scale, uint64_t minus_m, uint64_t (&sum)[2], uint32_t (&pk)[16]) {
#pragma unroll
  for (uint32_t c = 0; c < 16; ++c) {
    float a, b;
    unpair(fma2(pair(x[2 * c], x[2 * c + 1]), scale, minus_m), a, b);
    a = ex2(a);
    b = ex2(b);
    sum[c & 1] = add2(sum[c & 1], pair(a, b));
    pk[c] = pack2<T>(a, b);
  }
}

// Q rows [first, first + 128) of the item to a swizzled tile, 64 threads; rows
// past the item's are zeros
template <typename T, uint32_t HD>
__device__ __forceinline__ void load_q(const AttnChunksParams &p, const Segment &s, uint32_t first, uint32_t tile, uint32_t tid) {
  constexpr uint32_t CH = HD / 8, kStep = 64 / CH;  // pieces of a row; rows between a thread's pieces
  const uint32_t c = tid % CH, r0 = tid / CH;
  // row -> (token, head of the group), carried along: a division a piece made
  // these two warps the slowest part of short items
  const uint32_t rep = p.rep, dt = kStep / rep, dh = kStep - dt * rep;
  uint32_t tok = (first + r0) / rep, h = first + r0 - tok * rep;
  const T *base = reinterpret_cast<const T *>(p.q) + (uint64_t)s.chunk.q0 * p.qs + s.head * rep * HD + c * 8;
  const uint32_t rows = s.r1 - first;
#pragma unroll 8
  for (uint32_t r = r0; r < 128; r += kStep) {
    const bool live = r < rows;
    const T *x = live ? base + tok * p.qs + h * HD : base;
    const uint32_t dst = tile + (c >> 3) * (kTcPos * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    if (p.aligned) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(x), "r"(live ? 16u : 0u) : "memory");
    } else {
      const uint16_t *y = reinterpret_cast<const uint16_t *>(x);
      uint32_t v[4] = {};
      if (live)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = y[2 * i] | (uint32_t)y[2 * i + 1] << 16;
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
    }
    tok += dt;
    h += dh;
    if (h >= rep) {
      h -= rep;
      ++tok;
    }
  }
}

template <typename T, uint32_t HD, uint32_t G, typename PR>
__device__ void q_role(const PR &p, TcWalk<G> w, TcBars &b, uint32_t smem) {
  const uint32_t tid = threadIdx.x & 63;
  uint32_t n[2] = {0, 0};  // fills of each tile so far
  for (Segment s; w.next(p, s);) {
    if (s.hi <= s.lo) continue;
#pragma unroll
    for (uint32_t g = 0; g < G; ++g) {
      if (s.r0 + 128 * g >= s.r1) break;
      if (!wait_bar(&b.abort, &b.q_empty[g], (n[g] & 1) ^ 1)) return;
      load_q<T, HD>(p, s, s.r0 + 128 * g, smem + g * TcCfg<HD, G>::kTile, tid);
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      mbar_arrive(&b.q_full[g]);
      ++n[g];
    }
  }
}

// 32 bytes of a thread's row (aligned to 32)
__device__ __forceinline__ void st8(void *p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}

template <typename T, uint32_t HD, uint32_t G, typename PR>
__device__ void softmax_role(const PR &p, TcWalk<G> w, TcBars &b, uint32_t tmem, uint32_t g) {
  const uint32_t tid = threadIdx.x & 127, warp = tid >> 5;
  const uint32_t lanes = tmem + ((warp * 32) << 16);
  uint32_t n = 0;  // tiles of this group so far
  for (Segment s; w.next(p, s);) {
    const uint32_t row = s.r0 + 128 * g + tid;
    if (s.r0 + 128 * g >= s.r1) continue;  // the second Q tile is empty
    const bool live = row < s.r1, whole = TcWalk<G>::whole(s);
    const int32_t pos = s.chunk.first + (int32_t)(row / p.rep);
    // a warp past the item's last row only hands its (unused) rows on; within a
    // warp such rows ask for no masks
    const bool idle = row - tid % 32 >= s.r1;
    const uint32_t tiles = s.hi > s.lo ? s.u1 - s.u0 : 0;
    float m = -INFINITY, l = 0.0f;
    for (uint32_t k = 0; k < tiles; ++k, ++n) {
      // column c of the tile is position t0 + c; with first positions, its columns below `keep` are those
      uint32_t t0;
      int32_t keep = 0;
      if constexpr (PR::packed) {
        constexpr uint32_t kPages = kTcPos / kPageLen;
        const uint32_t n = sink_units<kPageLen>(p, s.lo), j = (s.u0 + k) * kPages;
        t0 = (s.lo / kPageLen + j - n) * kPageLen;
        keep = (int32_t)p.sinks - (int32_t)(j * kPageLen);
        if (n < s.lo / kPageLen) keep = min(keep, (int32_t)((n - min(n, j)) * kPageLen));  // the window's pages are elsewhere
      } else {
        t0 = unit_at<kTcPos>(p, s.lo, s.u0 + k);
      }
      if (!wait_bar(&b.abort, &b.s_full[g], n & 1)) return;
      if (idle) {
        mbar_arrive(&b.p_half[g]);
        mbar_arrive(&b.p_full[g]);
        continue;
      }
      fence_after();
      float x[kTcPos];
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) ld32(lanes + s_col<G>(g) + 32 * c, x + 32 * c);
      wait_ld();
      // rows of a warp that see all 128 positions need no mask
      const int32_t to = pos - (int32_t)t0 + 1;  // visible columns: [to - window, to)
      if (!__all_sync(0xFFFFFFFFu, !live || to >= (int32_t)kTcPos)) {
#pragma unroll
        for (int32_t c = 0; c < (int32_t)kTcPos; ++c)
          if (c >= to) x[c] = -INFINITY;
      }
      if (p.window && !__all_sync(0xFFFFFFFFu, !live || to <= (int32_t)p.window)) {
        const int32_t from = to - (int32_t)p.window;
        if (keep <= 0) {
#pragma unroll
          for (int32_t c = 0; c < (int32_t)kTcPos; ++c)
            if (c < from) x[c] = -INFINITY;
        } else if (keep < (int32_t)kTcPos) {
#pragma unroll
          for (int32_t c = 0; c < (int32_t)kTcPos; ++c)
            if (c < from && c >= keep) x[c] = -INFINITY;
        }
      }
      float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (uint32_t c = 4; c + 8 <= kTcPos; c += 8)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], fmaxf(x[c + e], x[c + 4 + e]));
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], x[kTcPos - 4 + e]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      float f = 1.0f;
      if (top > m + 8.0f) {
        f = ex2(m - top);
        m = top;
        l *= f;
      }
      if (k && __any_sync(0xFFFFFFFFu, f != 1.0f)) {
        if (!wait_bar(&b.abort, &b.o_full[g], (n - 1) & 1)) return;
        fence_after();
#pragma unroll 1
        for (uint32_t c = 0; c < HD; c += 32) {
          float o[32];
          ld32(lanes + o_col<G>(g) + c, o);
          wait_ld();
#pragma unroll
          for (uint32_t e = 0; e < 32; ++e) o[e] *= f;
          st32(lanes + o_col<G>(g) + c, reinterpret_cast<const uint32_t *>(o));
        }
      }
      const float ms = m == -INFINITY ? 0.0f : m;
      constexpr float kLift = __is_same(T, __half) ? 7.0f : 0.0f;
      const uint64_t scale = pair(p.scale_log2, p.scale_log2), minus_m = pair(kLift - ms, kLift - ms);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (uint32_t h = 0; h < 4; ++h) {
        uint32_t pk[16];
        weights32<T>(x + 32 * h, scale, minus_m, sum, pk);
        if (h == 2) {  // the first half is stored by now (and a rescaled output): its product with V begins
          wait_st();
          fence_before();
          mbar_arrive(&b.p_half[g]);
        }
        st16(lanes + s_col<G>(g) + 16 * h, pk);
      }
      wait_st();
      fence_before();
      mbar_arrive(&b.p_full[g]);
      float s0, s1, s2, s3;
      unpair(sum[0], s0, s1);
      unpair(sum[1], s2, s3);
      l += (s0 + s1) + (s2 + s3);
    }
    float *slot = TcWalk<G>::slot(p, s);
    const uint32_t r = row - s.r0, tok = row / p.rep;
    T *out = reinterpret_cast<T *>(p.out) + (uint64_t)(s.chunk.q0 + tok) * p.os + (s.head * p.rep + row - tok * p.rep) * HD;
    if (tiles) {
      if (!wait_bar(&b.abort, &b.o_full[g], (n - 1) & 1)) return;
      fence_after();
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
    for (uint32_t c = 0; c < HD; c += 32) {
      float o[32];
      if (tiles) {
        ld32(lanes + o_col<G>(g) + c, o);
        wait_ld();
      }
      if (l == 0.0f) {  // nothing seen (yet, within a split item): zeros, whatever the product left
#pragma unroll
        for (uint32_t e = 0; e < 32; ++e) o[e] = 0.0f;
      }
      if (!live) continue;
      if (!whole) {  // [32 rows][4 elements] blocks: a warp's store is 512 bytes in a row
#pragma unroll
        for (uint32_t e = 0; e < 32; e += 4)
          *reinterpret_cast<float4 *>(slot + tc_part(r, c + e, HD)) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        continue;
      }
#pragma unroll
      for (uint32_t q = 0; q < 32; q += 16) {
        uint32_t v[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = pack2<T>(o[q + 2 * e] * inv, o[q + 2 * e + 1] * inv);
        if (reinterpret_cast<uintptr_t>(out) % 32 == 0) {
          st8(out + c + q, v);
        } else {
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e) {
            reinterpret_cast<uint16_t *>(out)[c + q + 2 * e] = (uint16_t)v[e];
            reinterpret_cast<uint16_t *>(out)[c + q + 2 * e + 1] = (uint16_t)(v[e] >> 16);
          }
        }
      }
    }
    if (!whole && live) *reinterpret_cast<float2 *>(slot + 128 * G * HD + 2 * r) = make_float2(m, l);
    if (!whole && s.u0 == 0 && g == 0 && tid == 0) p.desc[blockIdx.x] = w.describe(s);
    fence_before();  // the next item's MMAs follow its q_full and p_full arrivals
  }
}

template <typename T, uint32_t HD, uint32_t G, typename PR>
__device__ void mma_role(const PR &p, TcWalk<G> w, TcBars &b, uint32_t smem, uint32_t tmem, uint32_t lead) {
  using C = TcCfg<HD, G>;
  constexpr uint32_t kType = __is_same(T, __half) ? 0u : 1u;  // f16 / bf16, A and B
  constexpr uint32_t kS = (1u << 4) | (kType << 7) | (kType << 10) | ((kTcPos / 8) << 17) | ((128 / 16) << 24);
  constexpr uint32_t kO = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | ((HD / 8) << 17) | ((128 / 16) << 24);  // B = V: rows are K
  // The warp stays together and one elected lane issues: with the whole loop in
  // one lane the operands' way into uniform registers made each MMA take some
  // 130 clocks to issue (637 us for 2048 rows over 16384 positions, 495 so).
  // Ring places and phases are counted on.
  const uint32_t q_lo = sdesc_lo(smem, 16), k_lo = sdesc_lo(smem + G * C::kTile, 16), v_lo = sdesc_lo(smem + G * C::kTile, C::kHalf);
  struct Place {  // of a fill in the ring (fills come K0 V0 K1 V1 ..)
    uint32_t st, ph;
    __device__ void step() {
      if (++st == C::kStages) {
        st = 0;
        ph ^= 1;
      }
    }
  } at{0, 0};
  uint32_t n[2] = {0, 0}, q_phase[2] = {0, 0};
  auto scores = [&](uint32_t g, uint32_t st) {
    const uint32_t q = q_lo + g * (C::kTile >> 4), k = k_lo + st * (C::kTile >> 4);
    if (lead) {
#pragma unroll
      for (uint32_t kk = 0; kk < HD / 16; ++kk) {
        const uint32_t off = kk / 4 * (C::kHalf >> 4) + kk % 4 * 2;
        mma_ss(tmem + s_col<G>(g), sdesc(q + off), sdesc(k + off), kS, kk);
      }
      commit(&b.s_full[g]);
    }
    __syncwarp();
  };
  for (Segment s; w.next(p, s);) {
    const uint32_t tiles = s.hi > s.lo ? s.u1 - s.u0 : 0, groups = G == 2 && s.r1 - s.r0 > 128 ? 2 : 1;
    if (!tiles) continue;
    if (!wait_bar(&b.abort, &b.full[at.st], at.ph)) return;
    for (uint32_t g = 0; g < groups; ++g) {
      if (!wait_bar(&b.abort, &b.q_full[g], q_phase[g])) return;
      q_phase[g] ^= 1;
      fence_after();
      scores(g, at.st);
      if (tiles == 1 && lead) commit(&b.q_empty[g]);
    }
    if (lead) commit(&b.empty[at.st]);
    at.step();
    for (uint32_t k = 0; k < tiles; ++k) {
      const Place v = at;
      at.step();
      const Place next = at;
      const bool more = k + 1 < tiles;
      if (more) at.step();
      if (!wait_bar(&b.abort, &b.full[v.st], v.ph)) return;
      const uint32_t vt = v_lo + v.st * (C::kTile >> 4);
      for (uint32_t g = 0; g < groups; ++g) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          if (!wait_bar(&b.abort, h ? &b.p_full[g] : &b.p_half[g], n[g] & 1)) return;
          fence_after();
          if (lead) {
#pragma unroll
            for (uint32_t kk = 4 * h; kk < 4 * h + 4; ++kk)
              mma_ts(tmem + o_col<G>(g), tmem + s_col<G>(g) + 8 * kk, sdesc(vt + kk * (2048 >> 4)), kO, k || kk);
          }
        }
        ++n[g];
        if (lead) commit(&b.o_full[g]);
        if (g + 1 == groups && lead) commit(&b.empty[v.st]);
        if (more) {
          if (g == 0 && !wait_bar(&b.abort, &b.full[next.st], next.ph)) return;
          scores(g, next.st);
          if (k + 2 == tiles && lead) commit(&b.q_empty[g]);  // the item's last scores
        }
      }
      if (more && lead) commit(&b.empty[next.st]);
    }
  }
}

// one warp; fills: how many it began
template <typename T, uint32_t HD, uint32_t G, typename PR>
__device__ void load_role(const PR &p, TcWalk<G> w, TcBars &b, uint32_t smem, const CUtensorMap *map, const CUtensorMap *row_map,
                          uint32_t &fills) {
  using C = TcCfg<HD, G>;
  const uint32_t lane = threadIdx.x & 31, ring = smem + G * C::kTile;
  uint32_t st = 0, ph = 1;
  for (Segment s; w.next(p, s);) {
    const uint32_t tiles = s.hi > s.lo ? s.u1 - s.u0 : 0;
    const uint32_t *pt = p.pg.page_table + (uint64_t)s.chunk.seq * p.pg.max_pages;
    auto look_up = [&](uint32_t t) -> uint32_t {
      return item_reads(p, s.lo, s.hi, t) ? __ldg(pt + t / kPageLen) : 0xFFFFFFFFu;
    };
    uint32_t next = unit_page<kTcPos>(p, s.lo, s.u0, lane & 7);  // where the lane's page of the tile begins
    uint32_t ahead = tiles ? look_up(next) : 0;
    for (uint32_t k = 0; k < tiles; ++k) {
      const uint32_t page = ahead, at = next;
      next = PR::packed ? unit_page<kTcPos>(p, s.lo, s.u0 + k + 1, lane & 7) : at + kTcPos;
      if (k + 1 < tiles) ahead = look_up(next);
      const bool used = item_reads(p, s.lo, s.hi, at);
      if (used && page >= p.pg.n_pages && p.err) atomicOr(p.err, kFlagPage);
      // A page with slots that nobody sees: V must not be NaN there (its weight 0
      // would not help), so its rows come one by one, the unseen ones from past
      // the end of the tensor, as zeros.
      const bool part = used && (at + kPageLen > s.hi || (at < s.lo && at + kPageLen > p.sinks));
      const uint32_t parts = __ballot_sync(0xFFFFFFFFu, part && lane < 8);
      for (uint32_t is_v = 0; is_v < 2; ++is_v) {
        const uint32_t dst = ring + st * C::kTile;
        if (!wait_bar(&b.abort, &b.empty[st], ph)) return;
        const bool go = fills + 1 != p.withhold;
        if (go && lane == 0) mbar_arrive_expect_tx(&b.full[st], C::kTile);
        __syncwarp();
        if (go && lane < 8 * (HD / 64) && !(is_v && part))
          tma_2d(dst + (lane >> 3) * C::kHalf + (lane & 7) * 2048, map, (int32_t)(lane >> 3) * 64, map_row(p.pg, page, is_v, s.head), &b.full[st]);
        if (go && is_v)
          for (uint32_t m = parts; m; m &= m - 1) {
            const uint32_t j = __ffs(m) - 1, pg = __shfl_sync(0xFFFFFFFFu, page, j), t = __shfl_sync(0xFFFFFFFFu, at, j) + (lane & 15), half = lane >> 4;
            const bool seen = item_sees(p, s.lo, s.hi, t);
            if (half < HD / 64)
              tma_2d(dst + half * C::kHalf + j * 2048 + (lane & 15) * 128, row_map, (int32_t)half * 64,
                     map_row(p.pg, seen ? pg : 0xFFFFFFFFu, 1, s.head) + (int32_t)(seen && pg < p.pg.n_pages ? lane & 15 : 0), &b.full[st]);
          }
        ++fills;
        if (++st == C::kStages) {
          st = 0;
          ph ^= 1;
        }
      }
    }
  }
}

template <typename T, uint32_t HD, uint32_t G, typename PR>
__global__ void __launch_bounds__(128 * G + 128, 3 - G) k_attn_tc(const PR p, const __grid_constant__ CUtensorMap map,
                                                            const __grid_constant__ CUtensorMap row_map) {
  using C = TcCfg<HD, G>;
  extern __shared__ __align__(1024) uint8_t raw[];
  const uint32_t pad = (1024u - (smem_u32(raw) & 1023u)) & 1023u, smem = smem_u32(raw) + pad;
  TcBars &b = *reinterpret_cast<TcBars *>(raw + pad + C::kBarOff);
  const uint32_t tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&row_map) : "memory");
  }
  TcWalk<G> w;
  w.start(p, 4, b.red);
  if (tid == 0) {
    p.desc[blockIdx.x].w = 0;
    for (uint32_t i = 0; i < C::kStages; ++i) {
      mbar_init(&b.full[i], 1);
      mbar_init(&b.empty[i], 1);
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&b.q_full[i], 64);
      mbar_init(&b.q_empty[i], 1);
      mbar_init(&b.s_full[i], 1);
      mbar_init(&b.p_half[i], 128);
      mbar_init(&b.p_full[i], 128);
      mbar_init(&b.o_full[i], 1);
    }
    mbar_init(&b.done, 1);
    b.abort = b.fills = 0;
    fence_mbar_init();
  }
  const bool any = !w.done();  // the same for the CTA
  if (any) {
    if (warp == 4 * G) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&b.tmem)), "r"(C::kTmem));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = b.tmem;
    // registers at launch: 384 x 168 = 256 x 224 + 128 x 56, or 256 x 128 =
    // 128 x 200 + 128 x 56
    if (warp < 4 * G) {
      if constexpr (G == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
      else asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
      softmax_role<T, HD, G>(p, w, b, tmem, warp >> 2);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
      if (warp == 4 * G) {
        uint32_t lead;  // issues the MMAs and the commits, which follow only its own MMAs
        asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(lead));
        mma_role<T, HD, G>(p, w, b, smem, tmem, lead);
        __syncwarp();
        if (lead) commit(&b.done);
        __syncwarp();
        mbar_wait_sleep(&b.done, 0);  // nothing is on its way to tensor memory after this
      } else if (warp == 4 * G + 1) {
        uint32_t fills = 0;
        load_role<T, HD, G>(p, w, b, smem, &map, &row_map, fills);
        b.fills = fills;
      } else {
        q_role<T, HD, G>(p, w, b, smem);
      }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (tid == 0 && b.abort && p.err) atomicOr(p.err, kFlagTimeout);
    // Copies that nobody waited for have to land before the CTA ends.  Whether
    // there are any is known only now: a wait may run out after the last copy has
    // begun.  (Their number stored at each copy instead: 242 -> 248 us for 2048
    // tokens over 8192 positions.)
    if (warp == 4 * G + 1 && b.abort)
      for (uint32_t n = b.fills, i = n > C::kStages ? n - C::kStages : 0; i < n; ++i)
        if (i + 1 != p.withhold) mbar_wait_sleep(&b.full[i % C::kStages], i / C::kStages & 1);
    if (warp == 4 * G) {
      fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem));
    }
  }
  pdl_wait();  // the launch before this one, with which it may have overlapped: the join waits for this one only
}

template <typename T, uint32_t HD, uint32_t G>
uint32_t launch_g(const AttnChunksParams &p, uint32_t n_sm, bool overlap, cudaStream_t st) {
  using C = TcCfg<HD, G>;
  CUtensorMap map, row_map;
  if (!page_map(p, kPageLen, &map) || !page_map(p, 1, &row_map)) return 0;
  const uint32_t ctas = (n_sm < kTcMaxCtas ? n_sm : kTcMaxCtas) * (3 - G);  // one or two an SM
  return with_sinks<PackedParams>(p, [&](auto a) -> uint32_t {
    using PR = decltype(a);
    if (cudaFuncSetAttribute(k_attn_tc<T, HD, G, PR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem) != cudaSuccess) return 0;
    if (overlap) return launch_pdl(k_attn_tc<T, HD, G, PR>, dim3(ctas), dim3(C::kThreads), C::kSmem, st, a, map, row_map) ? 0 : ctas;
    k_attn_tc<T, HD, G><<<ctas, C::kThreads, C::kSmem, st>>>(a, map, row_map);
    return cudaGetLastError() == cudaSuccess ? ctas : 0;
  });
}
template <typename T>
uint32_t launch_t(const AttnChunksParams &p, uint32_t n_sm, bool overlap, cudaStream_t st, uint32_t *R) {
  // No chunk above 128 rows: items of one Q tile, two CTAs an SM, which hide one
  // another's waits as the two Q tiles of a longer chunk's item do
  const bool one = (uint64_t)p.max_q * p.rep <= 128;
  *R = one ? 128 : 256;
  if (p.pg.head_dim == 64) return one ? launch_g<T, 64, 1>(p, n_sm, overlap, st) : launch_g<T, 64, 2>(p, n_sm, overlap, st);
  return one ? launch_g<T, 128, 1>(p, n_sm, overlap, st) : launch_g<T, 128, 2>(p, n_sm, overlap, st);
}

}  // namespace

uint32_t launch_attn_tc(const AttnChunksParams &p, uint32_t n_sm, bool overlap, cudaStream_t st, uint32_t *R) {
  return p.pg.dtype == FA_KV_F16 ? launch_t<__half>(p, n_sm, overlap, st, R) : launch_t<__nv_bfloat16>(p, n_sm, overlap, st, R);
}

}  // namespace fa
