// Operators on paged K/V (rotary append, attention of chunks, page copies and
// compaction) and the beam search's selection: launch parameters.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fishai_cuda.h"

namespace fa {

// bits of the operators' error words (FA_FLAG_*), apart from the kErr* bits
enum : uint32_t { kFlagPage = FA_FLAG_PAGE, kFlagRange = FA_FLAG_RANGE, kFlagTimeout = FA_FLAG_TIMEOUT };

constexpr uint32_t kMaxHeadDim = 256;  // of the operators on pages
constexpr uint32_t kPageLen = 16;      // positions of a page

inline uint32_t elem_size(int dtype) { return dtype == FA_KV_F32 ? 4 : 2; }
// bytes of one page of one layer (K and V)
inline uint64_t page_bytes(const fa_pages &p) {
  return (uint64_t)2 * p.n_kv_heads * kPageLen * p.head_dim * elem_size(p.dtype);
}

// ---- rotary positions with the append to the pages ----
struct RopeTable {                   // a kernel parameter (constant bank)
  double turns[kMaxHeadDim / 2];     // f_i / 2 pi: turns per position
  float scale;                       // factor on the turned elements
};
struct RopeAppendParams {
  fa_pages pg;
  uint32_t layer;
  int in_dtype;
  const void *q, *k, *v;
  uint64_t qs, ks, vs, os;           // row strides, elements
  uint32_t n_tokens, n_heads, rot, half_layout;
  const uint32_t *pos, *seq, *slot;
  void *out;
  uint32_t *err;
};
int launch_rope_append(const RopeAppendParams &p, const RopeTable &t, cudaStream_t st);

// ---- attention of chunks ----
struct AttnChunksParams {
  fa_pages pg;
  uint32_t layer;
  const void *q;
  void *out;
  uint64_t qs, os;
  uint32_t n_heads, rep;             // rep = n_heads / n_kv_heads: rows of a token per kv head
  uint32_t n_chunks, n_tokens, max_q;
  const uint32_t *q_start, *kv_len, *seq;
  float scale_log2;                  // scale * log2(e)
  uint32_t window;
  uint32_t aligned;                  // q and out rows are 16-byte aligned
  uint32_t rows_min, rows_max;       // a launch takes the chunks with rows_min <= q_len * rep <= rows_max
  float *part;                       // split items: two slots a CTA
  uint4 *desc;                       // per CTA: the item it starts and later CTAs continue (w = CTAs, 0: none)
  uint32_t *err;
  uint32_t withhold;                 // k_attn_tc: a CTA leaves out its copy of this number (from 1; 0: none), so that
                                     // the waits for it run out
};
// the `withhold` of the calls from now on (fa_debug_set)
void attn_withhold(uint32_t copy);
size_t attn_chunks_ws(uint32_t head_dim);
// ws: attn_chunks_ws(head_dim) bytes; p.part and p.desc are set from it
int launch_attn_chunks(const AttnChunksParams &p, void *ws, uint32_t n_sm, cudaStream_t st);

// ---- page copies ----
struct PageCopyParams {
  fa_pages pg;
  const uint32_t *src, *dst, *slots;
  uint32_t n;
  uint32_t *err;
};
int launch_page_copy(const PageCopyParams &p, cudaStream_t st);
struct PageCompactParams {
  fa_pages pg;
  const uint32_t *seq, *keep, *start;
  uint32_t n, n_keep;
  uint32_t *err;
};
int launch_page_compact(const PageCompactParams &p, cudaStream_t st);

// ---- beam search selection ----
constexpr uint32_t kBeamMaxK = 64, kBeamMaxBeams = 64, kBeamMaxSplits = 32;
struct BeamParams {
  const void *logits;
  int dtype;
  uint64_t ld;
  uint32_t n_batch, n_beams, vocab, k, eos, pad;
  const float *scores;
  const uint32_t *done;
  float *out_scores;
  uint32_t *out_parents, *out_tokens, *out_done;
  uint32_t splits, per;              // ranges of a row, elements of one (a multiple of the tile)
  float2 *stats;                     // [rows][splits] (max, sum of exp(x - max))
  uint2 *cand;                       // [rows][splits][k] (ordered value, token), descending; value 0: none
};
uint32_t beam_splits(uint32_t rows, uint32_t vocab, uint32_t *per);
int launch_beam_select(const BeamParams &p, cudaStream_t st);

}  // namespace fa
