// C entries of the operators on paged K/V and of the beam selection: argument
// checks, the device a call runs on, parameters.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <mutex>
#include <new>
#include <string>

#include "fa_host.hpp"
#include "paged_ops.hpp"

using namespace fa;

struct fa_rope {
  fa_rope_config cfg;
  RopeTable tab;
  double freqs[kMaxHeadDim / 2];
  double scale;
};

namespace {

// Runs a call on the device its buffers are on and puts the caller's current
// device back.
class OnDevice {
 public:
  explicit OnDevice(const char *who) : who_(who) {}
  ~OnDevice() {
    if (switched_) cudaSetDevice(before_);
  }
  // p: device (or managed) memory, of the same device as the others; null is
  // allowed only where the caller says so
  int add(const char *name, const void *p) {
    cudaPointerAttributes a{};
    const cudaError_t e = cudaPointerGetAttributes(&a, p);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(FA_ERR_CUDA, std::string(who_) + ": " + name + ": " + cudaGetErrorString(e));
    }
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
      return fail(FA_ERR_INVALID, std::string(who_) + ": " + name + " is not device memory");
    if (device_ >= 0 && a.device != device_)
      return fail(FA_ERR_INVALID, std::string(who_) + ": " + name + " is on device " + std::to_string(a.device) +
                                      ", other buffers on " + std::to_string(device_));
    device_ = a.device;
    return FA_OK;
  }
  int enter() {
    if (cudaGetDevice(&before_) != cudaSuccess) return fail(FA_ERR_CUDA, std::string(who_) + ": no CUDA device");
    if (before_ == device_) return FA_OK;
    if (cudaSetDevice(device_) != cudaSuccess) return fail(FA_ERR_CUDA, std::string(who_) + ": cannot use the buffers' device");
    switched_ = true;
    return FA_OK;
  }
  int sms() const {
    static std::mutex mu;
    static int count[64];
    if (device_ < 0 || device_ >= 64) return 148;
    std::lock_guard<std::mutex> lock(mu);
    if (!count[device_]) {
      int n = 0;
      if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device_) != cudaSuccess || n < 1) n = 148;
      count[device_] = n;
    }
    return count[device_];
  }

 private:
  const char *who_;
  int device_ = -1, before_ = 0;
  bool switched_ = false;
};

int invalid(const char *who, const std::string &what) { return fail(FA_ERR_INVALID, std::string(who) + ": " + what); }
int launched(const char *who, int rc) {
  if (!rc) return FA_OK;
  const cudaError_t e = cudaGetLastError();
  return fail(FA_ERR_CUDA, std::string(who) + ": launch failed" +
                               (e != cudaSuccess ? std::string(": ") + cudaGetErrorString(e) : std::string()));
}
// arrays of 32-bit words (null: not given); a load from an odd address would fault
int words(const char *who, std::initializer_list<const void *> arrays) {
  for (const void *p : arrays)
    if (reinterpret_cast<uintptr_t>(p) % 4) return invalid(who, "an array of 32-bit words is not 4-byte aligned");
  return FA_OK;
}
bool known(int dtype) { return dtype == FA_KV_F32 || dtype == FA_KV_F16 || dtype == FA_KV_BF16; }

// pages as every operator needs them; the table is not looked at where only
// page numbers are used
int check_pages(const char *who, const fa_pages *p, bool table) {
  if (!p) return invalid(who, "null argument pages");
  if (!p->base) return invalid(who, "null argument pages.base");
  if (table && !p->page_table) return invalid(who, "null argument pages.page_table");
  if (!known(p->dtype)) return invalid(who, "unknown element type of the pages");
  if (!p->n_layers || !p->n_pages || !p->n_kv_heads || !p->head_dim) return invalid(who, "zero size of the pages");
  if (p->head_dim % 8 || p->head_dim > kMaxHeadDim) return fail(FA_ERR_UNSUPPORTED, std::string(who) + ": head_dim is a multiple of 8 up to 256");
  if (p->n_kv_heads > 32767 || p->n_layers > 65535) return invalid(who, "more than 32767 kv heads or 65535 layers");
  if (table && (!p->n_seq || !p->max_pages)) return invalid(who, "empty page table");
  if (table && p->max_pages > (1u << 21)) return invalid(who, "more than 2^21 pages a sequence");
  if (table && reinterpret_cast<uintptr_t>(p->page_table) % 4) return invalid(who, "pages.page_table is not 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(p->base) % 16) return invalid(who, "pages.base is not 16-byte aligned");
  if (p->layer_stride % 8) return invalid(who, "pages.layer_stride is not a multiple of 8 elements");
  const uint64_t layer = (uint64_t)p->n_pages * 2 * p->n_kv_heads * kPageLen * p->head_dim;
  if (p->n_layers > 1 && p->layer_stride < layer) return invalid(who, "pages.layer_stride is smaller than a layer's pages");
  return FA_OK;
}

#define TRY(expr)                  \
  do {                             \
    const int rc_ = (expr);        \
    if (rc_ != FA_OK) return rc_;  \
  } while (0)

// n rows of `bytes` each, `stride` bytes apart
struct Rows {
  uintptr_t at;
  uint64_t stride, bytes;
};
Rows rows_of(const void *p, uint64_t stride, uint64_t row, uint32_t es) { return {reinterpret_cast<uintptr_t>(p), stride * es, row * es}; }
// Whether n rows of a and of b share a byte.  With one stride, as column ranges of
// one buffer have, row j of b starts r bytes behind the start of a's row j + d and
// ends before a's row j + d + 2; with two, whole spans are compared.
bool overlap(uint64_t n, const Rows &a, const Rows &b) {
  if (n > 1 && a.stride == b.stride) {
    if (a.at > b.at) return overlap(n, b, a);
    const uint64_t d = (b.at - a.at) / a.stride, r = (b.at - a.at) % a.stride;
    return (d < n && r < a.bytes) || (d + 1 < n && r + b.bytes > a.stride);
  }
  const uint64_t an = (n - 1) * a.stride + a.bytes, bn = (n - 1) * b.stride + b.bytes;
  return a.at < b.at + bn && b.at < a.at + an;
}

}  // namespace

extern "C" {

// ------------------------------------------------------------ rotary positions
void fa_rope_config_default(fa_rope_config *c, uint32_t head_dim, double base) {
  if (!c) return;
  *c = fa_rope_config{};
  c->head_dim = c->rot_dim = head_dim;
  c->layout = FA_ROPE_INTERLEAVED;
  c->scaling = FA_ROPE_PLAIN;
  c->base = base;
  c->factor = 1.0;
  c->context = 8192;
  c->low_turns = 1.0;
  c->high_turns = 4.0;
  c->beta_fast = 32.0;
  c->beta_slow = 1.0;
  c->attn_factor = 0.0;
}

int fa_rope_create(const fa_rope_config *c, fa_rope **out) {
  const char *who = "fa_rope_create";
  if (!c) return invalid(who, "null argument cfg");
  if (!out) return invalid(who, "null argument out");
  *out = nullptr;
  if (!c->head_dim || c->head_dim % 8 || c->head_dim > kMaxHeadDim)
    return fail(FA_ERR_UNSUPPORTED, std::string(who) + ": head_dim is a multiple of 8 up to 256");
  if (c->rot_dim < 2 || c->rot_dim % 2 || c->rot_dim > c->head_dim) return invalid(who, "rot_dim is even, 2 to head_dim");
  if (c->layout != FA_ROPE_INTERLEAVED && c->layout != FA_ROPE_HALF) return invalid(who, "unknown layout");
  if (c->scaling < FA_ROPE_PLAIN || c->scaling > FA_ROPE_YARN) return invalid(who, "unknown scaling");
  if (!(c->base > 1.0) || !std::isfinite(c->base)) return invalid(who, "base is a finite number above 1");
  if (c->scaling != FA_ROPE_PLAIN && (!(c->factor >= 1.0) || !std::isfinite(c->factor)))
    return invalid(who, "factor is a finite number, at least 1");
  const bool blend = c->scaling == FA_ROPE_LLAMA3 || c->scaling == FA_ROPE_YARN;
  if (blend && !c->context) return invalid(who, "context is zero");
  if (c->scaling == FA_ROPE_NTK && c->rot_dim < 4) return invalid(who, "NTK scaling needs rot_dim of at least 4");
  if (c->scaling == FA_ROPE_LLAMA3 && (!(c->low_turns > 0) || !(c->high_turns > c->low_turns) || !std::isfinite(c->high_turns)))
    return invalid(who, "0 < low_turns < high_turns");
  if (c->scaling == FA_ROPE_YARN && (!(c->beta_slow > 0) || !(c->beta_fast > c->beta_slow) || !std::isfinite(c->beta_fast) ||
                                     !(c->attn_factor >= 0) || !std::isfinite(c->attn_factor)))
    return invalid(who, "0 < beta_slow < beta_fast and attn_factor >= 0");
  fa_rope *r = new (std::nothrow) fa_rope();
  if (!r) return fail(FA_ERR_OOM, std::string(who) + ": out of memory");
  const double two_pi = 6.283185307179586476925286766559;
  const double rot = c->rot_dim, ctx = c->context;
  double base = c->base;
  if (c->scaling == FA_ROPE_NTK) base *= std::pow(c->factor, rot / (rot - 2.0));
  double lo = 0.0, hi = 0.0;
  if (c->scaling == FA_ROPE_YARN) {  // the pair that turns `beta` times in the context
    auto pair = [&](double beta) { return rot * std::log(ctx / (beta * two_pi)) / (2.0 * std::log(base)); };
    lo = std::max(std::floor(pair(c->beta_fast)), 0.0);
    hi = std::min(std::ceil(pair(c->beta_slow)), rot - 1.0);
  }
  r->cfg = *c;
  r->scale = 1.0;
  if (c->scaling == FA_ROPE_YARN) r->scale = c->attn_factor > 0 ? c->attn_factor : 0.1 * std::log(c->factor) + 1.0;
  for (uint32_t i = 0; i < c->rot_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rot);
    if (c->scaling == FA_ROPE_LINEAR) {
      f /= c->factor;
    } else if (c->scaling == FA_ROPE_LLAMA3) {
      const double t = std::min(1.0, std::max(0.0, (ctx * f / two_pi - c->low_turns) / (c->high_turns - c->low_turns)));
      f = f * t + f / c->factor * (1.0 - t);
    } else if (c->scaling == FA_ROPE_YARN) {
      const double t = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001)));
      f = f / c->factor * t + f * (1.0 - t);
    }
    r->freqs[i] = f;
    r->tab.turns[i] = f / two_pi;
  }
  r->tab.scale = (float)r->scale;
  *out = r;
  return FA_OK;
}
void fa_rope_free(fa_rope *r) { delete r; }
int fa_rope_freqs(const fa_rope *r, double *freqs, double *scale) {
  if (!r) return invalid("fa_rope_freqs", "null argument rope");
  if (freqs)
    for (uint32_t i = 0; i < r->cfg.rot_dim / 2; ++i) freqs[i] = r->freqs[i];
  if (scale) *scale = r->scale;
  return FA_OK;
}

int fa_rope_append(const fa_rope *r, const fa_pages *pages, uint32_t layer, int32_t in_dtype, const void *q,
                   uint64_t q_stride, const void *k, uint64_t k_stride, const void *v, uint64_t v_stride,
                   uint32_t n_tokens, uint32_t n_heads, const uint32_t *pos, const uint32_t *seq, const uint32_t *slot,
                   void *out, uint64_t out_stride, uint32_t *err, void *stream) {
  const char *who = "fa_rope_append";
  if (!r) return invalid(who, "null argument rope");
  TRY(check_pages(who, pages, true));
  if (layer >= pages->n_layers) return invalid(who, "layer out of range");
  if (r->cfg.head_dim != pages->head_dim) return invalid(who, "the rope's head_dim is not the pages'");
  if (!known(in_dtype)) return invalid(who, "unknown element type of q, k, v");
  if (!n_heads || n_heads > 32767) return invalid(who, "1 to 32767 heads");
  if (n_tokens > 0x7FFFFFFFu) return invalid(who, "too many tokens");
  const uint64_t hd = pages->head_dim, qw = n_heads * hd, kw = pages->n_kv_heads * hd;
  if (n_tokens > 1 && (q_stride < qw || out_stride < qw || k_stride < kw || v_stride < kw))
    return invalid(who, "a row stride is smaller than the row");
  if (!n_tokens) return FA_OK;
  if (!q || !k || !v || !pos || !seq || !out) return invalid(who, "null argument");
  const uint32_t ei = elem_size(in_dtype), eo = elem_size(pages->dtype);
  for (const void *b : {q, k, v})
    if (reinterpret_cast<uintptr_t>(b) % ei) return invalid(who, "q, k or v is not aligned to its element type");
  if (reinterpret_cast<uintptr_t>(out) % eo) return invalid(who, "out is not aligned to its element type");
  const bool in_place = q == out && in_dtype == pages->dtype && (q_stride == out_stride || n_tokens == 1);
  if (!in_place && overlap(n_tokens, rows_of(q, q_stride, qw, ei), rows_of(out, out_stride, qw, eo)))
    return invalid(who, "out overlaps q without being q");
  TRY(words(who, {pos, seq, slot, err}));
  OnDevice dev(who);
  TRY(dev.add("pages.base", pages->base));
  TRY(dev.add("pages.page_table", pages->page_table));
  TRY(dev.add("q", q));
  TRY(dev.add("k", k));
  TRY(dev.add("v", v));
  TRY(dev.add("pos", pos));
  TRY(dev.add("seq", seq));
  if (slot) TRY(dev.add("slot", slot));
  TRY(dev.add("out", out));
  if (err) TRY(dev.add("err", err));
  TRY(dev.enter());
  RopeAppendParams p{};
  p.pg = *pages;
  p.layer = layer;
  p.in_dtype = in_dtype;
  p.q = q, p.k = k, p.v = v;
  p.qs = q_stride, p.ks = k_stride, p.vs = v_stride, p.os = out_stride;
  p.n_tokens = n_tokens;
  p.n_heads = n_heads;
  p.rot = r->cfg.rot_dim;
  p.half_layout = r->cfg.layout == FA_ROPE_HALF;
  p.pos = pos, p.seq = seq, p.slot = slot;
  p.out = out;
  p.err = err;
  return launched(who, launch_rope_append(p, r->tab, (cudaStream_t)stream));
}

// ------------------------------------------------------------ attention
size_t fa_attn_chunks_ws(uint32_t head_dim) { return head_dim && head_dim <= kMaxHeadDim ? attn_chunks_ws(head_dim) : 0; }

int fa_attn_chunks(const fa_pages *pages, uint32_t layer, const void *q, uint64_t q_stride, uint32_t n_heads,
                   uint32_t n_chunks, const uint32_t *q_start, const uint32_t *kv_len, const uint32_t *seq,
                   uint32_t n_tokens, uint32_t max_q, float scale, uint32_t window, void *out, uint64_t out_stride,
                   void *ws, size_t ws_bytes, uint32_t *err, void *stream) {
  const char *who = "fa_attn_chunks";
  TRY(check_pages(who, pages, true));
  if (layer >= pages->n_layers) return invalid(who, "layer out of range");
  if (!n_heads || n_heads > 32767 || n_heads % pages->n_kv_heads)
    return invalid(who, "n_heads is a multiple of the pages' kv heads, at most 32767");
  if (!std::isfinite(scale) || scale < 0 || scale > 1e30f) return invalid(who, "scale is a number from 0 to 1e30");
  if ((uint64_t)n_tokens * n_heads > 0x7FFFFFFFu) return invalid(who, "2^31 or more query rows");
  if (n_chunks > 0x7FFFFFFFu) return invalid(who, "2^31 or more chunks");
  if (window > 0x7FFFFFFFu) window = 0;  // wider than any cache: none
  const uint64_t hd = pages->head_dim, qw = n_heads * hd;
  if (n_tokens > 1 && (q_stride < qw || out_stride < qw)) return invalid(who, "a row stride is smaller than the row");
  if (!n_tokens || !n_chunks || !max_q) return FA_OK;
  if (!q || !q_start || !kv_len || !out || !ws) return invalid(who, "null argument");
  if (!seq && n_chunks > pages->n_seq) return invalid(who, "more chunks than sequences");
  if (ws_bytes < attn_chunks_ws(pages->head_dim))
    return invalid(who, "workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(attn_chunks_ws(pages->head_dim)) + " needed");
  if (reinterpret_cast<uintptr_t>(ws) % 16) return invalid(who, "the workspace is not 16-byte aligned");
  const uint32_t es = elem_size(pages->dtype);
  if (reinterpret_cast<uintptr_t>(q) % es || reinterpret_cast<uintptr_t>(out) % es)
    return invalid(who, "q or out is not aligned to its element type");
  if (overlap(n_tokens, rows_of(q, q_stride, qw, es), rows_of(out, out_stride, qw, es)))
    return invalid(who, "out overlaps q");
  TRY(words(who, {q_start, kv_len, seq, err}));
  OnDevice dev(who);
  TRY(dev.add("pages.base", pages->base));
  TRY(dev.add("pages.page_table", pages->page_table));
  TRY(dev.add("q", q));
  TRY(dev.add("q_start", q_start));
  TRY(dev.add("kv_len", kv_len));
  if (seq) TRY(dev.add("seq", seq));
  TRY(dev.add("out", out));
  TRY(dev.add("ws", ws));
  if (err) TRY(dev.add("err", err));
  TRY(dev.enter());
  AttnChunksParams p{};
  p.pg = *pages;
  p.layer = layer;
  p.q = q;
  p.out = out;
  p.qs = q_stride;
  p.os = out_stride;
  p.n_heads = n_heads;
  p.rep = n_heads / pages->n_kv_heads;
  p.n_chunks = n_chunks;
  p.n_tokens = n_tokens;
  p.max_q = max_q < n_tokens ? max_q : n_tokens;
  p.q_start = q_start;
  p.kv_len = kv_len;
  p.seq = seq;
  p.scale_log2 = (float)((scale > 0 ? (double)scale : 1.0 / std::sqrt((double)hd)) * 1.4426950408889634);
  p.window = window;
  p.aligned = reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
              q_stride * es % 16 == 0 && out_stride * es % 16 == 0;
  p.err = err;
  return launched(who, launch_attn_chunks(p, ws, (uint32_t)dev.sms(), (cudaStream_t)stream));
}

// ------------------------------------------------------------ pages
int fa_pages_copy(const fa_pages *pages, const uint32_t *src, const uint32_t *dst, const uint32_t *slots, uint32_t n,
                  uint32_t *err, void *stream) {
  const char *who = "fa_pages_copy";
  TRY(check_pages(who, pages, false));
  if (n > 0x7FFFFFFFu) return invalid(who, "too many pages");
  if (!n) return FA_OK;
  if (!src || !dst) return invalid(who, "null argument");
  TRY(words(who, {src, dst, slots, err}));
  OnDevice dev(who);
  TRY(dev.add("pages.base", pages->base));
  TRY(dev.add("src", src));
  TRY(dev.add("dst", dst));
  if (slots) TRY(dev.add("slots", slots));
  if (err) TRY(dev.add("err", err));
  TRY(dev.enter());
  PageCopyParams p{};
  p.pg = *pages;
  p.src = src, p.dst = dst, p.slots = slots;
  p.n = n;
  p.err = err;
  return launched(who, launch_page_copy(p, (cudaStream_t)stream));
}

int fa_pages_compact(const fa_pages *pages, const uint32_t *seq, const uint32_t *keep, const uint32_t *keep_start,
                     uint32_t n, uint32_t n_keep, uint32_t *err, void *stream) {
  const char *who = "fa_pages_compact";
  TRY(check_pages(who, pages, true));
  if (n_keep > 0x7FFFFFFFu || n > 0x7FFFFFFFu) return invalid(who, "too many kept positions or sequences");
  if (!n || !n_keep) return FA_OK;
  if (!seq || !keep || !keep_start) return invalid(who, "null argument");
  TRY(words(who, {seq, keep, keep_start, err}));
  OnDevice dev(who);
  TRY(dev.add("pages.base", pages->base));
  TRY(dev.add("pages.page_table", pages->page_table));
  TRY(dev.add("seq", seq));
  TRY(dev.add("keep", keep));
  TRY(dev.add("keep_start", keep_start));
  if (err) TRY(dev.add("err", err));
  TRY(dev.enter());
  PageCompactParams p{};
  p.pg = *pages;
  p.seq = seq, p.keep = keep, p.start = keep_start;
  p.n = n;
  p.n_keep = n_keep;
  p.err = err;
  return launched(who, launch_page_compact(p, (cudaStream_t)stream));
}

// ------------------------------------------------------------ beam search
size_t fa_beam_select_ws(uint32_t n_batch, uint32_t n_beams, uint32_t vocab, uint32_t k) {
  if (!n_batch || !n_beams || !vocab || !k || n_beams > kBeamMaxBeams || k > kBeamMaxK || n_batch > (1u << 20) || vocab > (1u << 30)) return 0;
  uint32_t per = 0;
  const uint64_t parts = (uint64_t)n_batch * n_beams * beam_splits(n_batch * n_beams, vocab, &per);
  return parts * (sizeof(float2) + k * sizeof(uint2));
}

int fa_beam_select(const void *logits, int32_t dtype, uint64_t ld, uint32_t n_batch, uint32_t n_beams, uint32_t vocab,
                   const float *scores, const uint32_t *done, uint32_t k, uint32_t eos, uint32_t pad, float *out_scores,
                   uint32_t *out_parents, uint32_t *out_tokens, uint32_t *out_done, void *ws, size_t ws_bytes,
                   void *stream) {
  const char *who = "fa_beam_select";
  if (!known(dtype)) return invalid(who, "unknown element type of the logits");
  if (!n_beams || n_beams > kBeamMaxBeams || !k || k > kBeamMaxK) return invalid(who, "1 to 64 beams and 1 to 64 chosen");
  if (!vocab || vocab > (1u << 30)) return invalid(who, "vocabulary of 1 to 2^30 tokens");
  if (n_batch > (1u << 20)) return invalid(who, "more than 2^20 requests");
  if (pad >= vocab) return invalid(who, "pad is not a token");
  if (ld < vocab && (uint64_t)n_batch * n_beams > 1) return invalid(who, "a row stride is smaller than the row");
  if (!n_batch) return FA_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !ws) return invalid(who, "null argument");
  if (k != n_beams && (out_scores == scores || (done && out_done == done)))
    return invalid(who, "an output in place of its input needs k = n_beams");
  const size_t need = fa_beam_select_ws(n_batch, n_beams, vocab, k);
  if (ws_bytes < need) return invalid(who, "workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(need) + " needed");
  if (reinterpret_cast<uintptr_t>(ws) % 16) return invalid(who, "the workspace is not 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(logits) % elem_size(dtype)) return invalid(who, "logits are not aligned to their element type");
  TRY(words(who, {scores, done, out_scores, out_parents, out_tokens, out_done}));
  OnDevice dev(who);
  TRY(dev.add("logits", logits));
  TRY(dev.add("scores", scores));
  if (done) TRY(dev.add("done", done));
  TRY(dev.add("out_scores", out_scores));
  TRY(dev.add("out_parents", out_parents));
  TRY(dev.add("out_tokens", out_tokens));
  if (out_done) TRY(dev.add("out_done", out_done));
  TRY(dev.add("ws", ws));
  TRY(dev.enter());
  BeamParams p{};
  p.logits = logits;
  p.dtype = dtype;
  p.ld = ld;
  p.n_batch = n_batch;
  p.n_beams = n_beams;
  p.vocab = vocab;
  p.k = k;
  p.eos = eos;
  p.pad = pad;
  p.scores = scores;
  p.done = done;
  p.out_scores = out_scores;
  p.out_parents = out_parents;
  p.out_tokens = out_tokens;
  p.out_done = out_done;
  p.splits = beam_splits(n_batch * n_beams, vocab, &p.per);
  p.stats = static_cast<float2 *>(ws);
  p.cand = reinterpret_cast<uint2 *>(p.stats + (uint64_t)n_batch * n_beams * p.splits);
  return launched(who, launch_beam_select(p, (cudaStream_t)stream));
}

}  // extern "C"
