// Pages of a model's K/V cache shared between its sequences: fork, reorder
// (beam search), truncation and compaction.  The tables are kept on the host
// and uploaded where they change; only partly filled pages are copied.  What a
// call needs of memory is there before it changes the tables (ready, and the free
// list has room for every page from the beginning), so that one that fails leaves
// them as they were.  (The reference clones whole caches: src/kv_cache.rs:13
// derives Clone.)
#include <algorithm>

#include "model.hpp"
#include "paged_ops.hpp"

namespace fa {

#define CUDA_TRY(expr)                                                                                   \
  do {                                                                                                   \
    cudaError_t e_ = (expr);                                                                             \
    if (e_ != cudaSuccess) return fail(FA_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_)); \
  } while (0)
#define TRY(expr)                 \
  do {                            \
    const int rc_ = (expr);       \
    if (rc_ != FA_OK) return rc_; \
  } while (0)

fa_pages KvCache::pages() const {
  fa_pages p{};
  p.base = base;
  p.layer_stride = layer_stride;
  p.dtype = f16 ? FA_KV_F16 : FA_KV_F32;
  p.n_layers = m->cfg.n_layers;
  p.n_pages = (uint32_t)refs.size();
  p.n_kv_heads = m->cfg.n_kv_heads;
  p.head_dim = m->cfg.head_dim;
  p.page_table = page_table;
  p.n_seq = n_seq;
  p.max_pages = max_pages;
  return p;
}

uint32_t KvCache::take() {
  const uint32_t p = free_pages.back();
  free_pages.pop_back();
  refs[p] = 1;
  return p;
}
void KvCache::drop(uint32_t page) {
  if (--refs[page] == 0) free_pages.push_back(page);
}

uint32_t KvCache::used_pages() const {
  std::vector<uint8_t> seen(refs.size(), 0);
  uint32_t n = 0;
  for (uint32_t s = 0; s < n_seq; ++s)
    for (uint32_t i = 0; i * 16 < len[s]; ++i) {
      uint8_t &f = seen[table[(size_t)s * max_pages + i]];
      n += !f;
      f = 1;
    }
  return n;
}

int KvCache::upload(uint32_t seq) {
  CUDA_TRY(cudaMemcpyAsync(page_table + (size_t)seq * max_pages, row(seq), (size_t)max_pages * 4, cudaMemcpyHostToDevice,
                           m->stream));
  return FA_OK;
}

int KvCache::ready() {
  const size_t most = std::max(n_seq, max_pages);  // at most a move a sequence, or one an entry of a row
  moves.clear();
  moves.reserve(most);
  list.reserve(3 * most);
  if (scratch) return FA_OK;
  const size_t words = 3 * (size_t)std::max(n_seq, max_pages) + (size_t)max_pages * 16 + 8;
  if (cudaMalloc(&scratch, words * 4) != cudaSuccess) {
    cudaGetLastError();
    scratch = nullptr;
    return fail(FA_ERR_OOM, "page list allocation failed");
  }
  return FA_OK;
}

int KvCache::copy() {
  if (moves.empty()) return FA_OK;
  const uint32_t n = (uint32_t)moves.size();
  list.resize(3 * (size_t)n);
  for (uint32_t i = 0; i < n; ++i) {
    list[i] = moves[i].src;
    list[n + i] = moves[i].dst;
    list[2 * n + i] = moves[i].slots;
  }
  CUDA_TRY(cudaMemcpyAsync(scratch, list.data(), list.size() * 4, cudaMemcpyHostToDevice, m->stream));
  PageCopyParams p{};
  p.pg = pages();
  p.src = scratch;
  p.dst = scratch + n;
  p.slots = scratch + 2 * n;
  p.n = n;
  if (launch_page_copy(p, m->stream)) return fail(FA_ERR_CUDA, "page copy launch failed");
  return FA_OK;
}

// The model's stream is a non-blocking one, so nothing else orders it with the
// stream on which a caller has the operators on pages work.  An event costs less
// than a host wait, and the calls behind it end with one.
int KvCache::follow(cudaStream_t st) {
  CUDA_TRY(cudaSetDevice(m->device));
  if (!order) CUDA_TRY(cudaEventCreateWithFlags(&order, cudaEventDisableTiming));
  cudaError_t e = cudaEventRecord(order, st);
  if (e == cudaSuccess) e = cudaStreamWaitEvent(m->stream, order, 0);
  if (e == cudaSuccess) return FA_OK;
  cudaGetLastError();  // not sticky: later launch checks must not see it
  return fail(FA_ERR_CUDA, std::string("the cache cannot follow the caller's stream: ") + cudaGetErrorString(e));
}
int KvCache::settle() { return lent && m ? follow(cudaStreamLegacy) : FA_OK; }

int KvCache::fork(uint32_t src, uint32_t dst) {
  if (!m) return fail(FA_ERR_INVALID, "the cache's model was freed");
  if (src == dst) return FA_OK;
  CUDA_TRY(cudaSetDevice(m->device));
  TRY(ready());
  TRY(settle());
  const uint32_t full = len[src] / 16, rest = len[src] % 16;
  uint32_t *s = row(src), *d = row(dst);
  for (uint32_t i = 0; i < full; ++i) {
    if (d[i] == s[i]) continue;
    drop(d[i]);
    d[i] = s[i];
    ++refs[s[i]];
  }
  for (uint32_t i = full; i < max_pages; ++i)
    if (refs[d[i]] > 1) {
      drop(d[i]);
      d[i] = take();
    }
  len[dst] = len[src];
  TRY(upload(dst));
  if (rest) moves.push_back({s[full], d[full], rest});
  TRY(copy());
  return m->sync();
}

int KvCache::reorder(const uint32_t *parents, uint32_t n) {
  if (!m) return fail(FA_ERR_INVALID, "the cache's model was freed");
  bool same = true;
  for (uint32_t i = 0; i < n; ++i) same = same && parents[i] == i;
  if (same) return FA_OK;
  CUDA_TRY(cudaSetDevice(m->device));
  TRY(ready());
  TRY(settle());
  const std::vector<uint32_t> old(table.begin(), table.begin() + (size_t)n * max_pages), was(len.begin(), len.begin() + n);
  // one child of each parent takes over the parent's own pages: itself, else
  // the first; the other children get free ones
  std::vector<uint32_t> heir(n, n);
  for (uint32_t i = n; i-- > 0;) heir[parents[i]] = i;
  for (uint32_t i = 0; i < n; ++i)
    if (parents[i] == i) heir[i] = i;
  for (uint32_t p : old) --refs[p];
  auto keep = [&](uint32_t i, uint32_t e, uint32_t page) {
    row(i)[e] = page;
    ++refs[page];
  };
  for (uint32_t i = 0; i < n; ++i) {
    const uint32_t p = parents[i], full = was[p] / 16;
    for (uint32_t e = 0; e < (heir[p] == i ? max_pages : full); ++e) keep(i, e, old[(size_t)p * max_pages + e]);
    len[i] = was[p];
  }
  free_pages.clear();
  for (uint32_t p = (uint32_t)refs.size(); p-- > 0;)
    if (!refs[p]) free_pages.push_back(p);
  for (uint32_t i = 0; i < n; ++i) {
    const uint32_t p = parents[i], full = was[p] / 16;
    if (heir[p] == i) continue;
    for (uint32_t e = full; e < max_pages; ++e) row(i)[e] = take();
    if (was[p] % 16) moves.push_back({old[(size_t)p * max_pages + full], row(i)[full], was[p] % 16});
  }
  for (uint32_t i = 0; i < n; ++i)
    if (parents[i] != i) TRY(upload(i));
  TRY(copy());
  return m->sync();
}

int KvCache::truncate(uint32_t seq, uint32_t n) {
  const uint32_t full = n / 16, rest = n % 16;
  uint32_t *r = row(seq);
  bool changed = false;
  for (uint32_t i = full; i < max_pages; ++i) changed = changed || refs[r[i]] > 1;
  if (!changed) {
    len[seq] = n;
    return FA_OK;
  }
  if (!m) return fail(FA_ERR_INVALID, "the cache's model was freed");
  CUDA_TRY(cudaSetDevice(m->device));
  TRY(ready());
  TRY(settle());
  for (uint32_t i = full; i < max_pages; ++i)
    if (refs[r[i]] > 1) {
      const uint32_t page = r[i];
      drop(page);
      r[i] = take();
      if (i == full && rest) moves.push_back({page, r[i], rest});
    }
  len[seq] = n;
  TRY(upload(seq));
  TRY(copy());
  return m->sync();
}

int KvCache::compact(uint32_t seq, const uint32_t *keep, uint32_t n) {
  uint32_t j0 = 0;
  while (j0 < n && keep[j0] == j0) ++j0;
  if (j0 == n) return truncate(seq, n);
  if (!m) return fail(FA_ERR_INVALID, "the cache's model was freed");
  CUDA_TRY(cudaSetDevice(m->device));
  TRY(ready());
  TRY(settle());
  // pages that are written become the sequence's own, with their contents
  uint32_t *r = row(seq);
  for (uint32_t i = j0 / 16; i <= (n - 1) / 16; ++i)
    if (refs[r[i]] > 1) {
      const uint32_t page = r[i];
      drop(page);
      r[i] = take();
      moves.push_back({page, r[i], 16});
    }
  if (!moves.empty()) TRY(upload(seq));
  TRY(copy());
  const uint32_t head[3] = {seq, 0, n};
  uint32_t *at = scratch + 3 * (size_t)std::max(n_seq, max_pages);
  CUDA_TRY(cudaMemcpyAsync(at, head, sizeof head, cudaMemcpyHostToDevice, m->stream));
  CUDA_TRY(cudaMemcpyAsync(at + 3, keep, (size_t)n * 4, cudaMemcpyHostToDevice, m->stream));
  PageCompactParams p{};
  p.pg = pages();
  p.seq = at;
  p.start = at + 1;
  p.keep = at + 3;
  p.n = 1;
  p.n_keep = n;
  if (launch_page_compact(p, m->stream)) return fail(FA_ERR_CUDA, "page compaction launch failed");
  TRY(truncate(seq, n));
  return m->sync();
}

}  // namespace fa
