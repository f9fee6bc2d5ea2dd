// Beam search over the batched decode step: one graph per call holds the
// forward pass of all beams, the selection and the step's bookkeeping; between
// two replays the host reads the chosen parents and reorders the cache's page
// tables (only partly filled pages are copied).
#include <algorithm>
#include <cmath>
#include <limits>

#include "model.hpp"
#include "paged_ops.hpp"

namespace fa {

#define CUDA_TRY(expr)                                                                                   \
  do {                                                                                                   \
    cudaError_t e_ = (expr);                                                                             \
    if (e_ != cudaSuccess) return fail(FA_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_)); \
  } while (0)

namespace {
struct DevBuf {
  void *p = nullptr;
  ~DevBuf() {
    if (p) cudaFree(p);
  }
};
struct Graph {
  cudaGraph_t g = nullptr;
  cudaGraphExec_t e = nullptr;
  ~Graph() {
    if (e) cudaGraphExecDestroy(e);
    if (g) cudaGraphDestroy(g);
  }
};
}  // namespace

int Model::beam_search(KvCache &kv, uint32_t last_token, const fa_beam_config &c, std::vector<uint32_t> &parents,
                       std::vector<uint32_t> &tokens, std::vector<float> &scores, uint32_t *steps) {
  const uint32_t b = c.n_beams, len = kv.len[0], V = cfg.vocab_size;
  *steps = 0;
  int rc;
  if ((rc = ensure_rope(len + c.max_new + 1)) || (rc = ensure_batch_ws(b))) return rc;
  for (uint32_t r = 1; r < b; ++r)
    if ((rc = kv.fork(0, r))) return rc;
  // device state: scores, done, parents, tokens (read back together), history
  // of the bookkeeping kernel, selection workspace
  BeamParams bp{};
  const uint32_t splits = beam_splits(b, V, &bp.per);
  const size_t ws = (size_t)b * splits * (sizeof(float2) + b * sizeof(uint2));
  DevBuf state, hist, space;
  if (cudaMalloc(&state.p, (size_t)4 * b * 4) != cudaSuccess || cudaMalloc(&hist.p, (size_t)c.max_new * b * 4) != cudaSuccess ||
      cudaMalloc(&space.p, ws) != cudaSuccess) {
    cudaGetLastError();
    return fail(FA_ERR_OOM, "beam search buffers");
  }
  float *d_scores = static_cast<float *>(state.p);
  uint32_t *d_done = reinterpret_cast<uint32_t *>(d_scores + b), *d_parents = d_done + b, *d_tokens = d_parents + b;
  std::vector<SeqState> st(b);
  std::vector<uint32_t> host(4 * (size_t)b, 0);
  for (uint32_t r = 0; r < b; ++r) {
    st[r] = SeqState{};
    st[r].pos = len;
    st[r].len = len;
    st[r].token = last_token;
    // all beams begin alike, so only the first may be continued
    reinterpret_cast<float *>(host.data())[r] = r ? -std::numeric_limits<float>::infinity() : 0.0f;
    host[3 * b + r] = last_token;
  }
  CUDA_TRY(cudaMemcpyAsync(bws.states, st.data(), b * sizeof(SeqState), cudaMemcpyHostToDevice, stream));
  CUDA_TRY(cudaMemcpyAsync(state.p, host.data(), host.size() * 4, cudaMemcpyHostToDevice, stream));
  CUDA_TRY(cudaMemsetAsync(bws.step, 0, 4, stream));
  CUDA_TRY(cudaMemsetAsync(bws.err, 0, 4, stream));
  bp.logits = bws.logits;
  bp.dtype = FA_KV_F32;
  bp.ld = V;
  bp.n_batch = 1;
  bp.n_beams = b;
  bp.vocab = V;
  bp.k = b;
  bp.eos = c.eos;
  bp.pad = 0;  // what a finished beam is fed; its tokens are not looked at
  bp.scores = bp.out_scores = d_scores;
  bp.done = bp.out_done = d_done;
  bp.out_parents = d_parents;
  bp.out_tokens = d_tokens;
  bp.splits = splits;
  bp.stats = static_cast<float2 *>(space.p);
  bp.cand = reinterpret_cast<uint2 *>(bp.stats + (size_t)b * splits);
  Graph gr;
  CUDA_TRY(cudaStreamBeginCapture(stream, cudaStreamCaptureModeThreadLocal));
  rc = enqueue_batch_forward(kv, b, d_tokens);
  if (!rc && launch_beam_select(bp, stream)) rc = fail(FA_ERR_CUDA, "beam selection launch failed");
  if (!rc && launch_batch_step_end(bws.states, b, d_tokens, static_cast<uint32_t *>(hist.p), c.max_new, bws.step, stream))
    rc = fail(FA_ERR_CUDA, "step end launch failed");
  const cudaError_t ce = cudaStreamEndCapture(stream, &gr.g);
  if (rc) return rc;
  if (ce != cudaSuccess) return fail(FA_ERR_CUDA, std::string("graph capture failed: ") + cudaGetErrorString(ce));
  CUDA_TRY(cudaGraphInstantiate(&gr.e, gr.g, 0));
  for (uint32_t s = 0; s < c.max_new; ++s) {
    CUDA_TRY(cudaGraphLaunch(gr.e, stream));
    uint32_t e = 0;
    CUDA_TRY(cudaMemcpyAsync(host.data(), state.p, host.size() * 4, cudaMemcpyDeviceToHost, stream));
    CUDA_TRY(cudaMemcpyAsync(&e, bws.err, 4, cudaMemcpyDeviceToHost, stream));
    if ((rc = sync())) return rc;
    if (e & kErrWaitTimeout) return fail(FA_ERR_TIMEOUT, "beam search: a bounded device wait gave up");
    if (e & kErrContext) return fail(FA_ERR_CONTEXT, "position or KV capacity exceeded");
    if (e & kErrRange) return fail(FA_ERR_UNSUPPORTED, "an activation exceeds the f16 range of the tensor-core path");
    if (e) return fail(FA_ERR_INVALID, "token id out of range");
    parents.insert(parents.end(), host.begin() + 2 * b, host.begin() + 3 * b);
    tokens.insert(tokens.end(), host.begin() + 3 * b, host.begin() + 4 * b);
    const float *sc = reinterpret_cast<const float *>(host.data());
    scores.assign(sc, sc + b);
    *steps = s + 1;
    for (uint32_t r = 0; r < b; ++r) ++kv.len[r];
    if (std::all_of(host.begin() + b, host.begin() + 2 * b, [](uint32_t d) { return d != 0; })) break;
    if (s + 1 < c.max_new && (rc = kv.reorder(host.data() + 2 * b, b))) return rc;
  }
  return FA_OK;
}

}  // namespace fa
