"""beam — the selection step of a beam search on device logits, beside
sampling.Sampler; the page tables follow through KVCache.reorder."""
from __future__ import annotations

from . import _lib as L
from .paged import _code

NO_TOKEN = -1  # eos: no token ends a beam


def workspace_bytes(n_batch: int, n_beams: int, vocab: int, k: int) -> int:
    """bytes of the workspace of select()"""
    return L.lib().fa_beam_select_ws(n_batch, n_beams, vocab, k)


def _grid(t, name, shape, floating):
    if tuple(t.shape) != shape or t.element_size() != 4 or t.is_floating_point() != floating or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {'float32' if floating else 'int32'} {list(shape)} tensor is needed")
    return t.data_ptr()


def select(logits, scores, done, out_scores, out_parents, out_tokens, out_done, workspace, eos: int = NO_TOKEN,
           pad: int = 0, stream: int = 0):
    """The k best continuations of every request: logits [batch * beams, vocab]
    (any row stride), scores and done [batch, beams] (done may be None), out_*
    [batch, k] (out_done may be None; an out tensor may be its own input when
    k = beams).  Candidates, ties and beams that are done: fa_beam_select."""
    nb, beams = scores.shape
    k = out_scores.shape[1]
    if logits.dim() != 2 or logits.shape[0] != nb * beams:
        raise ValueError("logits: [batch * beams, vocab]")
    ld, inner = logits.stride()
    if inner != 1 and logits.shape[1] > 1:
        raise ValueError("logits: the elements of a row are not consecutive")
    if not workspace.is_contiguous():
        raise ValueError("workspace: contiguous")
    vocab = logits.shape[1]
    a, b = (nb, beams), (nb, k)
    L.check(L.lib().fa_beam_select(
        logits.data_ptr(), _code(logits, "logits"), ld if logits.shape[0] > 1 else vocab, nb, beams, vocab,
        _grid(scores, "scores", a, True), None if done is None else _grid(done, "done", a, False), k,
        eos & 0xFFFFFFFF, pad, _grid(out_scores, "out_scores", b, True), _grid(out_parents, "out_parents", b, False),
        _grid(out_tokens, "out_tokens", b, False), None if out_done is None else _grid(out_done, "out_done", b, False),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), stream))
