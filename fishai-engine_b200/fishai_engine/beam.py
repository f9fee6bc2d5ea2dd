"""beam — the selection step of a beam search on device logits, beside
sampling.Sampler; the page tables follow through KVCache.reorder."""
from __future__ import annotations

from . import _lib as L
from .paged import _DTYPES, _INTS, _code, _space

NO_TOKEN = -1  # eos: no token ends a beam


def workspace_bytes(n_batch: int, n_beams: int, vocab: int, k: int) -> int:
    """bytes of the workspace of select()"""
    return L.lib().fa_beam_select_ws(n_batch, n_beams, vocab, k)


def _grid(t, name, shape, ints):
    """address of a contiguous [batch, n] tensor of 32-bit whole numbers (ints) or f32"""
    if (t.dtype not in _INTS if ints else _DTYPES.get(t.dtype) != L.KV_F32) or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {'int32' if ints else 'float32'} {list(shape)} tensor is needed")
    return t.data_ptr()


def select(logits, scores, done, out_scores, out_parents, out_tokens, out_done, workspace, eos: int = NO_TOKEN,
           pad: int = 0, stream: int = 0):
    """The k best continuations of every request: logits [batch * beams, vocab]
    (any row stride), scores and done [batch, beams] (done may be None), out_*
    [batch, k] (out_done may be None; an out tensor may be its own input when
    k = beams).  Candidates, ties and beams that are done: fa_beam_select."""
    dt = _code(logits, "logits")
    if scores.dim() != 2 or out_scores.dim() != 2 or logits.dim() != 2:
        raise ValueError("scores [batch, beams], out_scores [batch, k], logits [batch * beams, vocab]")
    a, b = scores.shape, out_scores.shape
    nb, beams = a
    k = b[1]
    rows, vocab = logits.shape
    ld, inner = logits.stride()
    if rows != nb * beams or (inner != 1 and vocab > 1) or b[0] != nb:
        raise ValueError(f"logits: [{nb * beams}, vocab] with consecutive elements, and out of {nb} rows")
    if pad >> 32 or (eos != NO_TOKEN and eos >> 32):
        L.u32(pad=pad, eos=eos)
    wp, wn = _space(workspace)
    rc = L.lib().fa_beam_select(
        logits.data_ptr(), dt, ld if rows > 1 else vocab, nb, beams, vocab, _grid(scores, "scores", a, False),
        None if done is None else _grid(done, "done", a, True), k, eos & 0xFFFFFFFF, pad,
        _grid(out_scores, "out_scores", b, False), _grid(out_parents, "out_parents", b, True),
        _grid(out_tokens, "out_tokens", b, True), None if out_done is None else _grid(out_done, "out_done", b, True), wp, wn,
        stream)
    if rc:
        L.check(rc)
