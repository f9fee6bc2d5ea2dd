"""paged — operators on paged K/V in device memory: rotary positions with the
append of new keys and values, attention of chunks of new tokens, page copies
(forks) and compaction.  Beside tensor.scaled_dot_product_attention_device
(one contiguous cache) and KVCache (whose pages they also work on).

Buffers are framework tensors on the GPU (objects with data_ptr(), dtype, shape
and stride(), such as torch tensors); nothing is copied, allocated or waited
for, and `stream` is a cudaStream_t as int (0: the legacy default stream).
Index arrays are contiguous int32 or uint32 tensors.  `err`, one int32 in
device memory, collects FLAG_* bits of indices that the kernels refuse."""
from __future__ import annotations

import ctypes as C
import sys

from . import _lib as L

PAGE = 16  # positions of a page
NO_TOKEN = -1  # in int32 `seqs` of rope_append: the row is left out
FLAG_PAGE, FLAG_RANGE, FLAG_TIMEOUT = L.FLAG_PAGE, L.FLAG_RANGE, L.FLAG_TIMEOUT

_DTYPES = {}  # torch dtype -> FA_KV_*


def _code(t, name):
    """the FA_KV_* id of a tensor's element type"""
    if not _DTYPES:
        torch = sys.modules["torch"]
        _DTYPES.update({torch.float32: L.KV_F32, torch.float16: L.KV_F16, torch.bfloat16: L.KV_BF16})
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: element type {t.dtype} is not float32, float16 or bfloat16")
    return code


def _index(t, name, n=None):
    """address of a contiguous array of n 32-bit whole numbers; None passes"""
    if t is None:
        return None
    if t.dim() != 1 or t.element_size() != 4 or t.is_floating_point() or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous 1-d int32 tensor is needed")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name}: {t.shape[0]} entries, {n} needed")
    return t.data_ptr()


def _rows(t, name, width):
    """address and row stride of [n, width] rows with unit inner stride"""
    shape = t.shape
    if len(shape) == 2:
        if shape[1] != width:
            raise ValueError(f"{name}: rows of {shape[1]}, {width} needed")
        stride, inner = t.stride()
    elif len(shape) == 3:
        if shape[1] * shape[2] != width:
            raise ValueError(f"{name}: rows of {shape[1]} x {shape[2]}, {width} in all needed")
        stride, mid, inner = t.stride()
        if shape[1] > 1 and mid != shape[2]:
            raise ValueError(f"{name}: the heads of a row are not consecutive")
    else:
        raise ValueError(f"{name}: [tokens, heads * head_dim] or [tokens, heads, head_dim] needed")
    if inner != 1 and width > 1:
        raise ValueError(f"{name}: the elements of a row are not consecutive")
    return t.data_ptr(), max(stride, width) if shape[0] <= 1 else stride


class PagedKV:
    """Pages of K/V and the table that says where each sequence's positions are.

    pages: [layers, pages, 2, kv heads, 16, head_dim] (K, then V), float32,
    float16 or bfloat16; each layer contiguous.  page_table: int32
    [sequences, most pages]; positions 16 i .. 16 i + 15 of a sequence are in
    page page_table[sequence][i].  The tensors are kept alive by this object;
    their contents may change at any time."""

    def __init__(self, pages, page_table):
        if pages.dim() != 6 or pages.shape[2] != 2 or pages.shape[4] != PAGE:
            raise ValueError("pages: [layers, pages, 2, kv heads, 16, head_dim] needed")
        if pages.shape[0] == 0 or not pages[0].is_contiguous():
            raise ValueError("pages: each layer has to be contiguous")
        if page_table.dim() != 2 or page_table.element_size() != 4 or page_table.is_floating_point() or \
                not page_table.is_contiguous():
            raise ValueError("page_table: a contiguous int32 [sequences, pages] tensor is needed")
        self.pages, self.page_table = pages, page_table
        self._set(L.fa_pages(pages.data_ptr(), pages.stride(0), _code(pages, "pages"), pages.shape[0], pages.shape[1],
                             pages.shape[3], pages.shape[5], page_table.data_ptr(), page_table.shape[0],
                             page_table.shape[1]))

    @classmethod
    def of(cls, kv_cache) -> "PagedKV":
        """the pages of a model's KVCache (kept alive by this object)"""
        self = cls.__new__(cls)
        c = L.fa_pages()
        L.check(L.lib().fa_kv_pages(kv_cache._h, C.byref(c)))
        self.cache = kv_cache
        self._set(c)
        return self

    def _set(self, c):
        self._c = c
        self._ref = C.addressof(c)
        self.dtype, self.n_layers, self.n_pages = c.dtype, c.n_layers, c.n_pages
        self.n_kv_heads, self.head_dim, self.n_seq, self.max_pages = c.n_kv_heads, c.head_dim, c.n_seq, c.max_pages
        self._kv_width = c.n_kv_heads * c.head_dim


_LAYOUTS = {"interleaved": L.ROPE_INTERLEAVED, "half": L.ROPE_HALF}
_SCALINGS = {"none": L.ROPE_PLAIN, "linear": L.ROPE_LINEAR, "ntk": L.ROPE_NTK, "llama3": L.ROPE_LLAMA3,
             "yarn": L.ROPE_YARN}


class Rope:
    """Rotary frequencies of a head (fa_rope_create): layout "interleaved"
    (pairs 2i, 2i+1, as the model's own, src/tensor.rs:331-392) or "half" (pairs
    i, i + rot_dim/2), rot_dim elements turned, scaling "none", "linear", "ntk",
    "llama3" or "yarn" by `factor` beyond `context` positions."""

    def __init__(self, head_dim: int, rot_dim: int = None, base: float = 10000.0, layout: str = "interleaved",
                 scaling: str = "none", factor: float = 1.0, context: int = 8192, low_turns: float = 1.0,
                 high_turns: float = 4.0, beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 0.0):
        if layout not in _LAYOUTS or scaling not in _SCALINGS:
            raise ValueError(f"layout is one of {sorted(_LAYOUTS)}, scaling one of {sorted(_SCALINGS)}")
        self._h = None
        self.head_dim, self.rot_dim = head_dim, head_dim if rot_dim is None else rot_dim
        c = L.fa_rope_config(head_dim, self.rot_dim, _LAYOUTS[layout], _SCALINGS[scaling], base, factor, context,
                             low_turns, high_turns, beta_fast, beta_slow, attn_factor)
        h = C.c_void_p()
        L.check(L.lib().fa_rope_create(C.byref(c), C.byref(h)))
        self._h = h

    def __del__(self):
        if getattr(self, "_h", None):
            L.lib().fa_rope_free(self._h)
            self._h = None

    def freqs(self):
        """(the rot_dim/2 scaled frequencies, the factor on the turned elements)"""
        f, s = (C.c_double * (self.rot_dim // 2))(), C.c_double()
        L.check(L.lib().fa_rope_freqs(self._h, f, C.byref(s)))
        return list(f), s.value


def rope_append(kv: PagedKV, layer: int, rope: Rope, q, k, v, positions, seqs, out, slots=None, err=None,
                stream: int = 0):
    """Turns q and k by their tokens' positions, q to `out` ([tokens, heads *
    head_dim] of the pages' type; q itself if the types agree), and puts k and v
    at cache position slots[t] (default positions[t]) of sequence seqs[t].  q, k
    and v are rows of one type, with any row stride (slices of a fused
    projection).  seqs[t] = NO_TOKEN leaves a row out."""
    n = q.shape[0]
    dt = _code(q, "q")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v have one element type")
    if _code(out, "out") != kv.dtype:
        raise ValueError("out has another element type than the pages")
    if k.shape[0] != n or v.shape[0] != n or out.shape[0] != n:
        raise ValueError("q, k, v and out have one row for each token")
    width = q.shape[1] if len(q.shape) == 2 else q.shape[1] * q.shape[2]
    if width % kv.head_dim:
        raise ValueError("q: rows are whole heads")
    qp, qs = _rows(q, "q", width)
    kp, ks = _rows(k, "k", kv._kv_width)
    vp, vs = _rows(v, "v", kv._kv_width)
    op, os = _rows(out, "out", width)
    L.check(L.lib().fa_rope_append(rope._h, kv._ref, layer, dt, qp, qs, kp, ks, vp, vs, n, width // kv.head_dim,
                                   _index(positions, "positions", n), _index(seqs, "seqs", n),
                                   _index(slots, "slots", n), op, os, _index(err, "err"), stream))


def workspace_bytes(head_dim: int) -> int:
    """bytes of the workspace of attention(): fixed for a head size"""
    return L.lib().fa_attn_chunks_ws(head_dim)


def attention(kv: PagedKV, layer: int, q, q_start, kv_len, out, max_q: int, workspace, seqs=None, scale: float = 0.0,
              window: int = 0, err=None, stream: int = 0):
    """Attention of chunks of new tokens over the pages: rows q_start[c] ..
    q_start[c+1] of q and out are a chunk of sequence seqs[c] (default c), whose
    cache holds kv_len[c] positions with the chunk's own last.  Each token sees
    the positions up to its own (the last `window` of them where window > 0).
    max_q: no chunk is longer.  workspace: a uint8 tensor of
    workspace_bytes(head_dim), used by no other call that may run at the same
    time.  scale 0: 1 / sqrt(head_dim)."""
    n = q_start.shape[0] - 1
    if n < 0:
        raise ValueError("q_start: chunks + 1 entries")
    if _code(q, "q") != kv.dtype or out.dtype != q.dtype:
        raise ValueError("q and out have the pages' element type")
    width = q.shape[1] if len(q.shape) == 2 else q.shape[1] * q.shape[2]
    if width % kv.head_dim or out.shape[0] != q.shape[0]:
        raise ValueError("q: rows are whole heads, and out has as many rows")
    if window < 0 or max_q < 0:
        raise ValueError("window and max_q are not negative")
    qp, qs = _rows(q, "q", width)
    op, os = _rows(out, "out", width)
    if not workspace.is_contiguous():
        raise ValueError("workspace: contiguous")
    L.check(L.lib().fa_attn_chunks(kv._ref, layer, qp, qs, width // kv.head_dim, n, _index(q_start, "q_start"),
                                   _index(kv_len, "kv_len", n), _index(seqs, "seqs", n), q.shape[0], max_q, scale,
                                   window, op, os, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                                   _index(err, "err"), stream))


def copy_pages(kv: PagedKV, src, dst, slots=None, err=None, stream: int = 0):
    """Copies the first slots[i] positions (default: all 16) of page src[i] to
    page dst[i] in every layer."""
    n = src.shape[0]
    L.check(L.lib().fa_pages_copy(kv._ref, _index(src, "src"), _index(dst, "dst", n), _index(slots, "slots", n), n,
                                  _index(err, "err"), stream))


def compact(kv: PagedKV, seqs, keep, keep_start, err=None, stream: int = 0):
    """Keeps the positions keep[keep_start[i]:keep_start[i+1]] (ascending) of
    sequence seqs[i] as its first positions, in place and in every layer."""
    n = seqs.shape[0]
    L.check(L.lib().fa_pages_compact(kv._ref, _index(seqs, "seqs"), _index(keep, "keep"),
                                     _index(keep_start, "keep_start", n + 1), n, keep.shape[0], _index(err, "err"),
                                     stream))
