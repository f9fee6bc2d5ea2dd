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
_INTS = set()  # the 32-bit index types
_ONE = (1,)


def _learn():
    torch = sys.modules["torch"]
    _DTYPES.update({torch.float32: L.KV_F32, torch.float16: L.KV_F16, torch.bfloat16: L.KV_BF16})
    _INTS.update({torch.int32, torch.uint32})


# The checks run at every call, in front of kernels of a few microseconds: one
# look at dtype, stride and length each, the reasons worked out only on failure.
def _code(t, name):
    """the FA_KV_* id of a tensor's element type"""
    code = _DTYPES.get(t.dtype)
    if code is None:
        if not _DTYPES:
            _learn()
            return _code(t, name)
        raise ValueError(f"{name}: element type {t.dtype} is not float32, float16 or bfloat16")
    return code


def _index(t, name, n):
    """address of a contiguous array of n 32-bit whole numbers"""
    if t.shape != (n,) or t.dtype not in _INTS or (n > 1 and t.stride() != _ONE):
        if not _INTS:
            _learn()
            return _index(t, name, n)
        if t.dtype not in _INTS or t.dim() != 1:
            raise ValueError(f"{name}: a contiguous 1-d int32 tensor is needed")
        if t.shape[0] != n:
            raise ValueError(f"{name}: {t.shape[0]} entries, {n} needed")
        raise ValueError(f"{name}: a contiguous 1-d int32 tensor is needed")
    return t.data_ptr()


def _rows(t, name, n, width):
    """address and row stride of n rows of `width` consecutive elements, [n, width] or [n, heads, head_dim]"""
    shape, stride = t.shape, t.stride()
    if shape == (n, width):
        ok = stride[1] == 1
    else:
        ok = len(shape) == 3 and shape[0] == n and shape[1] * shape[2] == width and stride[2] == 1 and \
            (shape[1] == 1 or stride[1] == shape[2])
    if not ok:
        raise ValueError(f"{name}: {n} rows of {width} consecutive elements are needed, got {list(shape)} with strides {stride}")
    return t.data_ptr(), stride[0] if n > 1 else width


def _width(q, head_dim):
    """elements of a row of whole heads"""
    shape = q.shape
    width = shape[1] if len(shape) == 2 else shape[1] * shape[2] if len(shape) == 3 else 0
    if not width or width % head_dim:
        raise ValueError(f"q: [tokens, heads * {head_dim}] or [tokens, heads, {head_dim}] needed, got {list(shape)}")
    return width


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
        """The pages of a model's KVCache (kept alive by this object).  The
        cache's own calls follow work on the default stream; for work on another
        one call KVCache.wait first.  Its lengths do not count rows that
        rope_append writes behind them, and a row written below them changes in
        every sequence that shares its page."""
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
        L.u32(head_dim=head_dim, rot_dim=self.rot_dim, context=context)
        c = L.fa_rope_config(head_dim, self.rot_dim, _LAYOUTS[layout], _SCALINGS[scaling], base, factor, context,
                             low_turns, high_turns, beta_fast, beta_slow, attn_factor)
        h = C.c_void_p()
        L.check(L.lib().fa_rope_create(C.byref(c), C.byref(h)))
        self._h = h

    def __del__(self):
        if getattr(self, "_h", None) and L is not None:  # None: the interpreter is ending
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
    if layer >> 32:
        L.u32(layer=layer)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v have one element type")
    if _code(out, "out") != kv.dtype:
        raise ValueError("out has another element type than the pages")
    hd, kw = kv.head_dim, kv._kv_width
    width = _width(q, hd)
    qp, qs = _rows(q, "q", n, width)
    kp, ks = _rows(k, "k", n, kw)
    vp, vs = _rows(v, "v", n, kw)
    op, os = _rows(out, "out", n, width)
    rc = L.lib().fa_rope_append(rope._h, kv._ref, layer, dt, qp, qs, kp, ks, vp, vs, n, width // hd,
                                _index(positions, "positions", n), _index(seqs, "seqs", n),
                                None if slots is None else _index(slots, "slots", n), op, os,
                                None if err is None else _index(err, "err", 1), stream)
    if rc:
        L.check(rc)


def _space(t):
    """address and bytes of a contiguous workspace tensor"""
    if not t.is_contiguous():
        raise ValueError("workspace: contiguous")
    return t.data_ptr(), t.numel() * t.element_size()


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
    n, t = kv_len.shape[0], q.shape[0]
    if _code(q, "q") != kv.dtype or out.dtype != q.dtype:
        raise ValueError("q and out have the pages' element type")
    if (layer | max_q | window) >> 32:
        L.u32(layer=layer, max_q=max_q, window=window)
    hd = kv.head_dim
    width = _width(q, hd)
    qp, qs = _rows(q, "q", t, width)
    op, os = _rows(out, "out", t, width)
    rc = L.lib().fa_attn_chunks(kv._ref, layer, qp, qs, width // hd, n, _index(q_start, "q_start", n + 1),
                                _index(kv_len, "kv_len", n), None if seqs is None else _index(seqs, "seqs", n), t, max_q,
                                scale, window, op, os, *_space(workspace), None if err is None else _index(err, "err", 1),
                                stream)
    if rc:
        L.check(rc)


def copy_pages(kv: PagedKV, src, dst, slots=None, err=None, stream: int = 0):
    """Copies the first slots[i] positions (default: all 16) of page src[i] to
    page dst[i] in every layer."""
    n = src.shape[0]
    L.check(L.lib().fa_pages_copy(kv._ref, _index(src, "src", n), _index(dst, "dst", n),
                                  None if slots is None else _index(slots, "slots", n), n,
                                  None if err is None else _index(err, "err", 1), stream))


def compact(kv: PagedKV, seqs, keep, keep_start, err=None, stream: int = 0):
    """Keeps the positions keep[keep_start[i]:keep_start[i+1]] (ascending) of
    sequence seqs[i] as its first positions, in place and in every layer."""
    n = seqs.shape[0]
    L.check(L.lib().fa_pages_compact(kv._ref, _index(seqs, "seqs", n), _index(keep, "keep", keep.shape[0]),
                                     _index(keep_start, "keep_start", n + 1), n, keep.shape[0],
                                     None if err is None else _index(err, "err", 1), stream))
