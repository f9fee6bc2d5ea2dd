"""KVCache — src/kv_cache.rs:13-110, device resident and paged (16 positions
per page).  Unlike the reference's Vec<f32>, capacity is fixed at creation
(max_ctx); appends happen inside ModelWeights.forward on the device."""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib as L


class KVCache:
    def __init__(self, model, max_ctx: int = None, n_seq: int = 1, dtype: int = L.KV_F32):
        self.model = model
        cfg = model.config
        self.max_ctx = int(max_ctx or cfg.context_len)
        self.n_seq = n_seq
        self.dtype = dtype
        self._n_layers = cfg.n_layers
        # a tensor-parallel rank caches only the KV heads it holds
        self.kv_dim = getattr(model, "local_kv_heads", cfg.n_kv_heads) * cfg.head_dim
        h = C.c_void_p()
        L.check(L.lib().fa_kv_create(model._h, n_seq, self.max_ctx, dtype, C.byref(h)))
        self._h = h

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            L.lib().fa_kv_free(h)
            self._h = None

    def n_layers(self) -> int:
        return self._n_layers

    def get(self, layer: int, seq: int = 0):
        """KVCache::get (src/kv_cache.rs:66-69): (k, v) as flat f32 [len * n_kv * head_dim];
        raises IndexError for a bad layer where the reference panics."""
        if layer >= self._n_layers or layer < 0:
            raise IndexError(f"KV cache layer index out of range: {layer} >= {self._n_layers}")
        n = self.seq_len_with_dim(layer, self.kv_dim, seq) * self.kv_dim
        k = np.zeros(max(n, 1), dtype=np.float32)
        v = np.zeros(max(n, 1), dtype=np.float32)
        L.check(L.lib().fa_kv_get(self._h, seq, layer, L.f32_ptr(k), L.f32_ptr(v)))
        return k[:n], v[:n]

    def seq_len(self, layer: int) -> int:
        """KVCache::seq_len (src/kv_cache.rs:75-83) returns 0 in the reference
        whatever the content; kept as is.  Use seq_len_with_dim."""
        if layer >= self._n_layers:
            raise IndexError(f"KV cache layer index out of range: {layer} >= {self._n_layers}")
        return 0

    def seq_len_with_dim(self, layer: int, kv_dim: int, seq: int = 0) -> int:
        """src/kv_cache.rs:90-96"""
        if layer >= self._n_layers:
            raise IndexError(f"KV cache layer index out of range: {layer} >= {self._n_layers}")
        if kv_dim == 0:
            return 0
        n = C.c_uint32()
        L.check(L.lib().fa_kv_seq_len(self._h, seq, C.byref(n)))
        return n.value * self.kv_dim // kv_dim

    def clear(self, seq: int = -1):
        """src/kv_cache.rs:98-103"""
        L.check(L.lib().fa_kv_clear(self._h, seq))

    # ---- sequences that share pages (n_seq > 1; no counterpart in the reference) ----
    def fork(self, src: int, dst: int):
        """sequence dst becomes a copy of sequence src: whole pages are shared,
        a partly filled last page is copied"""
        L.u32(src=src, dst=dst)
        L.check(L.lib().fa_kv_fork(self._h, src, dst))

    def reorder(self, parents):
        """sequence i becomes a copy of what sequence parents[i] was, all at once
        (the step between two selections of a beam search)"""
        a, p = L.u32_list(parents)
        L.check(L.lib().fa_kv_reorder(self._h, p, a.size))

    def truncate(self, seq: int, length: int):
        """drops the positions from `length` on"""
        L.u32(seq=seq, length=length)
        L.check(L.lib().fa_kv_truncate(self._h, seq, length))

    def compact(self, seq: int, keep):
        """keeps the given ascending positions, as positions 0, 1, ...; their keys
        stay turned as they were stored"""
        L.u32(seq=seq)
        a, p = L.u32_list(keep)
        L.check(L.lib().fa_kv_compact(self._h, seq, p, a.size))

    def wait(self, stream: int = 0):
        """The calls on this cache after this one follow what is on `stream` (a
        cudaStream_t as int) now.  For work of paged's operators on the pages
        (PagedKV.of) on another stream than the default one, which every call
        follows by itself."""
        L.check(L.lib().fa_kv_wait(self._h, stream))

    def pages_used(self):
        """(pages that hold positions, each shared one once; pages of the cache)"""
        u, t = C.c_uint32(), C.c_uint32()
        L.check(L.lib().fa_kv_page_count(self._h, C.byref(u), C.byref(t)))
        return u.value, t.value
