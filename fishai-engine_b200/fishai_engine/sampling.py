"""Sampler — src/sampling.rs:14-310 on the device (Philox4x32-10 uniforms) —
and sample_logits, which draws from a caller's device logits and numbers."""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from . import _lib as L
from .paged import _DTYPES, _code, _count, _dense, _index


@dataclass
class SamplerConfig:
    """src/sampling.rs:16-80"""
    temperature: float = 0.7
    top_k: int = 40
    top_p: float = 0.95
    repetition_penalty: float = 1.15
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0

    @staticmethod
    def greedy():
        return SamplerConfig(0.0, 0, 1.0, 1.0, 0.0, 0.0)

    @staticmethod
    def creative():
        return SamplerConfig(1.2, 80, 0.98, 1.05, 0.0, 0.0)

    @staticmethod
    def precise():
        return SamplerConfig(0.3, 20, 0.9, 1.3, 0.1, 0.1)

    def _c(self):
        return L.fa_sampler_config(self.temperature, self.top_k, self.top_p, self.repetition_penalty,
                                   self.frequency_penalty, self.presence_penalty)


class Sampler:
    """Sampler::new / sample / observe_token / reset (src/sampling.rs:95-165).
    Categorical draws use Philox4x32-10 keyed by `seed` with the sample index
    as counter (the reference uses the unseeded rand::rng())."""

    def __init__(self, config: SamplerConfig = None, vocab: int = 0, seed: int = 0, seeds=None):
        """seeds: one Philox key per sequence row (batched decode); else one row keyed by seed"""
        self.config = config or SamplerConfig()
        self.vocab = vocab
        keys = list(seeds) if seeds is not None else [seed]
        self.n_seq = len(keys)
        arr = (C.c_uint64 * self.n_seq)(*keys)
        h = C.c_void_p()
        L.check(L.lib().fa_sampler_create(C.byref(self.config._c()), self.n_seq, vocab, arr, C.byref(h)))
        self._h = h

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            L.lib().fa_sampler_free(h)
            self._h = None

    def sample(self, logits) -> int:
        a = np.ascontiguousarray(np.asarray(logits, dtype=np.float32))
        out = C.c_uint32()
        L.check(L.lib().fa_sample(self._h, 0, L.f32_ptr(a), a.size, C.byref(out)))
        return out.value

    def observe_token(self, token_id: int):
        L.check(L.lib().fa_sampler_observe(self._h, 0, token_id))

    def reset(self):
        L.check(L.lib().fa_sampler_reset(self._h, -1))

    def token_freq(self, token_id: int) -> int:
        """token_freq[token_id] (0 for ids never observed)"""
        c = C.c_uint32()
        L.check(L.lib().fa_sampler_freq(self._h, 0, token_id, C.byref(c)))
        return c.value


def _floats(t, name, n):
    """address of a contiguous array of n float32"""
    if _DTYPES.get(t.dtype) != L.KV_F32 or t.shape != (n,) or (n > 1 and not _dense(t)):
        raise ValueError(f"{name}: a contiguous float32 [{n}] tensor is needed")
    return t.data_ptr()


def sample_logits(logits, u, ids, temperature=None, top_k=None, top_p=None, min_p=None, rows=None, logprobs=None, err=None,
                  stream: int = 0):
    """Draws ids[i] from row rows[i] (default i; NO_TOKEN: none) of device logits
    [rows, vocab] (float32, float16 or bfloat16, any row stride) with the random
    number u[i] in [0, 1) and the row's own temperature (0: greedy), top_k (0: off),
    top_p and min_p, and logprobs[i], its log-probability among what is kept.
    Framework tensors on the GPU: float32 but ids, rows, top_k (int32) and err (one
    int32, FLAG_* bits).  What is kept and drawn: fa_sample_logits."""
    dt = _code(logits, "logits")
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise ValueError("logits: [rows, vocab] with consecutive elements")
    m, vocab = shape
    n = _count(ids, "ids")
    if (m | vocab | n) >> 32:
        L.u32(rows=m, vocab=vocab, ids=n)
    rc = L.lib().fa_sample_logits(
        logits.data_ptr(), dt, stride[0] if m > 1 else vocab, m, vocab, None if rows is None else _index(rows, "rows", n), n,
        None if temperature is None else _floats(temperature, "temperature", n), None if top_k is None else _index(top_k, "top_k", n),
        None if top_p is None else _floats(top_p, "top_p", n), None if min_p is None else _floats(min_p, "min_p", n), _floats(u, "u", n),
        _index(ids, "ids", n), None if logprobs is None else _floats(logprobs, "logprobs", n),
        None if err is None else _index(err, "err", 1), stream)
    if rc:
        L.check(rc)
