"""Calls at the edges of what the paged operators and the beam selection allow,
as the host takes them: no GPU needed, no pointer is read."""
import ctypes as C

import numpy as np
import pytest

from fishai_engine import _lib as L
from fishai_engine import beam, paged
from fishai_engine.kv_cache import KVCache
from fishai_engine.model import ModelWeights
from test_cpu_paged import P, call_attn, call_beam, call_rope, pages


@pytest.mark.parametrize("chunks", [1 << 31, (1 << 32) - 128, (1 << 32) - 1])
def test_attention_refuses_more_chunks_than_the_kernels_count(chunks):
    assert call_attn(chunks=chunks, seq=P) == L.ERR_INVALID
    assert "chunks" in L.last_error()


def refused_as_overlapping(rc):
    return rc == L.ERR_INVALID and "overlap" in L.last_error()


@pytest.mark.parametrize("n", [1, 2, 5])
@pytest.mark.parametrize("stride", [128, 136, 256, 300])
def test_overlap_of_rows_is_told_by_the_element(n, stride):
    """q and out: rows of 128 two-byte elements at any distance, against the sets of bytes"""
    pg = pages(n_kv_heads=2, head_dim=64, layer_stride=2 * 2 * 16 * 64 * 8)
    q = P * 64
    mine = {q + 2 * (i * stride + e) for i in range(n) for e in range(128)}
    for by in list(range(-5 * 300, 5 * 300 + 1, 7)) + [0, 127, 128, -127, -128, stride - 128, 128 - stride, stride, -stride]:
        out = q + 2 * by
        shared = bool(mine & {out + 2 * (i * stride + e) for i in range(n) for e in range(128)})
        kw = dict(q=q, out=out, qs=stride, os=stride, heads=2, n=n)
        assert refused_as_overlapping(call_attn(pg, max_q=n, **kw)) == shared, by
        kw.update(k=q * 4, v=q * 8, ks=128, vs=128)
        assert refused_as_overlapping(call_rope(pg, **kw)) == (shared and by != 0), by  # in place is fine


def test_overlap_of_rows_of_two_strides_or_types_goes_by_the_whole_span():
    pg = pages(n_kv_heads=2, head_dim=64, layer_stride=2 * 2 * 16 * 64 * 8)
    kw = dict(q=P * 64, qs=256, heads=2, n=3)
    for out, os, shared in ((P * 64 + 256, 264, True), (P * 64 + 2 * (2 * 256 + 128), 264, False), (P * 64 - 2 * (2 * 264 + 128), 264, False)):
        assert refused_as_overlapping(call_attn(pg, out=out, os=os, **kw)) == shared
    kw.update(k=P * 256, v=P * 512, ks=128, vs=128, dt=L.KV_F32)  # q of four bytes, out of two: one stride in bytes
    for out, shared in ((P * 64 + 512, False), (P * 64 + 510, True), (P * 64 + 768, False), (P * 64 + 770, True), (P * 64, True)):
        assert refused_as_overlapping(call_rope(pg, out=out, os=512, **kw)) == shared, out


BIG = 1 << 32  # would arrive as 0


def test_wrappers_refuse_numbers_beyond_32_bits():
    import torch
    kv = paged.PagedKV(torch.zeros(1, 4, 2, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32))
    q, i = torch.zeros(3, 128), torch.zeros(3, dtype=torch.int32)
    ws = torch.empty(paged.workspace_bytes(64), dtype=torch.uint8)
    for layer in (BIG, -BIG, -1):
        with pytest.raises(ValueError):
            paged.rope_append(kv, layer, paged.Rope(64), q, q.clone(), q.clone(), i, i, q.clone())
        with pytest.raises(ValueError):
            paged.attention(kv, layer, q, i, i[:2], q.clone(), 3, ws)
    for bad in (dict(max_q=BIG), dict(max_q=-1), dict(window=BIG + 5), dict(window=-1)):
        with pytest.raises(ValueError):
            paged.attention(kv, 0, q, i, i[:2], q.clone(), **{"max_q": 3, **bad}, workspace=ws)
    for bad in (dict(head_dim=BIG + 64), dict(rot_dim=BIG + 64), dict(rot_dim=-2), dict(context=BIG + 1)):
        with pytest.raises(ValueError):
            paged.Rope(**{"head_dim": 64, **bad})
    sc, ii = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)
    for bad in (dict(eos=BIG + 2), dict(eos=-2), dict(pad=BIG), dict(pad=-1)):
        with pytest.raises(ValueError):
            beam.select(torch.zeros(6, 10), sc, ii, sc, ii, ii, ii, ws, **bad)


class NoLibrary:
    """a cache or model whose calls would reach the library with a null handle, which answers ERR_INVALID"""
    _h = None


@pytest.mark.parametrize("call", [lambda kv: kv.fork(BIG, 0), lambda kv: kv.fork(0, BIG + 1), lambda kv: kv.fork(-1, 0),
                                  lambda kv: kv.truncate(0, BIG + 5), lambda kv: kv.truncate(BIG, 1), lambda kv: kv.truncate(0, -1),
                                  lambda kv: kv.reorder(np.array([0, BIG])), lambda kv: kv.reorder(np.array([-1])), lambda kv: kv.reorder([0, BIG]),
                                  lambda kv: kv.compact(BIG, [0]), lambda kv: kv.compact(0, np.array([0, BIG + 3])), lambda kv: kv.compact(0, [-1])])
def test_cache_calls_refuse_numbers_beyond_32_bits(call):
    class Cache(NoLibrary, KVCache):
        def __init__(self):
            pass
    with pytest.raises(ValueError):
        call(Cache())


@pytest.mark.parametrize("bad", [dict(n_beams=BIG + 2), dict(n_beams=-1), dict(max_new=-1), dict(eos=BIG), dict(eos=-2), dict(max_new=BIG + 1)])
def test_generate_beams_refuses_numbers_beyond_32_bits(bad):
    class Model(NoLibrary, ModelWeights):
        def __init__(self):
            pass
    with pytest.raises(ValueError):
        Model().generate_beams(**{**dict(prompt_tokens=[5], n_beams=2, max_new=2), **bad})


ODD = P * 8 + 2


def rope_with_err(err):
    r, pg = paged.Rope(64), pages()
    return L.lib().fa_rope_append(r._h, C.addressof(pg), 0, L.KV_F16, P, 512, P * 2, 256, P * 3, 256, 3, 8, P, P, None, P * 4, 512, err, None)


PG = pages()


@pytest.mark.parametrize("call", [lambda: call_rope(pos=ODD), lambda: call_rope(seq=ODD), lambda: call_rope(slot=ODD), lambda: call_rope(pages(page_table=ODD)),
                                  lambda: call_attn(starts=ODD), lambda: call_attn(kv=ODD), lambda: call_attn(seq=ODD), lambda: call_attn(pages(page_table=ODD)),
                                  lambda: call_beam(scores=ODD), lambda: call_beam(done=ODD), lambda: call_beam(os=ODD), lambda: call_beam(op=ODD),
                                  lambda: call_beam(ot=ODD), lambda: call_beam(od=ODD),
                                  lambda: rope_with_err(ODD),
                                  lambda: L.lib().fa_attn_chunks(C.addressof(PG), 0, P, 512, 8, 2, P, P, None, 3, 3, 0.0, 0, P * 4, 512, P * 16,
                                                                 L.lib().fa_attn_chunks_ws(64), ODD, None),
                                  lambda: L.lib().fa_pages_copy(C.addressof(PG), ODD, P, None, 1, None, None),
                                  lambda: L.lib().fa_pages_copy(C.addressof(PG), P, ODD, None, 1, None, None),
                                  lambda: L.lib().fa_pages_copy(C.addressof(PG), P, P, ODD, 1, None, None),
                                  lambda: L.lib().fa_pages_copy(C.addressof(PG), P, P, None, 1, ODD, None),
                                  lambda: L.lib().fa_pages_compact(C.addressof(PG), ODD, P, P, 1, 4, None, None),
                                  lambda: L.lib().fa_pages_compact(C.addressof(PG), P, ODD, P, 1, 4, None, None),
                                  lambda: L.lib().fa_pages_compact(C.addressof(PG), P, P, ODD, 1, 4, None, None),
                                  lambda: L.lib().fa_pages_compact(C.addressof(PG), P, P, P, 1, 4, ODD, None)])
def test_arrays_of_words_at_odd_addresses_are_refused(call):
    """a kernel's load of four bytes there would fault"""
    assert call() == L.ERR_INVALID
    assert "4-byte aligned" in L.last_error()
