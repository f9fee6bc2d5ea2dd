"""Refusals of the operators around a serving step and what is computed on the host: no GPU needed.  Every case is refused
before any pointer is looked at or any kernel runs."""
import ctypes as C
import math

import pytest

from fishai_engine import _lib as L
from fishai_engine import paged

P = 0x30000  # an address that is never read


def pages(**kw):
    f = dict(base=0x10000, layer_stride=2 * 4 * 16 * 64 * 8, dtype=L.KV_F16, n_layers=2, n_pages=8, n_kv_heads=4, head_dim=64,
             page_table=0x20000, n_seq=2, max_pages=4)
    f.update(kw)
    return L.fa_pages(**f)


# ------------------------------------------------------------------ attention with first positions
def call_sinks(pg=None, layer=0, q=P, qs=512, heads=8, chunks=2, starts=P, kv=P, seq=None, n=3, max_q=3, scale=0.0, window=5, sinks=2,
               out=P * 4, os=512, ws=P * 16, ws_bytes=None):
    ws_bytes = L.lib().fa_attn_chunks_ws(64) if ws_bytes is None else ws_bytes
    return L.lib().fa_attn_chunks_sinks(C.addressof(pg or pages()), layer, q, qs, heads, chunks, starts, kv, seq, n, max_q, scale, window,
                                        sinks, out, os, ws, ws_bytes, None, None)


@pytest.mark.parametrize("bad", [dict(layer=2), dict(heads=0), dict(heads=6), dict(qs=511), dict(os=500), dict(scale=-1.0), dict(scale=math.nan),
                                 dict(q=None), dict(starts=None), dict(kv=None), dict(out=None), dict(ws=None), dict(chunks=3),
                                 dict(ws_bytes=100), dict(ws=P * 16 + 8), dict(q=P + 1), dict(out=P), dict(n=1 << 30), dict(starts=P + 2),
                                 dict(pg=pages(dtype=7)), dict(pg=pages(base=None)), dict(pg=pages(max_pages=0))], ids=str)
def test_attention_with_sinks_refuses(bad):
    assert call_sinks(**bad) == L.ERR_INVALID
    assert "fa_attn_chunks_sinks" in L.last_error()


def test_attention_with_sinks_of_nothing():
    assert call_sinks(n=0, q=None, out=None) == L.OK
    assert call_sinks(chunks=0, starts=None, kv=None) == L.OK


# ------------------------------------------------------------------ rotary positions with several axes
@pytest.mark.parametrize("bad", [dict(axes=[16, 17]), dict(axes=[32, 0]), dict(axes=[0, 32]), dict(axes=[8, 8, 8]), dict(axes=[2 ** 32 - 1, 33]),
                                 dict(axes=[1, 31], axis_order="turns"), dict(axes=[10, 10, 12], axis_order="turns"),
                                 dict(axes=[31, 1], axis_freqs="own", scaling="ntk", factor=2.0)], ids=str)
def test_axes_that_do_not_fit_are_refused(bad):
    with pytest.raises(L.FishaiError):
        paged.Rope(64, **bad)


@pytest.mark.parametrize("bad", [dict(axes=[]), dict(axes=[8] * 5), dict(axes=[32, -1]), dict(axes=[16, 16], axis_order="rows"),
                                 dict(axes=[16, 16], axis_freqs="mine"), dict(axes=[2 ** 32, 32])], ids=str)
def test_axes_that_python_refuses(bad):
    with pytest.raises(ValueError):
        paged.Rope(64, **bad)


def test_unknown_orders_are_refused_by_the_library():
    lib, cfg, h = L.lib(), L.fa_rope_config(), C.c_void_p()
    lib.fa_rope_config_default(C.byref(cfg), 64, 10000.0)
    four = C.c_uint32 * 4
    for ax in (L.fa_rope_axes(2, four(16, 16), 2, 0), L.fa_rope_axes(2, four(16, 16), 0, 2), L.fa_rope_axes(0, four(), 0, 0),
               L.fa_rope_axes(5, four(8, 8, 8, 8), 0, 0)):
        assert lib.fa_rope_create_axes(C.byref(cfg), C.byref(ax), C.byref(h)) == L.ERR_INVALID
    assert lib.fa_rope_create_axes(C.byref(cfg), None, C.byref(h)) == L.ERR_INVALID
    assert lib.fa_rope_create_axes(None, C.byref(L.fa_rope_axes(1, four(32), 0, 0)), C.byref(h)) == L.ERR_INVALID
    assert lib.fa_rope_axis_of(None, None) == L.ERR_INVALID


def test_axis_and_frequency_of_each_pair():
    assert paged.Rope(64).axis_of() == [0] * 32
    r = paged.Rope(64, axes=[12, 10, 10])
    assert r.axis_of() == [0] * 12 + [1] * 10 + [2] * 10
    assert r.freqs() == paged.Rope(64).freqs()
    # in turns: 0 1 2 0 1 2 .. as long as an axis has pairs, the rest is of axis 0
    assert paged.Rope(16, axes=[4, 3, 1], axis_order="turns").axis_of() == [0, 1, 2, 0, 1, 0, 0, 1]
    assert paged.Rope(16, axes=[5, 1, 2], axis_order="turns").axis_of() == [0, 1, 2, 0, 0, 2, 0, 0]
    # an axis's own series: that of a rope of its width
    r = paged.Rope(64, axes=[12, 10, 10], axis_freqs="own")
    assert r.freqs()[0] == paged.Rope(64, rot_dim=24).freqs()[0] + 2 * paged.Rope(64, rot_dim=20).freqs()[0]
    for scaling in ("linear", "ntk", "llama3", "yarn"):
        kw = dict(scaling=scaling, factor=4.0, context=2048)
        r = paged.Rope(64, axes=[14, 9, 9], axis_order="turns", axis_freqs="own", **kw)
        want = {a: iter(paged.Rope(64, rot_dim=2 * n, **kw).freqs()[0]) for a, n in enumerate([14, 9, 9])}
        assert r.freqs()[0] == [next(want[a]) for a in r.axis_of()]


def call_axes(r=None, pg=None, layer=0, dt=L.KV_F16, q=P, qs=512, k=P * 2, ks=256, v=P * 3, vs=256, n=3, heads=8, pos=P, ps=3, seq=P, slot=P,
              out=P * 4, os=512):
    r = r or paged.Rope(64, axes=[16, 16])
    return L.lib().fa_rope_append_axes(r._h, C.addressof(pg or pages()), layer, dt, q, qs, k, ks, v, vs, n, heads, pos, ps, seq, slot, out, os,
                                       None, None)


@pytest.mark.parametrize("bad", [dict(ps=2), dict(slot=None), dict(pos=None), dict(seq=None), dict(pos=P + 2), dict(q=None), dict(layer=2),
                                 dict(dt=5), dict(qs=511), dict(out=P + 512), dict(pg=pages(head_dim=128))], ids=str)
def test_append_with_axes_refuses(bad):
    assert call_axes(**bad) == L.ERR_INVALID
    assert "fa_rope_append_axes" in L.last_error()


def test_a_rope_of_several_axes_needs_their_positions():
    r = paged.Rope(64, axes=[16, 16])
    assert L.lib().fa_rope_append(r._h, C.addressof(pages()), 0, 1, P, 512, P * 2, 256, P * 3, 256, 3, 8, P, P, None, P * 4, 512, None,
                                  None) == L.ERR_INVALID
    assert call_axes(n=0, q=None, pos=None, seq=None, slot=None) == L.OK


# ------------------------------------------------------------------ the plan of a step
def call_plan(pool=None, seq=P, keep=P, add=P, n=3, rows=9, ln=P, ln_out=P, nf=P, nf_out=P, q_start=P, kv=P, last=P, pos=P, row_seq=P, slot=P,
              **fields):
    f = dict(page_table=0x20000, n_seq=4, max_pages=8, n_pages=100, free_pages=0x40000, free_cap=100)
    f.update(fields)
    made = L.fa_page_pool(**f)
    return L.lib().fa_step_plan(C.addressof(made) if pool is None else pool, seq, keep, add, n, rows, ln, ln_out, nf, nf_out, q_start, kv, last, pos, row_seq, slot, None, None)


@pytest.mark.parametrize("bad", [dict(pool=0), dict(page_table=None), dict(free_pages=None), dict(n_seq=0), dict(max_pages=0),
                                 dict(max_pages=(1 << 21) + 1), dict(n_pages=1 << 28), dict(n=4097), dict(n_seq=(1 << 18) + 1),
                                 dict(seq=None, n=5), dict(rows=1 << 31), dict(add=None), dict(ln=None), dict(ln_out=None), dict(nf=None),
                                 dict(nf_out=None), dict(q_start=None), dict(kv=None), dict(pos=None), dict(row_seq=None), dict(add=P + 1),
                                 dict(slot=P + 2), dict(page_table=0x20001)], ids=str)
def test_plan_refuses(bad):
    assert call_plan(**bad) in (L.ERR_INVALID, L.ERR_UNSUPPORTED)
    assert "fa_step_plan" in L.last_error()


# ------------------------------------------------------------------ sampling from given numbers
def call_sample(logits=P, dt=L.KV_F32, ld=100, m=3, vocab=100, rows=P, n=4, t=P, k=P, p=P, mp=P, u=P, ids=P, logs=P):
    return L.lib().fa_sample_logits(logits, dt, ld, m, vocab, rows, n, t, k, p, mp, u, ids, logs, None, None)


@pytest.mark.parametrize("bad", [dict(dt=3), dict(vocab=0), dict(vocab=393217, ld=1 << 20), dict(n=(1 << 20) + 1), dict(ld=99), dict(rows=None), dict(m=0),
                                 dict(logits=None), dict(u=None), dict(ids=None), dict(logits=P + 2), dict(u=P + 1), dict(ids=P + 2), dict(rows=P + 3),
                                 dict(t=P + 1), dict(k=P + 1), dict(p=P + 1), dict(mp=P + 1), dict(logs=P + 1)], ids=str)
def test_sample_logits_refuses(bad):
    assert call_sample(**bad) in (L.ERR_INVALID, L.ERR_UNSUPPORTED)
    assert "fa_sample_logits" in L.last_error()


def test_sampling_nothing():
    assert call_sample(n=0, logits=None, u=None, ids=None) == L.OK


# ------------------------------------------------------------------ what Python refuses before the library is called
def test_python_refuses_tensors_that_do_not_fit():
    torch = pytest.importorskip("torch")
    from fishai_engine import sampling
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    kv = paged.PagedKV(torch.zeros(1, 8, 2, 4, 16, 64, dtype=torch.float16), i(2, 4))
    args = dict(add=i(2), lengths=i(2), free_pages=i(8), n_free=i(1), q_start=i(3), kv_len=i(2), positions=i(5), row_seqs=i(5))
    for name, bad in (("add", i(2, 1)), ("lengths", i(3)), ("free_pages", i(2, 4)), ("n_free", i(2)), ("q_start", i(2)), ("kv_len", i(3)),
                      ("positions", torch.zeros(5)), ("row_seqs", i(4)), ("seqs", i(3)), ("keep", i(4)[::2]), ("slots", i(6)), ("last", i(1)),
                      ("lengths_out", i(1)), ("n_free_out", i(0)), ("err", i(2))):
        with pytest.raises(ValueError):
            paged.plan_step(kv, **{**args, name: bad})

    class OfACache:
        n_seq = 2

    with pytest.raises(ValueError, match="KVCache"):
        paged.plan_step(OfACache(), **args)
    x, f = torch.zeros(3, 50), lambda n: torch.zeros(n)  # noqa: E731
    good = dict(logits=x, u=f(3), ids=i(3))
    for name, bad in (("logits", x[0]), ("logits", x.t()), ("logits", x.double()), ("u", f(2)), ("u", i(3)), ("ids", f(3)), ("temperature", f(4)),
                      ("top_k", f(3)), ("top_p", f(6)[::2]), ("min_p", f(3).double()), ("rows", i(2)), ("logprobs", i(3)), ("err", i(3))):
        with pytest.raises(ValueError):
            sampling.sample_logits(**{**good, name: bad})
    r = paged.Rope(64, axes=[16, 16])
    q, k = torch.zeros(3, 512, dtype=torch.float16), torch.zeros(3, 256, dtype=torch.float16)
    for pos, slots in ((i(3), i(3)), (i(2, 3), None), (i(3, 2).t(), i(3)), (i(3, 3), i(3)), (f(6).view(2, 3), i(3)), (i(2, 6)[:, ::2], i(3))):
        with pytest.raises(ValueError):
            paged.rope_append(kv, 0, r, q, k, k, pos, i(3), torch.empty_like(q), slots=slots)
    with pytest.raises(ValueError):
        paged.attention(kv, 0, q, i(2), i(1), torch.empty_like(q), 3, torch.zeros(8, dtype=torch.uint8), window=5, sinks=2 ** 32)
