"""Refusals of the paged operators and the beam selection, and the rotary
frequencies, on the host: no GPU needed.  Every case is refused before any
pointer is looked at or any kernel runs."""
import ctypes as C
import math

import pytest

from fishai_engine import _lib as L
from fishai_engine import beam, paged


def pages(**kw):
    f = dict(base=0x10000, layer_stride=2 * 4 * 16 * 64 * 8, dtype=L.KV_F16, n_layers=2, n_pages=8, n_kv_heads=4, head_dim=64,
             page_table=0x20000, n_seq=2, max_pages=4)
    f.update(kw)
    return L.fa_pages(**f)


P = 0x30000  # an address that is never read


def rope(head_dim=64, **kw):
    return paged.Rope(head_dim, **kw)


def call_rope(pg=None, r=None, layer=0, dt=L.KV_F16, q=P, qs=512, k=P * 2, ks=256, v=P * 3, vs=256, n=3, heads=8, pos=P, seq=P,
              slot=None, out=P * 4, os=512):
    r = r or rope()
    return L.lib().fa_rope_append(r._h, C.addressof(pg or pages()), layer, dt, q, qs, k, ks, v, vs, n, heads, pos, seq, slot, out, os,
                                  None, None)


def call_attn(pg=None, layer=0, q=P, qs=512, heads=8, chunks=2, starts=P, kv=P, seq=None, n=3, max_q=3, scale=0.0, window=0,
              out=P * 4, os=512, ws=P * 16, ws_bytes=None):
    ws_bytes = L.lib().fa_attn_chunks_ws(64) if ws_bytes is None else ws_bytes
    return L.lib().fa_attn_chunks(C.addressof(pg or pages()), layer, q, qs, heads, chunks, starts, kv, seq, n, max_q, scale, window, out,
                                  os, ws, ws_bytes, None, None)


def call_beam(logits=P, dt=L.KV_F32, ld=100, batch=2, beams=3, vocab=100, scores=P, done=P, k=3, eos=2, pad=0, os=P * 2, op=P * 3,
              ot=P * 4, od=P * 5, ws=P * 16, ws_bytes=1 << 20):
    return L.lib().fa_beam_select(logits, dt, ld, batch, beams, vocab, scores, done, k, eos, pad, os, op, ot, od, ws, ws_bytes, None)


BAD_PAGES = [dict(base=None), dict(page_table=None), dict(dtype=3), dict(dtype=-1), dict(n_layers=0), dict(n_pages=0),
             dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(n_seq=0), dict(max_pages=0),
             dict(max_pages=(1 << 21) + 1), dict(base=0x10008), dict(layer_stride=2 * 4 * 16 * 64 * 8 - 8),
             dict(layer_stride=2 * 4 * 16 * 64 * 8 + 4), dict(n_kv_heads=40000), dict(n_layers=70000)]


@pytest.mark.parametrize("bad", BAD_PAGES, ids=[f"{k}={v}" for b in BAD_PAGES for k, v in b.items()])
def test_bad_pages_are_refused(bad):
    refused = (L.ERR_INVALID, L.ERR_UNSUPPORTED)
    assert call_rope(pages(**bad)) in refused
    assert call_attn(pages(**bad)) in refused
    assert L.lib().fa_pages_compact(C.addressof(pages(**bad)), P, P, P, 1, 4, None, None) in refused
    if not set(bad) & {"page_table", "n_seq", "max_pages"}:  # a copy does not look at the table
        assert L.lib().fa_pages_copy(C.addressof(pages(**bad)), P, P, None, 1, None, None) in refused


@pytest.mark.parametrize("bad", [dict(layer=2), dict(dt=5), dict(heads=0), dict(qs=511), dict(ks=255), dict(vs=255), dict(os=511),
                                 dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(seq=None), dict(out=None),
                                 dict(q=P + 1), dict(out=P * 4 + 1), dict(out=P + 512), dict(dt=L.KV_F32, out=P)], ids=str)
def test_rope_append_refuses(bad):
    assert call_rope(**bad) == L.ERR_INVALID
    assert L.last_error()


def test_rope_of_another_head_size_is_refused():
    assert call_rope(r=rope(128)) == L.ERR_INVALID


def test_null_handles():
    lib = L.lib()
    pg = pages()
    assert lib.fa_rope_append(None, C.addressof(pg), 0, 0, P, 1, P, 1, P, 1, 1, 1, P, P, None, P, 1, None, None) == L.ERR_INVALID
    assert lib.fa_rope_create(None, None) == L.ERR_INVALID
    assert lib.fa_rope_freqs(None, None, None) == L.ERR_INVALID
    assert lib.fa_kv_pages(None, None) == L.ERR_INVALID
    assert lib.fa_kv_fork(None, 0, 0) == L.ERR_INVALID
    assert lib.fa_kv_reorder(None, None, 1) == L.ERR_INVALID
    assert lib.fa_kv_truncate(None, 0, 0) == L.ERR_INVALID
    assert lib.fa_kv_compact(None, 0, None, 0) == L.ERR_INVALID
    assert lib.fa_kv_page_count(None, None, None) == L.ERR_INVALID
    lib.fa_rope_free(None)


@pytest.mark.parametrize("bad", [dict(layer=2), dict(heads=0), dict(heads=6), dict(qs=511), dict(os=500), dict(scale=-1.0),
                                 dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e31), dict(q=None), dict(starts=None), dict(kv=None),
                                 dict(out=None), dict(ws=None), dict(chunks=3), dict(ws_bytes=100), dict(ws=P * 16 + 8),
                                 dict(q=P + 1), dict(out=P), dict(out=P + 1024), dict(n=1 << 30)], ids=str)
def test_attention_refuses(bad):
    assert call_attn(**bad) == L.ERR_INVALID
    assert L.last_error()


@pytest.mark.parametrize("bad", [dict(dt=9), dict(beams=0), dict(beams=65), dict(k=0), dict(k=65), dict(vocab=0), dict(pad=100),
                                 dict(vocab=(1 << 30) + 1, ld=1 << 31), dict(ld=99), dict(logits=None), dict(scores=None),
                                 dict(os=None), dict(op=None), dict(ot=None), dict(ws=None), dict(ws_bytes=10),
                                 dict(ws=P * 16 + 8), dict(logits=P + 2), dict(k=2, os=P), dict(k=2, od=P), dict(batch=1 << 21)],
                         ids=str)
def test_beam_select_refuses(bad):
    assert call_beam(**bad) == L.ERR_INVALID
    assert L.last_error()


def test_nothing_to_do_is_fine_without_buffers():
    assert call_rope(n=0, q=None, k=None, v=None, out=None, pos=None, seq=None) == L.OK
    assert call_attn(n=0, q=None, out=None) == L.OK
    assert call_attn(chunks=0, starts=None, kv=None) == L.OK
    assert call_beam(batch=0, logits=None) == L.OK
    assert L.lib().fa_pages_copy(C.addressof(pages()), None, None, None, 0, None, None) == L.OK
    assert L.lib().fa_pages_compact(C.addressof(pages()), None, None, None, 0, 0, None, None) == L.OK


@pytest.mark.parametrize("bad", [dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(rot_dim=0), dict(rot_dim=3),
                                 dict(rot_dim=66), dict(base=1.0), dict(base=math.nan), dict(scaling="linear", factor=0.5),
                                 dict(scaling="ntk", factor=2.0, rot_dim=2), dict(scaling="llama3", factor=2.0, high_turns=1.0),
                                 dict(scaling="yarn", factor=2.0, beta_fast=1.0), dict(scaling="yarn", factor=2.0, context=0),
                                 dict(scaling="yarn", factor=2.0, attn_factor=-1.0), dict(scaling="llama3", factor=math.inf)], ids=str)
def test_rope_config_refuses(bad):
    with pytest.raises(L.FishaiError):
        paged.Rope(**{"head_dim": 64, **bad})
    with pytest.raises(ValueError):
        paged.Rope(64, layout="neither")


def want_freqs(rot, base, scaling, factor, context):
    out, scale = [], 1.0
    if scaling == "ntk":
        base *= factor ** (rot / (rot - 2))
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        turns = context * f / (2 * math.pi)
        if scaling == "linear":
            f /= factor
        elif scaling == "llama3":
            keep = 0.0 if turns < 1 else 1.0 if turns > 4 else (turns - 1) / 3
            f *= keep + (1 - keep) / factor
        elif scaling == "yarn":
            lo = max(0, math.floor(rot * math.log(context / (32 * 2 * math.pi)) / (2 * math.log(base))))
            hi = min(rot - 1, math.ceil(rot * math.log(context / (2 * math.pi)) / (2 * math.log(base))))
            slow = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            f *= 1 - slow + slow / factor
            scale = 0.1 * math.log(factor) + 1
        out.append(f)
    return out, scale


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "llama3", "yarn"])
@pytest.mark.parametrize("rot,base", [(64, 10000.0), (24, 500000.0), (2, 10.0), (4, 10000.0)])
def test_frequencies(scaling, rot, base):
    if scaling == "ntk" and rot < 4:
        pytest.skip("no such scaling")
    r = paged.Rope(64, rot_dim=rot, base=base, scaling=scaling, factor=8.0, context=8192)
    f, s = r.freqs()
    wf, ws = want_freqs(rot, base, scaling, 8.0, 8192)
    # a handful of 64-bit operations each
    assert all(abs(a - b) <= 1e-14 * b for a, b in zip(f, wf)) and len(f) == rot // 2
    assert abs(s - ws) <= 1e-15 * ws


def test_workspace_sizes():
    assert paged.workspace_bytes(0) == 0 and paged.workspace_bytes(512) == 0
    assert 0 < paged.workspace_bytes(64) < paged.workspace_bytes(128) < 96 << 20
    assert beam.workspace_bytes(0, 4, 100, 4) == 0 and beam.workspace_bytes(1, 65, 100, 4) == 0
    assert 0 < beam.workspace_bytes(32, 12, 200000, 16) < 16 << 20


def test_host_tensors_are_refused():
    """memory that is not a GPU's is an error, not a fault (on a machine without a GPU: no device)"""
    import torch
    kv = paged.PagedKV(torch.zeros(1, 4, 2, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32))
    q = torch.zeros(3, 128)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(L.FishaiError) as e:
        paged.rope_append(kv, 0, paged.Rope(64), q, q.clone(), q.clone(), i, i, q.clone())
    assert e.value.code in (L.ERR_INVALID, L.ERR_CUDA)


def test_wrappers_check_shapes_and_types():
    import torch
    pg = torch.zeros(1, 4, 2, 2, 16, 64)
    table = torch.zeros(2, 2, dtype=torch.int32)
    for bad in (torch.zeros(4, 2, 2, 16, 64), torch.zeros(1, 4, 3, 2, 16, 64), torch.zeros(1, 4, 2, 2, 8, 64), pg.double(),
                pg.transpose(3, 4)):
        with pytest.raises(ValueError):
            paged.PagedKV(bad, table)
    for bad in (table.long(), table.float(), table.t()[:1], table[0]):
        with pytest.raises(ValueError):
            paged.PagedKV(pg, bad)
    kv = paged.PagedKV(pg, table)
    r = paged.Rope(64)
    q, i = torch.zeros(3, 128), torch.zeros(3, dtype=torch.int32)
    ok = dict(q=q, k=q.clone(), v=q.clone(), positions=i, seqs=i, out=q.clone())
    for bad in (dict(k=q.half()), dict(out=q.half()), dict(positions=i.long()), dict(positions=i[:2]), dict(seqs=i.float()),
                dict(k=torch.zeros(3, 64)), dict(v=torch.zeros(2, 128)), dict(q=torch.zeros(3, 100)), dict(q=torch.zeros(128, 3).t())):
        with pytest.raises(ValueError):
            paged.rope_append(kv, 0, r, **{**ok, **bad})
    ws = torch.empty(paged.workspace_bytes(64), dtype=torch.uint8)
    ok = dict(q=q, q_start=i, kv_len=i[:2], out=q.clone(), max_q=3, workspace=ws)
    for bad in (dict(q=q.half()), dict(out=q.half()), dict(kv_len=i), dict(q_start=i.long()), dict(window=-1), dict(max_q=-1),
                dict(out=torch.zeros(2, 128)), dict(seqs=i), dict(q_start=i[:0])):
        with pytest.raises(ValueError):
            paged.attention(kv, 0, **{**ok, **bad})
    sc, ii = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)
    ok = dict(logits=torch.zeros(6, 10), scores=sc, done=ii, out_scores=sc, out_parents=ii, out_tokens=ii, out_done=ii, workspace=ws)
    for bad in (dict(logits=torch.zeros(5, 10)), dict(scores=sc.double()), dict(done=ii.long()), dict(out_tokens=ii[:1]),
                dict(logits=torch.zeros(10, 6).t())):
        with pytest.raises(ValueError):
            beam.select(**{**ok, **bad})
