"""Calls at the edges of what the paged operators and the beam selection allow,
as the host takes them: no GPU needed, no pointer is read."""
import pytest

from fishai_engine import _lib as L
from test_cpu_paged import P, call_attn, call_rope, pages


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
