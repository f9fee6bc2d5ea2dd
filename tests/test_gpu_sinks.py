"""Attention with a sliding window beside first positions that stay visible, against a plain 64-bit form."""
import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from fishai_engine import paged  # noqa: E402

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def call(pages, table, q, start, kvs, window, sinks, max_q=None, out=None, err=None, stream=0, ws=None, scale=0.0):
    out = torch.full_like(q, 7.0) if out is None else out
    ws = torch.empty(paged.workspace_bytes(pages.shape[5]), dtype=torch.uint8, device="cuda") if ws is None else ws
    most = max([b - a for a, b in zip(start, start[1:])] + [0])
    paged.attention(paged.PagedKV(pages, table), 0, q, i32(start), i32(kvs), out, max_q=max_q or most, workspace=ws, window=window, sinks=sinks,
                    err=err, stream=stream, scale=scale)
    return out


def check(qs, kvs, heads, kvh, hd, dtype, window, sinks, seed=0, wide=0, max_q=None):
    pages, table = R.make_cache(kvs, 1, kvh, hd, dtype, seed, junk=10 ** 6)
    pages, table = S.empty_gap(pages, table, qs, kvs, window, sinks)
    if wide:  # a table made for long sequences picks other kernels
        table = torch.cat((table, torch.full((len(kvs), wide - table.shape[1]), 10 ** 6, dtype=torch.int32, device="cuda")), 1)
    start = [sum(qs[:i]) for i in range(len(qs) + 1)]
    n = start[-1]
    q = randn(seed + 1, n + 2, heads * hd, dtype=dtype)  # two rows behind the last chunk
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = call(pages, table, q, start, kvs, window, sinks, err=err, max_q=max_q)
    want, tol = S.attention(pages, table, q, start, kvs, heads, 0.0, window, sinks)
    got = out.double().view_as(want)
    assert int(err) == 0 and bool((got[n:] == 7.0).all())
    assert not bool(torch.isnan(got).any())
    assert n == 0 or bool(((got - want).abs() <= tol)[:n].all()), float(((got - want).abs() - tol)[:n].max())


GEOM = [(8, 2, 64), (4, 4, 128), (32, 8, 128), (7, 1, 128), (6, 2, 72), (5, 5, 256)]


@pytest.mark.parametrize("heads,kvh,hd", GEOM)
@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 1), (40, 4), (64, 130), (500, 17)])
def test_single_tokens(heads, kvh, hd, t, window, sinks):
    check([1] * 7, [1, 2, 15, 16, 17, 333, 1000], heads, kvh, hd, R.TYPES[t], window, sinks, seed=1)


@pytest.mark.parametrize("heads,kvh,hd", GEOM)
@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 4), (33, 5), (100, 128), (16, 16)])
def test_mixed_chunks(heads, kvh, hd, t, window, sinks):
    check([1, 0, 5, 40, 129, 1, 300], [40, 33, 5, 100, 129, 700, 555], heads, kvh, hd, R.TYPES[t], window, sinks, seed=2)


# sinks and window edge to edge, one apart, overlapping; inside a page, a tile of 32, 64 and 128 positions and across them
@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("sinks", [1, 15, 16, 17, 63, 64, 127, 128, 129, 200, 255, 256, 257, 1000])
def test_gap_sizes(t, sinks):
    for q in (1, 6, 70, 200):
        for window in (1, 100, 500 - sinks - q if sinks + q < 499 else 3, 501 - sinks - q if sinks + q < 500 else 2):
            check([q], [500], 8, 2, 64, R.TYPES[t], max(1, window), sinks, seed=sinks)


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("wide", [0, 2048])
def test_long_caches(t, wide):
    """one launch of clusters and work split over the GPU; the first positions of a split item are a piece of their own"""
    dt = R.TYPES[t]
    check([1], [20000], 8, 2, 128, dt, 9000, 4, seed=5, wide=wide)
    check([1], [20000], 8, 8, 128, dt, 700, 333, seed=5, wide=wide)
    check([1, 1, 2], [9999, 3, 5000], 4, 1, 64, dt, 2000, 100, seed=6, wide=wide)
    check([200], [6000], 2, 1, 128, dt, 1500, 70, seed=8, wide=wide)
    check([1 + i % 3 for i in range(40)], [37 + i * 911 % 2960 for i in range(40)], 32, 8, 128, dt, 600, 4, seed=9, wide=wide)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_chunks(t, hd):
    """items of 128 and 256 rows of many tiles, among them some that begin in the first positions and some past them"""
    dt = R.TYPES[t]
    check([700, 900, 500, 130], [700, 1400, 600, 130], 32, 8, hd, dt, 200, 40, seed=16)
    check([33] * 60, [33 + 37 * i for i in range(60)], 16, 4, hd, dt, 90, 7, seed=17)
    check([1500], [4000], 16, 8, hd, dt, 1000, 150, seed=18)
    check([600], [600], 8, 8, hd, dt, 129, 128, seed=19)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_rows_that_see_nothing(t):
    check([9, 4, 150], [4, 0, 3], 8, 2, 128, R.TYPES[t], 2, 3, seed=4)


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 5), (10 ** 6, 3), (30, 10 ** 6), (2 ** 32 - 1, 2 ** 32 - 1), (30, 0)])
def test_without_a_gap_it_is_the_other_entry(t, window, sinks):
    """no window, one wider than the cache, first positions beyond its end, none: as fa_attn_chunks, bit for bit"""
    qs, kvs = [1, 40, 200], [300, 90, 250]
    pages, table = R.make_cache(kvs, 1, 2, 64, R.TYPES[t], 3)
    q, start = randn(4, 241, 8 * 64, dtype=R.TYPES[t]), [0, 1, 41, 241]
    a = call(pages, table, q, start, kvs, window, sinks)
    b = call(pages, table, q, start, kvs, 30 if sinks == 0 else 0, 0)
    assert torch.equal(a, b)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_unaligned_rows_and_scale(t):
    pages, table = R.make_cache([300], 1, 2, 64, R.TYPES[t], 12)
    for n in (1, 20, 150):
        buf = randn(5, n, 515, dtype=R.TYPES[t])
        res = torch.full((n, 515), 7.0, dtype=R.TYPES[t], device="cuda")
        call(pages, table, buf[:, 1:513], [0, n], [300], 50, 9, out=res[:, 1:513], scale=0.3)
        want, tol = S.attention(pages, table, buf[:, 1:513].contiguous(), [0, n], [300], 8, 0.3, 50, 9)
        assert bool(((res[:, 1:513].double().reshape(want.shape) - want).abs() <= tol).all())
        assert bool((res[:, 0] == 7.0).all()) and bool((res[:, 513:] == 7.0).all())


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_bad_pages_are_flagged_where_they_are_read(t):
    """a page of the first positions, of the window, and one between them that nobody looks at"""
    for q in (1, 40):
        kvs = [1000, 1000]
        pages, table = R.make_cache(kvs, 1, 2, 64, R.TYPES[t], 42)
        x, start = randn(10, 2 * q, 4 * 64, dtype=R.TYPES[t]), [0, q, 2 * q]
        good = call(pages, table, x, start, kvs, 100, 20)
        for entry, flag in ((0, paged.FLAG_PAGE), (1, paged.FLAG_PAGE), (2, 0), (30, 0), (62, paged.FLAG_PAGE)):
            bad = table.clone()
            bad[1, entry] = pages.shape[1]
            err = torch.zeros(1, dtype=torch.int32, device="cuda")
            out = call(pages, bad, x, start, kvs, 100, 20, err=err)
            assert int(err) == flag
            assert torch.equal(out[:q], good[:q])
            assert flag or torch.equal(out, good)


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_captured_and_replayed_on_another_stream(t):
    qs, kvs = [1, 50, 1], [5000, 300, 77]
    pages, table = R.make_cache(kvs, 1, 2, 128, R.TYPES[t], 21)
    kv, start, ln = paged.PagedKV(pages, table), i32([0, 1, 51, 52]), i32(kvs)
    q = randn(1, 52, 8 * 128, dtype=R.TYPES[t])
    out, ws = torch.zeros_like(q), torch.empty(paged.workspace_bytes(128), dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        paged.attention(kv, 0, q, start, ln, out, max_q=50, workspace=ws, window=64, sinks=4, stream=st.cuda_stream)
    for seed in (2, 3):
        q.copy_(randn(seed, 52, 8 * 128, dtype=R.TYPES[t]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want, tol = S.attention(pages, table, q, [0, 1, 51, 52], kvs, 8, 0.0, 64, 4)
        assert bool(((out.double().view_as(want) - want).abs() <= tol).all())


def test_repeated_calls_give_the_same_bits():
    qs, kvs = [1, 200, 1, 700], [9000, 3000, 100, 2000]
    pages, table = R.make_cache(kvs, 1, 2, 128, torch.bfloat16, 22)
    q = randn(1, sum(qs), 8 * 128, dtype=torch.bfloat16)
    start = [sum(qs[:i]) for i in range(5)]
    first = call(pages, table, q, start, kvs, 700, 40)
    for _ in range(5):
        assert torch.equal(call(pages, table, q, start, kvs, 700, 40), first)


@pytest.mark.parametrize("q", [1, 40, 200])
def test_pages_beyond_32_bits_of_elements(q):
    """a small cache whose pages lie at the end of a large one"""
    small, table = R.make_cache([700, 333], 1, 8, 128, torch.float16, 31)
    n = small.shape[1]
    pages = torch.empty(1, 2 ** 17 + 9000, 2, 8, 16, 128, dtype=torch.float16, device="cuda")  # 4.6e9 elements
    pages[0, -n:] = small[0]
    moved = table + (pages.shape[1] - n)
    x = randn(1, 2 * q, 16 * 128, dtype=torch.float16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = call(pages, moved, x, [0, q, 2 * q], [700, 333], 100, 20, err=err)
    assert int(err) == 0 and torch.equal(out, call(small, table, x, [0, q, 2 * q], [700, 333], 100, 20))
    want, tol = S.attention(small, table, x, [0, q, 2 * q], [700, 333], 16, 0.0, 100, 20)
    assert bool(((out.double().view_as(want) - want).abs() <= tol).all())
    del pages
    torch.cuda.empty_cache()
