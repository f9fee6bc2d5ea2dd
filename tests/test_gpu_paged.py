"""Operators on paged K/V (rotary append, attention of chunks, page copies,
compaction) and the beam selection against plain 64-bit forms."""
import ctypes as C
import math
import random

import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402
from fishai_engine import _lib as L  # noqa: E402
from fishai_engine import beam, paged  # noqa: E402

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def same_bits(a, b):
    """equal, NaN included"""
    kind = {4: torch.int32, 2: torch.int16}[a.element_size()]
    return bool((a.contiguous().view(kind) == b.contiguous().view(kind)).all())


# ------------------------------------------------------------------ rotary append
def rope_case(tokens, heads, kvh, hd, tin, tout, seed=0, spare_row=False, fused=True, **kw):
    r = paged.Rope(hd, **kw)
    rng = random.Random(seed)
    n_seq = 3
    lens = [tokens + 20 + i for i in range(n_seq)]
    pages, table = R.make_cache(lens, 2, kvh, hd, tout, seed)
    before = pages.clone()
    seqs = [rng.randrange(n_seq) for _ in range(tokens)]
    used = [list(range(n)) for n in lens]
    for u in used:
        rng.shuffle(u)
    slots = [used[s].pop() for s in seqs]
    pos = [rng.choice([0, 1, s, 10 ** 6 + s, 2 ** 31 - 1 - s]) for s in slots]
    if spare_row:
        seqs[tokens // 2] = paged.NO_TOKEN
    w = (heads + 2 * kvh) * hd
    rows = randn(seed + 1, tokens, w, dtype=tin)
    q, k, v = rows[:, : heads * hd], rows[:, heads * hd: (heads + kvh) * hd], rows[:, (heads + kvh) * hd:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    out = torch.full((tokens, heads * hd), 7.0, dtype=tout, device="cuda")
    return dict(r=r, pages=pages, before=before, table=table, seqs=seqs, slots=slots, pos=pos, q=q, k=k, v=v, out=out)


def rope_check(c, heads, kvh, hd, layout):
    freqs, scale = c["r"].freqs()
    live = torch.tensor([s >= 0 for s in c["seqs"]], device="cuda")
    pos = torch.tensor(c["pos"], device="cuda")
    u = R.half_step(c["out"].dtype)
    # sines and cosines: the angle's fraction of a turn is rounded once to f32 (2^-25 of at most 1/2 turn, times 2 pi
    # < 2^-22.3), sincospi is good to 2 ulp (2^-23), three f32 operations follow (3 2^-24) and the scale (2^-24)
    e = (2 ** -22.3 + 2 ** -22 + 5 * 2 ** -24)

    def close(got, x, n):
        want, size = R.rope_rows(x, pos, freqs, scale, c["r"].rot_dim, layout, n, hd)
        tol = u * want.abs() + (1 + u) * e * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)
        bad = ((got.double().view_as(want) - want).abs() > tol)[live]
        assert not bool(bad.any())

    close(c["out"], c["q"], heads)
    assert bool((c["out"][~live] == 7.0).all())
    want = c["before"].clone()
    got_k = torch.zeros(len(c["seqs"]), kvh, hd, dtype=c["out"].dtype, device="cuda")
    for t, (s, sl) in enumerate(zip(c["seqs"], c["slots"])):
        if s < 0:
            continue
        page = int(c["table"][s, sl // 16])
        got_k[t] = c["pages"][1, page, 0, :, sl % 16]
        want[1, page, 0, :, sl % 16] = got_k[t]
        want[1, page, 1, :, sl % 16] = c["v"][t].float().view(kvh, hd).to(want.dtype)
    close(got_k.flatten(1), c["k"], kvh)
    assert same_bits(c["pages"], want)  # V exactly, and nothing else touched


ROPES = [dict(), dict(layout="half"), dict(rot_dim=24), dict(rot_dim=2, layout="half"), dict(rot_dim=40, layout="half", scaling="linear", factor=4.0),
         dict(scaling="llama3", base=500000.0, factor=8.0), dict(layout="half", scaling="yarn", factor=16.0, context=4096),
         dict(scaling="ntk", factor=3.0, rot_dim=12)]


@pytest.mark.parametrize("kw", ROPES, ids=str)
@pytest.mark.parametrize("tin,tout", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "bf16"), ("bf16", "f32")])
def test_rope_append(kw, tin, tout):
    c = rope_case(9, 6, 2, 64, R.TYPES[tin], R.TYPES[tout], seed=len(str(kw)), spare_row=True, **kw)
    paged.rope_append(paged.PagedKV(c["pages"], c["table"]), 1, c["r"], c["q"], c["k"], c["v"], i32(c["pos"]), i32(c["seqs"]), c["out"],
                      slots=i32(c["slots"]))
    rope_check(c, 6, 2, 64, kw.get("layout", "interleaved"))


@pytest.mark.parametrize("tokens,heads,kvh,hd", [(1, 1, 1, 8), (1, 32, 8, 128), (5, 3, 3, 256), (700, 7, 1, 72), (64, 64, 8, 128)])
def test_rope_append_sizes(tokens, heads, kvh, hd):
    c = rope_case(tokens, heads, kvh, hd, torch.float16, torch.float16, seed=tokens, fused=False)
    paged.rope_append(paged.PagedKV(c["pages"], c["table"]), 1, c["r"], c["q"].view(tokens, heads, hd), c["k"], c["v"], i32(c["pos"]),
                      i32(c["seqs"]), c["out"], slots=i32(c["slots"]))
    rope_check(c, heads, kvh, hd, "interleaved")


def test_rope_append_in_place_and_unaligned_rows():
    for off in (0, 1):
        c = rope_case(11, 4, 2, 64, torch.bfloat16, torch.bfloat16, seed=3)
        wide = torch.empty(11, 8 * 64 + 3, dtype=torch.bfloat16, device="cuda")
        wide[:, off: off + 4 * 64] = c["q"]
        q = wide[:, off: off + 4 * 64]
        c["q"] = q.clone()
        paged.rope_append(paged.PagedKV(c["pages"], c["table"]), 1, c["r"], q, c["k"], c["v"], i32(c["pos"]), i32(c["seqs"]), q,
                          slots=i32(c["slots"]))
        c["out"] = q.contiguous()
        rope_check(c, 4, 2, 64, "interleaved")


def test_rope_append_flags_what_it_refuses():
    kvh, hd = 2, 64
    pages, table = R.make_cache([40, 40], 1, kvh, hd, torch.float16, 1)
    table[1, 1] = pages.shape[1]  # no such page
    before = pages.clone()
    q, k = randn(1, 4, 2 * hd, dtype=torch.float16), randn(2, 4, kvh * hd, dtype=torch.float16)
    for seqs, slots, flag in (([2, 0, 0, 0], [3, 4, 5, 6], L.FLAG_RANGE), ([0, 0, 0, 0], [48, 4, 5, 6], L.FLAG_RANGE),
                              ([1, 0, 0, 0], [16, 4, 5, 6], L.FLAG_PAGE)):
        pages.copy_(before)
        err, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full_like(q, 7.0)
        paged.rope_append(paged.PagedKV(pages, table), 0, paged.Rope(hd), q, k, k, i32([1, 2, 3, 4]), i32(seqs), out, slots=i32(slots), err=err)
        assert int(err) == flag
        assert bool((out[0] == 7.0).all()) and not bool((out[1:] == 7.0).all(1).any())
        changed = (pages.view(torch.int16) != before.view(torch.int16)).any(-1).any(0).any(1).any(1)  # [page, slot]
        assert int(changed.sum()) == 3


# ------------------------------------------------------------------ attention
def attn(pages, table, q, q_start, kv_len, heads, max_q=None, seqs=None, scale=0.0, window=0, layer=0, out=None, err=None, stream=0,
         workspace=None):
    hd = pages.shape[5]
    out = torch.full_like(q, 7.0) if out is None else out
    ws = torch.empty(paged.workspace_bytes(hd), dtype=torch.uint8, device="cuda") if workspace is None else workspace
    most = max([b - a for a, b in zip(q_start, q_start[1:])] + [0])
    paged.attention(paged.PagedKV(pages, table), layer, q, i32(q_start), i32(kv_len), out, max_q=most if max_q is None else max_q,
                    workspace=ws, seqs=None if seqs is None else i32(seqs), scale=scale, window=window, err=err, stream=stream)
    return out


def attn_check(qs, kvs, heads, kvh, hd, dtype, window=0, scale=0.0, seed=0, **kw):
    pages, table = R.make_cache(kvs, 1, kvh, hd, dtype, seed, junk=10 ** 6)
    err = kw.setdefault("err", torch.zeros(1, dtype=torch.int32, device="cuda"))
    start = [sum(qs[:i]) for i in range(len(qs) + 1)]
    q = randn(seed + 1, start[-1] + 2, heads * hd, dtype=dtype)  # two rows behind the last chunk
    out = attn(pages, table, q, start, kvs, heads, window=window, scale=scale, **kw)
    want, tol = R.attention(pages, table, 0, q, i32(start), i32(kvs), None, heads, scale, window)
    got = out.double().view_as(want)
    n = start[-1]
    assert int(err) == 0
    assert bool((got[n:] == 7.0).all())
    off = ((got - want).abs() - tol)[:n]
    assert not bool(torch.isnan(got).any())
    assert n == 0 or float(off.max()) <= 0, (float(off.max()), int((off > 0).sum()))


GEOM = [(8, 2, 64), (4, 4, 128), (32, 8, 128), (7, 1, 128), (16, 2, 64), (6, 2, 72), (3, 1, 8), (5, 5, 256)]


@pytest.mark.parametrize("heads,kvh,hd", GEOM)
@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_attention_single_tokens(heads, kvh, hd, t):
    attn_check([1] * 7, [1, 2, 15, 16, 17, 333, 1000], heads, kvh, hd, R.TYPES[t], seed=1)


@pytest.mark.parametrize("heads,kvh,hd", GEOM)
@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_attention_mixed_chunks(heads, kvh, hd, t):
    attn_check([1, 0, 5, 40, 129, 1, 300], [40, 33, 5, 100, 129, 700, 555], heads, kvh, hd, R.TYPES[t], seed=2)


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (16, 4, 128), (2, 2, 40)])
@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 5000])
def test_attention_window(heads, kvh, hd, t, window):
    attn_check([1, 3, 150, 33], [200, 3, 170, 444], heads, kvh, hd, R.TYPES[t], window=window, seed=3)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("qs,kvs", [([4, 1, 20], [0, 0, 0]), ([9, 1, 2], [4, 0, 1]), ([150], [3]), ([0, 0], [5, 0])])
def test_attention_rows_that_see_nothing(t, qs, kvs):
    """a chunk longer than its cache: the tokens before position 0 see nothing and give zeros"""
    attn_check(qs, kvs, 8, 2, 128, R.TYPES[t], seed=4)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_attention_chunk_lengths(n, t):
    attn_check([n], [n + 37], 8, 2, 128, R.TYPES[t], seed=n)
    attn_check([n], [n], 4, 4, 64, R.TYPES[t], seed=n)


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_attention_split_long_cache(t):
    """one token, a long cache: the work is split over the GPU and joined"""
    attn_check([1], [20000], 8, 2, 128, R.TYPES[t], seed=5)
    attn_check([1, 1], [9999, 3], 4, 1, 64, R.TYPES[t], seed=6)
    attn_check([1], [12345], 8, 1, 128, R.TYPES[t], window=7000, seed=7)
    attn_check([5], [8000], 8, 8, 128, R.TYPES[t], seed=8)
    attn_check([200], [6000], 2, 1, 128, R.TYPES[t], seed=8)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_several_items_a_cta(t, hd):
    """more items than SMs, of one to a dozen tiles: buffers and barriers are used again and again"""
    attn_check([700, 900, 500, 130], [700, 1400, 600, 130], 32, 8, hd, R.TYPES[t], seed=16)
    attn_check([33] * 60, [33 + 7 * i for i in range(60)], 16, 4, hd, R.TYPES[t], seed=17)
    attn_check([2000], [2000], 16, 8, hd, R.TYPES[t], window=300, seed=18)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_batches_of_long_caches(t, hd):
    """each CTA goes round its ring of copies dozens of times, over several items"""
    kvs = [37 + i * 911 % 2960 for i in range(40)]
    attn_check([1] * 40, kvs, 32, 8, hd, R.TYPES[t], seed=19)
    attn_check([1 + i % 3 for i in range(40)], kvs, 64, 8, hd, R.TYPES[t], seed=20)
    attn_check([1 + i % 8 for i in range(40)], kvs, 32, 8, hd, R.TYPES[t], window=1500, seed=21)
    attn_check([16 - i % 3 for i in range(40)], kvs, 16, 4, hd, R.TYPES[t], seed=22)


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_attention_many_chunks(t):
    rng = random.Random(3)
    kvs = [rng.randint(1, 60) for _ in range(700)]
    attn_check([rng.choice([1, 1, 2, min(9, k)]) if k > 1 else 1 for k in kvs], kvs, 4, 1, 64, R.TYPES[t], seed=9)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", [(2, 1, 64), (12, 3, 128), (16, 2, 80), (4, 4, 256)])
@pytest.mark.parametrize("qs,kvs,window", [([1], [511], 0), ([2], [2], 0), ([1, 0, 1], [130, 9, 1], 0), ([2, 1], [0, 700], 0),
                                           ([1, 2], [90, 1], 33), ([1], [8000], 0), ([1], [40], 1)])
def test_attention_of_few_chunks_in_a_small_and_a_large_table(t, heads, kvh, hd, qs, kvs, window):
    """the kernels for short caches and those for long ones (the table's width decides), rows that see nothing among them"""
    dtype = R.TYPES[t]
    pages, table = R.make_cache(kvs, 2, kvh, hd, dtype, 41, junk=10 ** 6)
    wide = torch.full((len(kvs), 1100), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    start = [sum(qs[:i]) for i in range(len(qs) + 1)]
    q = randn(9, start[-1] + 1, heads * hd, dtype=dtype)
    want, tol = R.attention(pages, table, 1, q, i32(start), i32(kvs), None, heads, 0.0, window)
    for tb in (table, wide):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = attn(pages, tb, q, start, kvs, heads, max_q=max(qs), window=window, layer=1, out=torch.full_like(q, 7.0), err=err)
        assert int(err) == 0 and bool((out[start[-1]:] == 7.0).all())
        got = out[: start[-1]].double().view(-1, heads, hd)
        assert bool(((got - want[: start[-1]]).abs() <= tol[: start[-1]]).all())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 1, 64), (12, 3, 128), (32, 8, 128)])
@pytest.mark.parametrize("qs,kvs,window", [([17], [17], 0), ([70], [70], 0), ([20], [900], 0), ([33, 0, 5], [400, 9, 5], 0), ([20, 4], [0, 0], 0),
                                           ([150], [3], 0), ([40, 9], [130, 4], 33), ([64], [300], 1), ([128, 1], [128, 200], 0)])
def test_attention_of_short_chunks_in_a_small_and_a_large_table(t, heads, kvh, hd, qs, kvs, window):
    """more than 16 rows a kv head: the kernel for short calls and those for long caches, rows of any alignment"""
    dtype = R.TYPES[t]
    pages, table = R.make_cache(kvs, 1, kvh, hd, dtype, 43, junk=10 ** 6)
    wide = torch.full((len(kvs), 1100), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    start = [sum(qs[:i]) for i in range(len(qs) + 1)]
    for spare in (0, 3):  # rows 16-byte aligned, and not
        q = randn(11, start[-1] + 1, heads * hd + spare, dtype=dtype)[:, spare:]
        want, tol = R.attention(pages, table, 0, q.contiguous(), i32(start), i32(kvs), None, heads, 0.0, window)
        for tb in (table, wide):
            err, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full_like(q, 7.0)
            attn(pages, tb, q, start, kvs, heads, window=window, out=out, err=err)
            assert int(err) == 0 and bool((out[start[-1]:] == 7.0).all())
            got = out[: start[-1]].double().view(-1, heads, hd)
            assert bool(((got - want[: start[-1]]).abs() <= tol[: start[-1]]).all())


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_attention_refuses_and_flags_in_a_small_table_too(t):
    """a chunk that is refused beside one that is not, and a page out of range, where each item is a cluster"""
    dtype = R.TYPES[t]
    pages, table = R.make_cache([40, 50], 1, 2, 64, dtype, 42)
    q = randn(10, 4, 4 * 64, dtype=dtype)
    good = attn(pages, table, q, [0, 1, 2], [40, 50], 4)
    for start, lens, seqs, flag in (([0, 1, 2], [40, 10 ** 6], None, paged.FLAG_RANGE), ([0, 1, 2], [40, 50], [0, 2], paged.FLAG_RANGE),
                                    ([0, 1, 9], [40, 50], None, paged.FLAG_RANGE)):
        err, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full_like(q, 7.0)
        attn(pages, table, q, start, lens, 4, max_q=1, seqs=seqs, out=out, err=err)
        assert int(err) == flag and same_bits(out[:1], good[:1]) and bool((out[1:] == 7.0).all())
    bad = table.clone()
    bad[1, 2] = pages.shape[1]
    err, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full_like(q, 7.0)
    attn(pages, bad, q, [0, 1, 2], [40, 50], 4, out=out, err=err)
    assert int(err) == paged.FLAG_PAGE and same_bits(out[:1], good[:1]) and bool((out[2:] == 7.0).all())


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_attention_scale_and_sharp_scores(t):
    attn_check([3, 200], [300, 260], 8, 2, 64, R.TYPES[t], scale=1.5, seed=10)
    attn_check([3, 200], [300, 260], 8, 2, 64, R.TYPES[t], scale=0.001, seed=10)


def test_attention_sequence_numbers_and_layers():
    pages, table = R.make_cache([50, 80, 33], 3, 2, 128, torch.float16, 11)
    q = randn(1, 6, 4 * 128, dtype=torch.float16)
    start, kv, seqs = [0, 2, 3, 6], [80, 33, 79], [1, 2, 1]  # one sequence twice
    for layer in (0, 2):
        out = attn(pages, table, q, start, kv, 4, seqs=seqs, layer=layer)
        want, tol = R.attention(pages, table, layer, q, i32(start), i32(kv), seqs, 4, 0.0, 0)
        assert bool(((out.double().view_as(want) - want).abs() <= tol).all())


@pytest.mark.parametrize("n", [1, 20, 150])
def test_attention_strides_and_alignment(n):
    """rows of a wider buffer, aligned to 16 bytes and not"""
    pages, table = R.make_cache([200], 1, 2, 64, torch.bfloat16, 12)
    for off, wide in ((0, 520), (8, 528), (1, 515)):
        buf = randn(5, n, wide, dtype=torch.bfloat16)
        res = torch.full((n, wide), 7.0, dtype=torch.bfloat16, device="cuda")
        q, out = buf[:, off: off + 512], res[:, off: off + 512]
        attn(pages, table, q, [0, n], [200], 8, out=out)
        want, tol = R.attention(pages, table, 0, q, i32([0, n]), i32([200]), None, 8, 0.0, 0)
        assert bool(((out.double().reshape(want.shape) - want).abs() <= tol).all())
        keep = torch.ones(wide, dtype=torch.bool, device="cuda")
        keep[off: off + 512] = False
        assert bool((res[:, keep] == 7.0).all())


def test_attention_refused_chunks_are_flagged_and_left():
    pages, table = R.make_cache([64, 64, 64], 1, 2, 64, torch.float16, 13)
    q = randn(1, 12, 4 * 64, dtype=torch.float16)
    for start, kv, seqs, max_q, bad in (([0, 4, 8, 12], [60, 65, 60], None, 4, 1),   # longer than the table
                                        ([0, 4, 8, 12], [60, 60, 60], [0, 3, 2], 4, 1),  # no such sequence
                                        ([0, 4, 8, 13], [60, 60, 60], None, 5, 2),   # rows that q has not
                                        ([0, 2, 8, 12], [60, 60, 60], None, 4, 1)):  # longer than max_q
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = attn(pages, table, q, start, kv, 4, max_q=max_q, seqs=seqs, err=err)
        assert int(err) == L.FLAG_RANGE
        for c in range(3):
            rows = out[start[c]: start[c + 1]]
            assert bool((rows == 7.0).all()) == (c == bad)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    table[1, 2] = pages.shape[1]
    out = attn(pages, table, q, [0, 4, 8, 12], [60, 60, 60], 4, err=err)
    assert int(err) == L.FLAG_PAGE
    want, tol = R.attention(pages, table.clamp_max(0) + table * (table < pages.shape[1]), 0, q, i32([0, 4, 8, 12]), i32([60, 60, 60]), None,
                            4, 0.0, 0)
    ok = (out.double().view_as(want) - want).abs() <= tol
    assert bool(ok[:4].all()) and bool(ok[8:].all())


def test_attention_masked_places_may_hold_anything():
    """positions behind kv_len and before every token's window hold NaN and infinities (make_cache fills unused slots with NaN)"""
    for dtype in (torch.float16, torch.float32):
        pages, table = R.make_cache([300], 1, 2, 128, dtype, 14)
        first = table[0, : 4].long()  # positions 0 .. 63, before the windows below
        pages[:, first] = float("inf")
        for n in (1, 30, 140):
            q = randn(2, n, 4 * 128, dtype=dtype)
            out = attn(pages, table, q, [0, n], [299], 4, window=299 - n - 64)
            want, tol = R.attention(pages, table, 0, q, i32([0, n]), i32([299]), None, 4, 0.0, 299 - n - 64)
            assert bool(((out.double().view_as(want) - want).abs() <= tol).all())


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_attention_is_repeatable_and_captured(t):
    pages, table = R.make_cache([3000, 100, 700], 1, 2, 128, R.TYPES[t], 15)
    q = randn(3, 160, 8 * 128, dtype=R.TYPES[t])
    start, kv = i32([0, 1, 3, 160]), i32([3000, 100, 700])
    kvv = paged.PagedKV(pages, table)
    ws = torch.empty(paged.workspace_bytes(128), dtype=torch.uint8, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)
    paged.attention(kvv, 0, q, start, kv, a, 160, ws)
    ws.fill_(0xFF)  # what the workspace held does not matter
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        paged.attention(kvv, 0, q, start, kv, b, 160, ws, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        b.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        assert same_bits(a, b)
    # new lengths in the same buffers: the graph follows them
    kv.copy_(i32([2000, 50, 600]))
    g.replay()
    paged.attention(kvv, 0, q, start, kv, a, 160, ws)
    torch.cuda.synchronize()
    assert same_bits(a, b)


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layers,kvh,hd", [(1, 1, 8), (3, 2, 64), (2, 8, 128), (2, 3, 256)])
def test_copy_pages(t, layers, kvh, hd):
    pages, table = R.make_cache([16 * 40], layers, kvh, hd, R.TYPES[t], 20)
    ids = table[0].tolist()
    src, dst = ids[:17], ids[20:37]
    slots = list(range(17))  # none .. a whole page
    want = pages.clone()
    for a, b, n in zip(src, dst, slots):
        want[:, b, :, :, :n] = want[:, a, :, :, :n]
    kv = paged.PagedKV(pages, table)
    paged.copy_pages(kv, i32(src), i32(dst), slots=i32(slots))
    assert same_bits(pages, want)
    paged.copy_pages(kv, i32(src), i32(dst))
    for a, b in zip(src, dst):
        want[:, b] = want[:, a]
    assert same_bits(pages, want)


def test_copy_pages_refuses_bad_numbers():
    pages, table = R.make_cache([16 * 8], 2, 2, 64, torch.float16, 21)
    n = pages.shape[1]
    want = pages.clone()
    for src, dst, slots, flag in (([n, 0], [1, 2], [16, 16], L.FLAG_PAGE), ([1, 0], [-1, 2], [16, 16], L.FLAG_PAGE),
                                  ([1, 0], [3, 2], [17, 16], L.FLAG_RANGE)):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        paged.copy_pages(paged.PagedKV(pages, table), i32(src), i32(dst), slots=i32(slots), err=err)
        want[:, 2] = want[:, 0]
        assert int(err) == flag and same_bits(pages, want)


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("layers,kvh,hd", [(1, 1, 8), (3, 2, 64), (2, 4, 256)])
def test_compact(t, layers, kvh, hd):
    lens = [1, 16, 17, 500, 130]
    pages, table = R.make_cache(lens, layers, kvh, hd, R.TYPES[t], 22)
    rng = random.Random(1)
    keeps = [[p for p in range(n) if rng.random() < 0.5] for n in lens]
    keeps[0] = [0]
    keeps[2] = [16]
    keeps[4] = list(range(130))
    order = [3, 1, 0, 2, 4]
    want = pages.clone()
    for s in order:
        for j, p in enumerate(keeps[s]):
            want[:, table[s, j // 16], :, :, j % 16] = pages[:, table[s, p // 16], :, :, p % 16]
    flat = [p for s in order for p in keeps[s]]
    start = [sum(len(keeps[s]) for s in order[:i]) for i in range(6)]
    paged.compact(paged.PagedKV(pages, table), i32(order), i32(flat), i32(start))
    assert same_bits(pages, want)


def test_compact_refuses_bad_lists():
    pages, table = R.make_cache([64, 64], 1, 2, 64, torch.float16, 23)
    before = pages.clone()
    kv = paged.PagedKV(pages, table)
    for seqs, keep, start, same in (([2], [1, 2], [0, 2], True), ([0], [1, 2], [0, 3], True), ([0], [1, 2], [1, 0], True),
                                    ([0], [70], [0, 1], True), ([0], [0, 1, 1], [0, 3], True), ([0], [0, 5, 4], [0, 3], False)):
        pages.copy_(before)
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        paged.compact(kv, i32(seqs), i32(keep), i32(start), err=err)
        assert int(err) == L.FLAG_RANGE
        assert same_bits(pages, before) == same


# ------------------------------------------------------------------ beam selection
def beam_run(logits, scores, done, k, eos=2, pad=0):
    nb, beams = scores.shape
    o = [torch.full((nb, k), 99, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32, torch.int32)]
    ws = torch.empty(max(16, beam.workspace_bytes(nb, beams, logits.shape[1], k)), dtype=torch.uint8, device="cuda")
    beam.select(logits, scores, done, *o, workspace=ws, eos=eos, pad=pad)
    return [x.cpu() for x in o]


def beam_check(logits, scores, done, k, eos=2, pad=0):
    got = beam_run(logits, scores, done, k, eos, pad)
    want = R.beam_select(logits.cpu(), scores.cpu(), None if done is None else done.cpu(), k, eos, pad)
    for g, w in zip(got[1:], want[1:]):
        assert torch.equal(g, w)
    # the sum of a row in f32 (each thread's part at most a few hundred terms, exp good to 2^-22): below 2^-17 of the log;
    # one rounding of the score
    fin = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(got[0]), fin)
    assert bool(((got[0].double() - want[0]).abs()[fin] <= 2 ** -17 + 2 ** -24 * want[0].abs()[fin]).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nb,beams,vocab,k", [(1, 1, 1, 1), (1, 4, 128256, 4), (3, 5, 32000, 7), (2, 8, 777, 64), (5, 64, 300, 64),
                                              (40, 3, 4097, 2), (1, 1, 50000, 64), (2, 2, 3, 8), (1, 2, 300001, 16)])
def test_beam_select(t, nb, beams, vocab, k):
    x = (3 * randn(vocab, nb * beams, vocab)).to(R.TYPES[t])
    scores = -5 * torch.rand(nb, beams, device="cuda")
    done = (torch.rand(nb, beams, device="cuda") < 0.2).int()
    beam_check(x, scores, done, k, eos=min(2, vocab - 1), pad=0)
    beam_check(x, scores, None, k, eos=-1, pad=vocab - 1)


@pytest.mark.parametrize("nb,beams,vocab,k", [(1, 12, 128256, 16), (1, 1, 128256, 64), (1, 64, 128256, 64), (3, 20, 9000, 33), (2, 40, 40000, 64)])
def test_beam_select_of_many_lists(nb, beams, vocab, k):
    """requests whose rows are split: more candidates than threads"""
    x = 3 * randn(vocab + k, nb * beams, vocab)
    scores = -0.1 * torch.rand(nb, beams, device="cuda", generator=torch.Generator("cuda").manual_seed(k))
    done = torch.zeros(nb, beams, dtype=torch.int32, device="cuda")
    done[:, beams // 2] = beams > 2
    beam_check(x, scores, done, k)


@pytest.mark.parametrize("nb,beams,vocab,k", [(1, 2, 128256, 64), (1, 64, 70000, 64), (1, 12, 50000, 16)])
def test_beam_select_of_equal_candidates(nb, beams, vocab, k):
    """every candidate as good as the next: more of them reach the bound than are placed at once"""
    x = torch.zeros(nb * beams, vocab, device="cuda")
    beam_check(x, torch.zeros(nb, beams, device="cuda"), None, k)
    x[:, ::7] = 1.0
    beam_check(x, torch.zeros(nb, beams, device="cuda"), None, k)


def test_beam_select_ties_go_to_the_lowest():
    for vocab in (50, 5000, 70000):
        x = torch.zeros(6, vocab, device="cuda")
        scores = torch.zeros(2, 3, device="cuda")
        got = beam_run(x, scores, None, 5)
        assert got[1].tolist() == [[0] * 5] * 2 and got[2].tolist() == [list(range(5))] * 2
        x[:, vocab // 2:] = 1.0
        got = beam_run(x, scores, None, 4)
        assert got[2].tolist() == [[vocab // 2 + i for i in range(4)]] * 2
        scores[:, 0] = -1.0  # beams 1 and 2 are equal
        got = beam_run(x, scores, None, 3)
        assert got[1].tolist() == [[1] * 3] * 2


def test_beam_select_rising_and_falling_rows():
    """rows in which every tile beats, or ties with, what came before"""
    v = torch.arange(60000, device="cuda", dtype=torch.float32)
    x = torch.stack([v / 6000, -v / 6000, (v % 7) / 7, (v // 4096).float(), torch.where(v % 4096 == 5, 3.0, 0.0), -v.sqrt() / 10])
    scores = torch.tensor([[0.0, -1.0, -2.0, -0.5, 0.0, 0.0]], device="cuda")
    for k in (1, 3, 16, 64):
        beam_check(x, scores, None, k)


def test_beam_select_special_values():
    inf, nan = math.inf, math.nan
    x = 2 * randn(3, 8, 9000)
    x[0] = -inf                          # no candidates
    x[1, 5:] = -inf                      # five candidates
    x[2] = nan
    x[2, 7] = 1.0                        # one
    x[3, 100] = inf                      # the largest f32: takes all the mass
    x[4, [3, 8000]] = inf                # half each
    x[5] = torch.finfo(torch.float32).min
    x[6, ::2] = nan
    scores = torch.tensor([[0.0, -1.0, -2.0, -3.0, -4.0, -5.0, -6.0, -7.0]], device="cuda")
    for k in (4, 8, 20):
        beam_check(x, scores, None, k)
        for j in range(8):  # each row alone
            beam_check(x[j: j + 1], scores[:, j: j + 1], None, k)


def test_beam_select_dead_and_finished_beams():
    x = randn(4, 4 * 3, 500)
    scores = torch.tensor([[0.0, -math.inf, math.nan, math.inf], [-math.inf] * 4, [-1.0, -2.0, -0.5, -3.0]], device="cuda")
    done = i32([[0, 0, 0, 0], [1, 0, 0, 1], [1, 1, 1, 1]])
    for k in (1, 4, 6):
        beam_check(x, scores, done, k, pad=7)


def test_beam_select_in_place_strided_unaligned_and_captured():
    nb, beams, vocab = 2, 4, 6001
    wide = 2 * randn(9, nb * beams, vocab + 10)
    for off in (0, 4, 1):
        x = wide[:, off: off + vocab]
        scores, done = -torch.rand(nb, beams, device="cuda"), torch.zeros(nb, beams, dtype=torch.int32, device="cuda")
        done[1, 2] = 1
        want = beam_run(x, scores, done, beams)
        s0, d0 = scores.clone(), done.clone()
        par, tok = torch.empty_like(done), torch.empty_like(done)
        ws = torch.empty(beam.workspace_bytes(nb, beams, vocab, beams), dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            beam.select(x, scores, done, scores, par, tok, done, workspace=ws, stream=torch.cuda.current_stream().cuda_stream)
        for _ in range(2):
            scores.copy_(s0)
            done.copy_(d0)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip((scores, par, tok, done), want):
                assert torch.equal(a.cpu(), b)


# ------------------------------------------------------------------ refusals that need a device
def test_host_memory_is_refused():
    pages, table = R.make_cache([20], 1, 2, 64, torch.float16, 30)
    kv = paged.PagedKV(pages, table)
    q, i = randn(1, 1, 128, dtype=torch.float16), i32([0])
    for bad in ("q", "k", "out", "seqs"):
        a = dict(q=q, k=q.clone(), v=q.clone(), positions=i, seqs=i, out=q.clone())
        a[bad] = a[bad].cpu()
        with pytest.raises(L.FishaiError) as e:
            paged.rope_append(kv, 0, paged.Rope(64), **a)
        assert e.value.code == L.ERR_INVALID
    with pytest.raises(L.FishaiError) as e:
        paged.copy_pages(paged.PagedKV(pages.cpu(), table), i, i)
    assert e.value.code == L.ERR_INVALID


def test_work_is_on_the_given_stream():
    """a call on a side stream waits for what is before it there"""
    pages, table = R.make_cache([512], 1, 2, 128, torch.float16, 31)
    s = torch.cuda.Stream()
    q = torch.zeros(1, 512, dtype=torch.float16, device="cuda")
    new = randn(5, 1, 512, dtype=torch.float16)
    want = attn(pages, table, new, [0, 1], [512], 4)
    out = torch.empty_like(q)
    ws = torch.empty(paged.workspace_bytes(128), dtype=torch.uint8, device="cuda")
    start, kv = i32([0, 1]), i32([512])
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        q.copy_(new)
        paged.attention(paged.PagedKV(pages, table), 0, q, start, kv, out, 1, ws, stream=s.cuda_stream)
    s.synchronize()
    assert same_bits(out, want)


def test_two_streams_with_workspaces_of_their_own():
    """two attention calls and two selections that may run at the same time"""
    pages, table = R.make_cache([5000, 900], 1, 2, 128, torch.float16, 32)
    q = randn(6, 300, 8 * 128, dtype=torch.float16)
    kv = paged.PagedKV(pages, table)
    calls = [([0, 1, 3], [5000, 900], 2), ([0, 200, 300], [4000, 800], 200)]
    want = [attn(pages, table, q, a, b, 8, max_q=m) for a, b, m in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    ws = [torch.empty(paged.workspace_bytes(128), dtype=torch.uint8, device="cuda") for _ in calls]
    out = [torch.full_like(q, 7.0) for _ in calls]
    args = [(i32(a), i32(b), m) for a, b, m in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for (a, b, m), s, w, o in zip(args, streams, ws, out):
            paged.attention(kv, 0, q, a, b, o, m, w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(same_bits(o, w) for o, w in zip(out, want))
    x = 3 * randn(8, 2, 8, 50000)
    scores = -torch.rand(2, 8, device="cuda")
    sel = [beam_run(x[i], scores[i: i + 1], None, 8) for i in range(2)]
    outs = [[torch.empty(1, 8, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32, torch.int32)] for _ in range(2)]
    bw = [torch.empty(beam.workspace_bytes(1, 8, 50000, 8), dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            beam.select(x[i], scores[i: i + 1], None, *outs[i], workspace=bw[i], eos=2, stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, sel):
        assert all(torch.equal(a.cpu(), b) for a, b in zip(o, w))


@pytest.mark.parametrize("t,n_pages", [("f16", 140000), ("f32", 70000)])
def test_offsets_beyond_32_bits(t, n_pages):
    """a layer of more than 2^31 elements (f16: 2^32), sequences in its last pages"""
    dtype, kvh, hd, H = R.TYPES[t], 8, 128, 16
    small, stable = R.make_cache([700, 40, 333], 1, kvh, hd, dtype, 33)
    n = small.shape[1]
    pages = torch.empty(1, n_pages, 2, kvh, 16, hd, dtype=dtype, device="cuda")
    pages[0, n_pages - n:] = small[0]
    table = torch.where(stable < n, stable + (n_pages - n), stable).to(torch.int32).contiguous()
    kv = paged.PagedKV(pages, table)
    for start, lens in (([0, 1, 2, 3], [700, 40, 333]), ([0, 200, 201, 230], [700, 40, 333])):
        q = randn(7, start[-1], H * hd, dtype=dtype)
        a, b = attn(pages, table, q, start, lens, H), attn(small, stable, q, start, lens, H)
        assert same_bits(a, b)
    rows = randn(8, 3, (H + 2 * kvh) * hd, dtype=dtype)
    parts = rows[:, : H * hd], rows[:, H * hd: (H + kvh) * hd], rows[:, (H + kvh) * hd:]
    outs = []
    for p, tb in ((pages, table), (small, stable)):
        out = torch.empty(3, H * hd, dtype=dtype, device="cuda")
        paged.rope_append(paged.PagedKV(p, tb), 0, paged.Rope(hd), *parts, i32([5, 6, 7]), i32([0, 2, 1]), out)
        paged.copy_pages(paged.PagedKV(p, tb), tb[0, :3].contiguous(), tb[2, :3].contiguous(), slots=i32([16, 3, 9]))
        paged.compact(paged.PagedKV(p, tb), i32([0]), i32([3, 8, 200, 699]), i32([0, 4]))
        outs.append(out)
    assert same_bits(*outs) and same_bits(pages[0, n_pages - n:], small[0])
