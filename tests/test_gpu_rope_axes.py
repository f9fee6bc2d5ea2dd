"""Rotary positions with several axes against a plain 64-bit form."""
import random

import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402
from fishai_engine import _lib as L  # noqa: E402
from fishai_engine import paged  # noqa: E402

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def turned(x, pos, rope, layout, heads, hd):
    """(rows, size of the terms of each element); pos [axes, tokens]"""
    freqs, scale = rope.freqs()
    rot = rope.rot_dim
    x = x.double().view(x.shape[0], heads, hd).clone()
    a = torch.stack([pos[ax].double() * f for ax, f in zip(rope.axis_of(), freqs)], 1)
    c, s = (a.cos() * scale)[:, None], (a.sin() * scale)[:, None]
    i0 = torch.arange(0, rot, 2) if layout == "interleaved" else torch.arange(rot // 2)
    i1 = i0 + 1 if layout == "interleaved" else i0 + rot // 2
    u, v = x[..., i0].clone(), x[..., i1].clone()
    x[..., i0], x[..., i1] = u * c - v * s, u * s + v * c
    size = x.abs()
    size[..., i0] = size[..., i1] = (u.abs() + v.abs()) * scale
    return x, size


def check(tokens, heads, kvh, hd, tin, tout, layout, seed=0, stream=None, broadcast=False, gap=0, **kw):
    rope = paged.Rope(hd, layout=layout, **kw)
    n_axes = rope.n_axes
    rng = random.Random(seed)
    lens = [tokens + 20 + i for i in range(3)]
    pages, table = R.make_cache(lens, 2, kvh, hd, tout, seed)
    before = pages.clone()
    seqs = [rng.randrange(3) for _ in range(tokens)]
    used = [list(range(n)) for n in lens]
    for u in used:
        rng.shuffle(u)
    slots = [used[s].pop() for s in seqs]
    if tokens > 2:
        seqs[1] = paged.NO_TOKEN
    pos = i32([[rng.choice([0, 1, 77, 10 ** 6 + 5, 2 ** 31 - 1, rng.randrange(5000)]) for _ in range(tokens + gap)] for _ in range(n_axes)])
    if broadcast:
        pos = pos[:1].expand(n_axes, -1)
    pos = pos[:, gap:]
    w = (heads + 2 * kvh) * hd
    rows = randn(seed + 1, tokens, w, dtype=tin)
    q, k, v = rows[:, : heads * hd], rows[:, heads * hd: (heads + kvh) * hd], rows[:, (heads + kvh) * hd:]
    out = torch.full((tokens, heads * hd), 7.0, dtype=tout, device="cuda")
    err = i32([0])
    paged.rope_append(paged.PagedKV(pages, table), 1, rope, q, k, v, pos if n_axes > 1 else pos[0].contiguous(), i32(seqs), out, slots=i32(slots),
                      err=err)
    assert int(err) == 0
    live = torch.tensor([s >= 0 for s in seqs], device="cuda")
    u = R.half_step(tout)
    # the angle's fraction of a turn is rounded once to f32 (2^-25 of at most 1/2 turn, times 2 pi < 2^-22.3), sincospi is
    # good to 2 ulp (2^-23), three f32 operations follow (3 2^-24) and the scale (2^-24); the 64-bit angle here is off by
    # at most 2^31 f 2^-53 radians
    e = 2 ** -22.3 + 2 ** -22 + 5 * 2 ** -24 + 2 ** -21

    def close(got, x, n):
        want, size = turned(x, pos, rope, layout, n, hd)
        tol = u * want.abs() + (1 + u) * e * size + (2.0 ** -25 if tout == torch.float16 else 0)
        assert not bool(((got.double().view_as(want) - want).abs() > tol)[live].any())

    close(out, q, heads)
    assert bool((out[~live] == 7.0).all())
    want = before.clone()
    got_k = torch.zeros(tokens, kvh, hd, dtype=tout, device="cuda")
    for t, (s, sl) in enumerate(zip(seqs, slots)):
        if s < 0:
            continue
        page = int(table[s, sl // 16])
        got_k[t] = pages[1, page, 0, :, sl % 16]
        want[1, page, 0, :, sl % 16] = got_k[t]
        want[1, page, 1, :, sl % 16] = v[t].float().view(kvh, hd).to(tout)
    close(got_k.flatten(1), k, kvh)
    bits = {4: torch.int32, 2: torch.int16}[pages.element_size()]
    assert torch.equal(pages.view(bits), want.view(bits))  # V exactly, and nothing else touched


AXES = [dict(axes=[16, 24, 24], axis_order="blocks"), dict(axes=[24, 20, 20], axis_order="turns"), dict(axes=[32, 32], axis_freqs="own"),
        dict(axes=[1, 1], rot_dim=4), dict(axes=[6, 2, 2, 2], rot_dim=24, axis_order="turns", axis_freqs="own"),
        dict(axes=[22, 21, 21], axis_order="turns", scaling="ntk", factor=4.0, axis_freqs="own"),
        dict(axes=[16, 16], rot_dim=64, scaling="yarn", factor=8.0, context=4096), dict(axes=[40, 24], scaling="llama3", factor=8.0, base=5e5),
        dict(axes=[64]), dict(axes=[10, 30, 24], scaling="linear", factor=2.5, axis_freqs="own")]


@pytest.mark.parametrize("kw", AXES, ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tin,tout", [("f32", "f16"), ("bf16", "bf16"), ("f16", "f32")])
def test_axes(kw, layout, tin, tout):
    check(9, 6, 2, 128, R.TYPES[tin], R.TYPES[tout], layout, seed=len(str(kw)), **kw)


@pytest.mark.parametrize("tokens,heads,kvh,hd", [(1, 1, 1, 8), (1, 32, 8, 128), (5, 3, 3, 256), (700, 7, 1, 72), (1300, 4, 2, 64), (64, 64, 8, 128)])
def test_sizes(tokens, heads, kvh, hd):
    check(tokens, heads, kvh, hd, torch.float16, torch.float16, "half", seed=tokens, axes=[hd // 2 - 2, 1, 1], axis_order="turns")


# heads that are turned in part, in 16-byte pieces: what is turned ends in either half of the head
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot", [(16, 16), (80, 48), (96, 80), (112, 96), (128, 32), (240, 32), (256, 256)])
@pytest.mark.parametrize("tin,tout", [("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
def test_partly_turned_heads(hd, rot, layout, tin, tout):
    check(701, 5, 1, hd, R.TYPES[tin], R.TYPES[tout], layout, rot_dim=rot, axes=[rot // 2 - 3, 2, 1], axis_order="turns")


def test_row_strides_of_the_positions():
    check(17, 4, 2, 64, torch.float16, torch.float16, "half", axes=[12, 10, 10], gap=5)
    check(17, 4, 2, 64, torch.float16, torch.float16, "half", axes=[12, 10, 10], broadcast=True)
    check(1, 4, 2, 64, torch.float16, torch.float16, "half", axes=[12, 10, 10])


def test_text_turns_as_with_one_axis():
    """all axes at the same position and shared frequencies: the bits of a rope of one axis"""
    hd, n = 128, 40
    pages, table = R.make_cache([60], 1, 2, hd, torch.bfloat16, 3)
    two = pages.clone()
    q, k = randn(1, n, 4 * hd, dtype=torch.bfloat16), randn(2, n, 2 * hd, dtype=torch.bfloat16)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    pos, slot, seq = torch.arange(900, 900 + n, device="cuda", dtype=torch.int32), i32(list(range(n))), i32([0] * n)
    paged.rope_append(paged.PagedKV(pages, table), 0, paged.Rope(hd, layout="half"), q, k, k, pos, seq, a, slots=slot)
    paged.rope_append(paged.PagedKV(two, table), 0, paged.Rope(hd, layout="half", axes=[24, 20, 20], axis_order="turns"), q, k, k,
                      pos.expand(3, -1).contiguous(), seq, b, slots=slot)
    assert torch.equal(a, b) and torch.equal(pages.view(torch.int16), two.view(torch.int16))


def test_captured_and_replayed():
    hd, n = 64, 5
    pages, table = R.make_cache([40], 1, 1, hd, torch.float16, 3)
    kv, rope = paged.PagedKV(pages, table), paged.Rope(hd, layout="half", axes=[16, 8, 8])
    q, k = randn(1, n, 2 * hd, dtype=torch.float16), randn(2, n, hd, dtype=torch.float16)
    out, pos, seq, slot = torch.zeros_like(q), i32([[1] * n] * 3), i32([0] * n), i32(list(range(n)))
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        paged.rope_append(kv, 0, rope, q, k, k, pos, seq, out, slots=slot, stream=st.cuda_stream)
    pos.copy_(i32([[3, 4, 4, 4, 9], [3, 4, 4, 5, 9], [3, 4, 5, 4, 9]]))
    graph.replay()
    torch.cuda.synchronize()
    want, size = turned(q, pos, rope, "half", 2, hd)
    assert bool(((out.double().view_as(want) - want).abs() <= 2 ** -11 * want.abs() + 2 ** -19 * size + 2 ** -25).all())


def test_bad_indices_are_flagged():
    hd = 64
    pages, table = R.make_cache([40, 40], 1, 2, hd, torch.float16, 1)
    table[1, 1] = pages.shape[1]
    before = pages.clone()
    q, k = randn(1, 4, 2 * hd, dtype=torch.float16), randn(2, 4, 2 * hd, dtype=torch.float16)
    rope = paged.Rope(hd, axes=[20, 12])
    for seqs, slots, flag in (([2, 0, 0, 0], [3, 4, 5, 6], L.FLAG_RANGE), ([0, 0, 0, 0], [48, 4, 5, 6], L.FLAG_RANGE), ([1, 0, 0, 0], [16, 4, 5, 6], L.FLAG_PAGE)):
        pages.copy_(before)
        err, out = i32([0]), torch.full_like(q, 7.0)
        paged.rope_append(paged.PagedKV(pages, table), 0, rope, q, k, k, i32([[1, 2, 3, 4], [5, 6, 7, 8]]), i32(seqs), out, slots=i32(slots), err=err)
        assert int(err) == flag
        assert bool((out[0] == 7.0).all()) and not bool((out[1:] == 7.0).all(1).any())
