"""Calls at the edges of what the operators on paged K/V and the beam selection
allow, against plain 64-bit forms."""
import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402
from fishai_engine import paged  # noqa: E402
from test_gpu_paged import attn, beam_check, beam_run, i32, randn, rope_case, rope_check, same_bits  # noqa: E402

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ beam selection
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [50, 4096, 4099, 40000])
@pytest.mark.parametrize("k", [1, 4, 16, 64])
def test_beam_select_zeros_of_both_signs_are_equal(t, vocab, k):
    """ties go to the lowest token whatever the zeros' signs, and no candidate is lost to them"""
    v = torch.arange(vocab, device="cuda")
    zero = torch.zeros(vocab, device="cuda")
    last = v % 4096 >= min(4096 - 1024, vocab // 2)
    low = -1.0 - v / vocab
    x = torch.stack([torch.where(last & (v % 4 == 3), zero, -zero),    # a thread's largest is +0.0, its first equal -0.0
                     torch.where(last, zero, -zero),
                     torch.where(v % 2 == 0, zero, -zero),
                     -zero,
                     torch.where(v == 5, -zero, torch.where(v == 10, zero, low)),
                     torch.where(v % 7 == 3, -zero, torch.where(v % 7 == 5, zero, low))]).to(R.TYPES[t])
    assert bool(torch.signbit(x).any()) and not bool(torch.signbit(x[:3]).all())
    n = x.shape[0]
    beam_check(x, torch.tensor([[0.0, -0.0, -0.0, 0.0, -0.0, 0.0]], device="cuda"), None, k)
    beam_check(x, torch.zeros(1, n, device="cuda"), None, k, eos=0)
    for j in range(n):  # each row alone
        beam_check(x[j: j + 1], torch.full((1, 1), -0.0, device="cuda"), None, k)


def test_beam_select_scores_of_zero_of_both_signs_are_equal():
    """finished beams stand at their own score; equal ones go to the lowest beam"""
    x = randn(3, 4, 900)
    done = i32([[1, 1, 1, 0]])
    for scores in ([-0.0, 0.0, -0.0, -3.0], [0.0, -0.0, 0.0, -3.0], [-0.0, -0.0, 0.0, 0.0]):
        for k in (1, 2, 3, 8):
            beam_check(x, torch.tensor([scores], device="cuda"), done, k, pad=3)


def lse_bound(vocab):
    """what fa_beam_select allows a row's log-sum to be off by"""
    return (128 + vocab / 512) * 2.0 ** -24


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,spread", [(100, 3.0), (32000, 3.0), (128256, 0.05), (128256, 3.0), (128256, 12.0)])
def test_beam_select_tells_beams_apart_beyond_the_bound_of_the_sum(t, vocab, spread):
    """the same logits in another order (one exact sum, other f32 ones), scores just more than twice the bound apart"""
    gap = 2.05 * lse_bound(vocab)
    for seed in range(6):
        row = (spread * randn(seed, vocab)).to(R.TYPES[t])
        row[0] = 14.0 * spread  # the best of every row by far, in another place of each
        g = torch.Generator("cuda").manual_seed(seed)
        x = torch.stack([row[torch.randperm(vocab, device="cuda", generator=g)] for _ in range(8)])
        place = torch.randperm(8, generator=torch.Generator().manual_seed(seed))
        scores = (-1.0 - gap * place.double()).float()[None].cuda()
        got = beam_run(x, scores, None, 8)
        want = R.beam_select(x.cpu(), scores.cpu(), None, 8, 2, 0)
        assert got[1].tolist() == [torch.argsort(place).tolist()] and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert bool(((got[0].double() - want[0]).abs() <= lse_bound(vocab) + 2.0 ** -24 * want[0].abs()).all())


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("t,heads,hd,chunks", [("f32", 4096, 8, 1000), ("f16", 4096, 64, 500)])
def test_attention_of_more_work_than_the_split_counts_is_refused(t, heads, hd, chunks):
    """chunks over a cache of 2^25 positions (one page again and again): 2^32 tiles a CTA and more are flagged, no row is written"""
    most = 1 << 21
    tiles, ctas = most * 16 // (64 if t == "f32" else 32), 3 * torch.cuda.get_device_properties(0).multi_processor_count
    assert chunks * heads * tiles >= ctas << 32
    pages = torch.zeros(1, 1, 2, heads, 16, hd, dtype=R.TYPES[t], device="cuda")
    table = torch.zeros(1, most, dtype=torch.int32, device="cuda")
    q = randn(1, chunks, heads * hd, dtype=R.TYPES[t])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attn(pages, table, q, list(range(chunks + 1)), [16 * most] * chunks, heads, seqs=[0] * chunks, err=err)
    assert int(err) == paged.FLAG_RANGE and bool((out == 7.0).all())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("n,kv,wide", [(1, 6000, 0), (1, 30000, 0), (3, 6000, 40000), (12, 1500, 0), (30, 5000, 0), (100, 9000, 0)])
@pytest.mark.parametrize("nats", [12.0, 17.5, 20.0])
def test_attention_weights_far_below_the_largest_count(t, heads, kvh, hd, n, kv, wide, nats):
    """one position far above thousands of equal ones, whose weights together are what the output is made of.  A weight of
    f16 has a relative half step of 2^-11 down to 2^-29 of the largest (2^-21 where items go to tcgen05) and is within
    2^-40 (2^-32) of it below that"""
    dtype = R.TYPES[t]
    per = max(kv, wide) // 16 + 1
    pages = torch.zeros(1, per, 2, kvh, 16, hd, dtype=dtype, device="cuda")
    table = torch.arange(per, dtype=torch.int32, device="cuda")[None].contiguous()
    pages[0, :, 1] = 1.0
    pages[0, 0, 0, :, 0, 0] = nats * hd ** 0.5 / 4
    pages[0, 0, 1, :, 0] = 0.0
    q = torch.zeros(n, heads * hd, dtype=dtype, device="cuda")
    q[:, ::hd] = 4.0
    out = attn(pages, table, q, [0, n], [kv], heads)
    want, tol = R.attention(pages, table, 0, q, i32([0, n]), i32([kv]), None, heads, 0.0, 0)
    if t == "f16":
        tol = tol + kv * (2.0 ** -40 if n * heads // kvh <= 16 else 2.0 ** -32)
    assert bool(((out.double().view_as(want) - want).abs() <= tol).all())


# ------------------------------------------------------------------ buffers
@pytest.mark.parametrize("n", [1, 3, 40, 150])
@pytest.mark.parametrize("order", ["q first", "out first"])
def test_q_and_out_as_column_ranges_of_one_buffer(n, order):
    """rows of both interleave in memory, but no element is shared"""
    pages, table = R.make_cache([200], 1, 2, 64, torch.float16, 12)
    buf = randn(5, n, 1024 + 8, dtype=torch.float16)
    a, b = buf[:, :512], buf[:, 520:]
    q, out = (a, b) if order == "q first" else (b, a)
    was = buf.clone()
    attn(pages, table, q, [0, n], [200], 8, out=out)
    want, tol = R.attention(pages, table, 0, q.contiguous(), i32([0, n]), i32([200]), None, 8, 0.0, 0)
    assert bool(((out.double().reshape(want.shape) - want).abs() <= tol).all())
    assert same_bits(q, was[:, :512] if order == "q first" else was[:, 520:]) and same_bits(buf[:, 512: 520], was[:, 512: 520])
    c = rope_case(n, 8, 2, 64, torch.float16, torch.float16, seed=7)
    q.copy_(c["q"])
    paged.rope_append(paged.PagedKV(c["pages"], c["table"]), 1, c["r"], q, c["k"], c["v"], i32(c["pos"]), i32(c["seqs"]), out,
                      slots=i32(c["slots"]))
    c["out"] = out.contiguous()
    rope_check(c, 8, 2, 64, "interleaved")
    assert same_bits(q, c["q"])


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("keep,moved", [([5, 1], {0: 5}), ([3, 1, 2, 9], {0: 3, 3: 9}), ([0, 7, 2, 3, 20], {1: 7, 4: 20}), ([1, 1], {0: 1})])
def test_compact_flags_a_position_that_does_not_ascend_where_it_would_stay(keep, moved):
    """keep[j] == j needs no copy, but is out of order behind a larger one"""
    pages, table = R.make_cache([40], 2, 2, 64, torch.float16, 24)
    want = pages.clone()
    at = lambda p: (slice(None), int(table[0, p // 16]), slice(None), slice(None), p % 16)  # noqa: E731
    for j, p in moved.items():
        want[at(j)] = pages[at(p)]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.compact(paged.PagedKV(pages, table), i32([0]), i32(keep), i32([0, len(keep)]), err=err)
    assert int(err) == paged.FLAG_RANGE
    assert same_bits(pages, want)


# ------------------------------------------------------------------ rotary append
@pytest.mark.parametrize("tokens", [601, 1199, 1203, 1601, 2050])
@pytest.mark.parametrize("tin,tout,kw", [("f16", "f16", {}), ("bf16", "bf16", dict(layout="half")), ("f32", "f32", {}), ("f32", "f16", dict(rot_dim=24))])
def test_rope_append_of_several_tokens_a_cta(tokens, tin, tout, kw):
    """two and four tokens a CTA, the last one with fewer, a row left out inside a group"""
    c = rope_case(tokens, 6, 2, 64, R.TYPES[tin], R.TYPES[tout], seed=tokens, spare_row=True, **kw)
    paged.rope_append(paged.PagedKV(c["pages"], c["table"]), 1, c["r"], c["q"], c["k"], c["v"], i32(c["pos"]), i32(c["seqs"]), c["out"],
                      slots=i32(c["slots"]))
    rope_check(c, 6, 2, 64, kw.get("layout", "interleaved"))


# ------------------------------------------------------------------ more than a grid's 65535
def test_copy_pages_of_more_pairs_than_a_grid_holds():
    n = 65535 + 200
    pages = randn(1, 2, 2 * n, 2, 1, 16, 8, dtype=torch.float16)
    src = torch.randperm(2 * n, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    src, dst = src[:n].contiguous(), src[n:].contiguous()
    slots = (torch.arange(n, device="cuda") % 17).int()
    want = pages.clone()
    copied = (torch.arange(16, device="cuda") < slots[:, None])[None, :, None, None, :, None]
    want[:, dst.long()] = torch.where(copied, pages[:, src.long()], pages[:, dst.long()])
    paged.copy_pages(paged.PagedKV(pages, i32([[0]])), src, dst, slots=slots)
    assert same_bits(pages, want)


@pytest.mark.parametrize("layers,n", [(1, 65535 + 70), (3, 21845 * 2 + 5)])
def test_compact_of_more_sequences_than_a_grid_holds(layers, n):
    """one page a sequence: positions 3, 5, 11 stay"""
    pages = randn(2, layers, n, 2, 1, 16, 8, dtype=torch.float16)
    table = torch.randperm(n, generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()[:, None].contiguous()
    want = pages.clone()
    want[:, :, :, :, :3] = pages[:, :, :, :, [3, 5, 11]]
    paged.compact(paged.PagedKV(pages, table), torch.arange(n, dtype=torch.int32, device="cuda"), i32([3, 5, 11] * n),
                  (3 * torch.arange(n + 1, device="cuda")).int())
    assert same_bits(pages, want)


def test_beam_select_of_more_rows_than_a_grid_holds():
    """1100 x 64 beams: the same as in parts of 100 requests"""
    nb, beams, vocab, k = 1100, 64, 40, 5
    x = randn(4, nb * beams, vocab)
    scores = -torch.rand(nb, beams, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    done = (torch.rand(nb, beams, device="cuda", generator=torch.Generator("cuda").manual_seed(6)) < 0.2).int()
    got = beam_run(x, scores, done, k)
    for a in range(0, nb, 100):
        part = beam_run(x[a * beams: (a + 100) * beams], scores[a: a + 100], done[a: a + 100], k)
        assert all(torch.equal(g[a: a + 100], p) for g, p in zip(got, part))
    for a in (0, 1023, 1024, 1099):  # row 65535 is a beam of request 1023
        beam_check(x[a * beams: (a + 1) * beams], scores[a: a + 1], done[a: a + 1], k)


# ------------------------------------------------------------------ graphs
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_append_copies_and_compaction_captured_and_replayed(t):
    """one graph of a step's rope_append, a fork's copies, a compaction and the attention over it; the lists in its
    buffers change between replays"""
    kvh, hd, heads = 2, 64, 8
    pages, table = R.make_cache([200, 90, 40], 2, kvh, hd, R.TYPES[t], 60, spare=6)
    at = int(pages.shape[1])
    was = pages.clone()
    used = {int(x) for s, n in enumerate((200, 90, 40)) for x in table[s, : -(-n // 16)]}
    free = [p for p in range(at) if p not in used]
    rope, kv = paged.Rope(hd), paged.PagedKV(pages, table)
    rows = randn(7, 3, (heads + 2 * kvh) * hd, dtype=R.TYPES[t])
    q, k, v = rows[:, : heads * hd], rows[:, heads * hd: (heads + kvh) * hd], rows[:, (heads + kvh) * hd:]
    ws = torch.empty(paged.workspace_bytes(hd), dtype=torch.uint8, device="cuda")
    lists = [dict(pos=[199, 89, 39], src=[int(table[0, 3]), int(table[1, 0])], dst=free[:2], slots=[16, 5], keep=[0, 3, 50, 51, 120], ks=[0, 5],
                  lens=[5, 90, 40]),
             dict(pos=[10, 20, 30], src=[int(table[2, 1]), int(table[0, 7])], dst=free[2:4], slots=[8, 16], keep=[1, 2, 4, 100, 199], ks=[0, 4],
                  lens=[4, 60, 31])]
    b = {n: i32(x) for n, x in lists[0].items()}
    seqs, one, start = i32([0, 1, 2]), i32([0]), i32([0, 1, 2, 3])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    turned, out = torch.empty_like(rows[:, : heads * hd]), torch.empty_like(rows[:, : heads * hd])

    def step(stream):
        paged.rope_append(kv, 1, rope, q, k, v, b["pos"], seqs, turned, err=err, stream=stream)
        paged.copy_pages(kv, b["src"], b["dst"], slots=b["slots"], err=err, stream=stream)
        paged.compact(kv, one, b["keep"], b["ks"], err=err, stream=stream)
        paged.attention(kv, 1, turned, start, b["lens"], out, 1, ws, err=err, stream=stream)

    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        step(torch.cuda.current_stream().cuda_stream)
    for values in lists + lists[:1]:
        for n, x in values.items():
            b[n].copy_(i32(x))
        results = []
        for run in (lambda: step(0), g.replay):
            pages.copy_(was)
            turned.fill_(9.0), out.fill_(9.0)
            torch.cuda.synchronize()
            run()
            torch.cuda.synchronize()
            results.append((pages.clone(), turned.clone(), out.clone()))
        assert int(err) == 0 and all(same_bits(x, y) for x, y in zip(*results))
        assert not same_bits(results[0][0], was) and not bool(results[0][2].isnan().any())
