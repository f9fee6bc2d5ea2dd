"""Sampling from given random numbers against a plain 64-bit form, a row at a time."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import serving_ref as S  # noqa: E402
from fishai_engine import paged, sampling  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NEAR_ONE = 1 - 2.0 ** -24


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def f32(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def logits_of(kind, n, vocab, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(n, vocab, device="cuda", generator=g)
    if kind == "text":  # a few tokens stand out
        x = 2 * x
        at = (torch.rand(n, min(vocab, 40), device="cuda", generator=g) * vocab).long().clamp_max(vocab - 1)
        x.scatter_add_(1, at, 9 * torch.rand(at.shape, device="cuda", generator=g) + 2)
    elif kind == "wide":
        x = 30 * x
    elif kind == "flat":
        x = 1e-3 * x
    elif kind == "equal":
        x = torch.full_like(x, -3.25)
    elif kind == "two":
        x = torch.where(x > 0.5, 1.0, -1.0)
    elif kind == "masked":
        off = torch.rand(n, vocab, device="cuda", generator=g)
        x = torch.where(off < 0.3, -math.inf, torch.where(off < 0.5, math.nan, torch.where(off < 0.7, torch.finfo(dtype).min, 3 * x)))
        x[:, vocab // 2] = 1.0
    return x.to(dtype)


def check(x, u, t=None, k=None, p=None, mp=None, rows=None, flags=0):
    """every row drawn as the definition says; t .. mp: lists or None"""
    n = len(u)
    ids, logs, err = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.full((n,), 7.0, device="cuda"), i32([0])
    sampling.sample_logits(x, f32(u), ids, temperature=None if t is None else f32(t), top_k=None if k is None else i32(k),
                           top_p=None if p is None else f32(p), min_p=None if mp is None else f32(mp), rows=None if rows is None else i32(rows),
                           logprobs=logs, err=err)
    assert int(err) == flags
    for i in range(n):
        f = lambda v, off: off if v is None else float(torch.tensor(v[i], dtype=torch.float32))  # noqa: E731  as the f32 that was given
        r = i if rows is None else rows[i]
        want, logp = S.sample(x[r], f(u, 0), f(t, 1.0), 0 if k is None else k[i], f(p, 1.0), f(mp, 0.0))
        got, lp = int(ids[i]), float(logs[i])
        assert got in want, (i, got, want, u[i], None if t is None else t[i], None if k is None else k[i], None if p is None else p[i])
        # one rounding to f32; the 64-bit sums of either side are off by some 10^-13
        assert lp == logp[got] or abs(lp - logp[got]) <= 2.0 ** -24 * abs(logp[got]) + 1e-12, (i, lp, logp[got])
    return ids


KINDS = ["text", "wide", "flat", "equal", "two", "masked"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 513, 5000, 32000, 128256])
def test_all_cuts(kind, t, vocab):
    rng = random.Random(vocab)
    n = 24
    x = logits_of(kind, n, vocab, TYPES[t], vocab)
    u = [rng.choice([0.0, NEAR_ONE, rng.random(), rng.random(), rng.random()]) for _ in range(n)]
    temp = [rng.choice([0.0, 1.0, 0.7, 1.3, 0.05, 30.0, 1e-6, 1e6]) for _ in range(n)]
    k = [rng.choice([0, 0, 1, 2, 50, 1024, 1025, 3000, vocab - 1, vocab, vocab + 1]) for _ in range(n)]
    p = [rng.choice([1.0, 2.0, 0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 0.99999, NEAR_ONE]) for _ in range(n)]
    mp = [rng.choice([0.0, 0.0, 0.05, 0.5, 1.0]) for _ in range(n)]
    check(x, u)
    check(x, u, temp)
    check(x, u, temp, k)
    check(x, u, temp, None, p)
    check(x, u, None, None, None, mp)
    check(x, u, temp, k, p, mp)


@pytest.mark.parametrize("vocab", [3, 4097, 65537, 262144, 393216])
def test_vocabularies(vocab):
    x = logits_of("text", 3, vocab, torch.float32, 5)
    check(x, [0.1, 0.5, 0.9], [1.0, 0.8, 0.0], [0, 50, 0], [0.9, 1.0, 1.0], [0.0, 0.01, 0.0])
    x = logits_of("flat", 3, vocab, torch.bfloat16, 6)
    check(x, [0.1, 0.5, 0.9], [1.0, 0.8, 1.0], [0, 2000, vocab // 2], [0.9, 1.0, 0.7])


@pytest.mark.parametrize("n", [1, 2, 63, 300, 1000])
def test_many_rows(n):
    rng = random.Random(n)
    x = logits_of("text", n, 3001, torch.float16, n)
    check(x, [rng.random() for _ in range(n)], [rng.uniform(0.5, 1.5) for _ in range(n)], [rng.choice([0, 20]) for _ in range(n)],
          [rng.uniform(0.5, 1.0) for _ in range(n)], [rng.choice([0.0, 0.1]) for _ in range(n)])


@pytest.mark.parametrize("n,vocab", [(300, 65537), (300, 70000), (300, 100001), (150, 131073), (150, 151000), (150, 200000)])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_many_long_rows_in_16_bits(n, vocab, t):
    """as few CTAs a row as shared memory allows would have more groups of elements than a warp has lanes"""
    rng = random.Random(vocab)
    x = logits_of("text", 4, vocab, TYPES[t], vocab)
    rows = [rng.randrange(4) for _ in range(n)]
    u, temp = [rng.choice([0.0, NEAR_ONE, rng.random(), rng.random()]) for _ in range(n)], [rng.choice([0.7, 1.0, 5.0, 40.0]) for _ in range(n)]
    check(x, u, temp, rows=rows)
    check(x, u, temp, [rng.choice([0, 30, 1500, vocab // 2]) for _ in range(n)], [rng.choice([1.0, 0.9, 0.5]) for _ in range(n)], rows=rows)


@pytest.mark.parametrize("n", [297, 480, 511, 512, 513])
@pytest.mark.parametrize("where", ["none", "all", "first", "last", "scattered", "one"])
def test_rows_with_long_cuts_anywhere(n, where):
    """more rows than run at once, of which some go by a histogram: each is drawn once, whatever the order"""
    rng = random.Random(n)
    lengthy = {"none": [], "all": range(n), "first": range(40), "last": range(n - 40, n), "scattered": range(0, n, 7), "one": [n // 2]}[where]
    vocab = 700
    k, p, t = [rng.choice([0, 1, 20, 128, vocab]) for _ in range(n)], [1.0] * n, [rng.choice([0.7, 1.0, 1.5]) for _ in range(n)]
    for i in lengthy:
        k[i], p[i] = rng.choice([(0, 0.9), (vocab + 5, 0.5), (129, 1.0), (400, 0.8)])
    for i in range(3, n, 11):
        t[i] = 0.0
    x = logits_of("text", n, vocab, torch.float32, n)
    rows = list(range(n))
    rng.shuffle(rows)
    check(x, [rng.random() for _ in range(n)], t, k, p, None, rows)


def test_answers_over_the_settings():
    """ids in the place of top_k, log-probabilities in that of the temperatures or of top_p"""
    n = 400
    rng = random.Random(7)
    x = logits_of("text", n, 900, torch.float32, 7)
    u = f32([rng.random() for _ in range(n)])
    k, p = i32([rng.choice([0, 0, 30, 200]) for _ in range(n)]), f32([rng.choice([1.0, 0.9, 0.6]) for _ in range(n)])
    t = f32([rng.choice([0.0, 0.8, 1.2]) for _ in range(n)])
    ids, logs = i32([-7] * n), torch.zeros(n, device="cuda")
    sampling.sample_logits(x, u, ids, temperature=t, top_k=k, top_p=p, logprobs=logs)
    for over in ("k and t", "p"):
        kk, pp, tt, own = k.clone(), p.clone(), t.clone(), torch.zeros_like(ids)
        out, lp = (kk, tt) if over == "k and t" else (own, pp)
        sampling.sample_logits(x, u, out, temperature=tt, top_k=kk, top_p=pp, logprobs=lp)
        assert torch.equal(out, ids) and torch.equal(lp, logs)


def test_the_place_of_a_cut_among_equal_values():
    """a few distinct values, thousands of each: the cut falls inside one, at an id"""
    x = torch.tensor([[float((i * 7919) % 5) for i in range(40000)]] * 8, device="cuda")
    check(x, [0.0, 0.3, 0.6, NEAR_ONE] * 2, None, [1500, 7000, 8000, 8001, 9000, 16000, 39999, 1], None)
    check(x, [0.0, 0.3, 0.6, NEAR_ONE] * 2, None, None, [0.1, 0.5, 0.61, 0.64, 0.9, 0.99, 0.001, 0.8])
    check(x, [0.5] * 8, None, [9000, 20000, 39000, 16000, 16001, 5000, 3000, 8000], [0.5, 0.9, 0.99, 0.6, 0.999, 0.3, 0.95, 0.01])


def test_zeros_of_both_signs_are_equal():
    x = torch.zeros(2, 3000, device="cuda")
    x[:, ::2] = -0.0
    x[:, 2500:] = -5.0
    check(x, [0.0, 0.9], [1.0, 0.0], [3, 0])
    check(x, [NEAR_ONE, 0.2], None, [2000, 3])


def test_infinities():
    x = logits_of("text", 4, 1000, torch.float32, 3)
    x[0, 77] = math.inf
    x[1, [5, 9]] = math.inf
    x[2] = -math.inf
    x[2, 123] = -1e30
    x[3] = torch.finfo(torch.float32).max
    check(x, [0.3, 0.7, 0.5, 0.5], None, [0, 0, 5, 7], [1.0, 0.6, 0.9, 1.0])


def test_rows_without_candidates():
    x = logits_of("text", 3, 1000, torch.float32, 3)
    x[1] = -math.inf
    x[2] = math.nan
    for kw in ({}, dict(t=[0.0] * 3), dict(k=[5] * 3, p=[0.9] * 3)):
        check(x, [0.3, 0.7, 0.5], flags=paged.FLAG_RANGE, **kw)


def test_rows_of_choice_and_none():
    x = logits_of("text", 5, 2000, torch.float16, 3)
    check(x, [0.3, 0.7, 0.5, 0.1], rows=[4, 4, 0, 2])
    ids, logs = i32([-7] * 3), f32([7.0] * 3)
    sampling.sample_logits(x, f32([0.5] * 3), ids, rows=i32([1, paged.NO_TOKEN, 3]), logprobs=logs)
    assert int(ids[1]) == -7 and float(logs[1]) == 7.0 and int(ids[0]) >= 0 and int(ids[2]) >= 0


@pytest.mark.parametrize("bad", [dict(u=1.0), dict(u=-1e-9), dict(u=math.nan), dict(t=-1.0), dict(t=1e-7), dict(t=1e7), dict(t=math.nan), dict(t=math.inf),
                                 dict(p=-0.1), dict(p=math.nan), dict(mp=1.5), dict(mp=-0.1), dict(mp=math.nan), dict(row=5), dict(row=-2)], ids=str)
def test_bad_settings_are_flagged_and_leave_the_row(bad):
    x = logits_of("text", 3, 700, torch.float32, 3)
    a = dict(u=0.5, t=1.0, p=0.9, mp=0.1, row=1)
    a.update(bad)
    ids, logs, err = i32([-7] * 3), f32([7.0] * 3), i32([0])
    sampling.sample_logits(x, f32([0.5, a["u"], 0.5]), ids, temperature=f32([1.0, a["t"], 1.0]), top_p=f32([0.9, a["p"], 0.9]),
                           min_p=f32([0.1, a["mp"], 0.1]), rows=i32([0, a["row"], 2]), logprobs=logs, err=err)
    assert int(err) == paged.FLAG_RANGE and int(ids[1]) == -7 and float(logs[1]) == 7.0 and int(ids[0]) >= 0 and int(ids[2]) >= 0


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_strides_and_alignment(t):
    wide = logits_of("text", 4, 3011, TYPES[t], 8)
    for off, vocab in ((0, 3000), (1, 3000), (8, 2999), (5, 1), (3, 3008)):
        check(wide[:, off: off + vocab], [0.2, 0.4, 0.6, 0.8], None, [0, 40, 0, 2000], [0.9, 1.0, 0.5, 1.0])
        check(wide[1:2, off: off + vocab], [0.4])


def test_frequencies_follow_the_weights():
    """an even grid of numbers draws each token as often as its share says, to one count at either border"""
    x = logits_of("text", 1, 50, torch.float32, 2)
    n = 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    ids = torch.empty(n, dtype=torch.int32, device="cuda")
    sampling.sample_logits(x, u, ids, rows=i32([0] * n), temperature=torch.full((n,), 0.9, device="cuda"))
    share = torch.softmax(x[0].double() / 0.9, 0) * n
    counts = torch.bincount(ids.long(), minlength=50)
    assert bool(((counts - share).abs() <= 1.0 + 1e-6).all())
    assert bool((ids[1:] >= ids[:-1]).all())  # by id


def test_captured_replayed_and_the_same_bits():
    x = logits_of("text", 16, 128256, torch.float32, 9)
    flat = logits_of("flat", 16, 128256, torch.float32, 10)
    u, ids, logs = torch.rand(16, device="cuda"), i32([0] * 16), f32([0.0] * 16)
    p = f32([0.9] * 8 + [1.0] * 8)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        sampling.sample_logits(x, u, ids, top_p=p, logprobs=logs, stream=st.cuda_stream)
    for data in (x.clone(), flat):
        x.copy_(data)
        graph.replay()
        torch.cuda.synchronize()
        first = ids.clone(), logs.clone()
        check(x, u.tolist(), None, None, p.tolist())
        for _ in range(5):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(ids, first[0]) and torch.equal(logs, first[1])


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_large_logits_and_small_temperatures(t):
    """the step of the type at the maximum is far above what the temperature tells apart"""
    big = {"f32": 1e7, "f16": 6e4, "bf16": 1e30}[t]
    x = logits_of("text", 4, 3000, torch.float32, 11) / 16
    for scale in (1.0, -1.0):
        check((big * scale * (1 + x / 4096)).to(TYPES[t]), [0.0, 0.4, 0.8, NEAR_ONE], [1e-6, 1e-3, 1.0, 1e6], [0, 50, 0, 2000], [0.9, 1.0, 0.5, 1.0])


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_infinity_beside_the_largest_number_of_a_type(t):
    x = logits_of("text", 3, 5000, TYPES[t], 12)
    x[:, 40] = torch.finfo(TYPES[t]).max
    x[0, [7, 4000]] = math.inf
    x[1, 4999] = math.inf
    x[1, 3] = math.nan
    for k in (None, [3] * 3, [600] * 3):
        check(x, [0.2, 0.6, 0.9], [1.0, 0.5, 1.0], k, [0.9, 1.0, 0.7])
        check(x, [0.2, 0.6, 0.9], [0.0] * 3, k)


def test_rows_beyond_32_bits_of_elements():
    x = torch.empty(34000, 128256, dtype=torch.float16, device="cuda")  # 4.36e9
    for r in (0, 33999):
        x[r] = logits_of("text", 1, 128256, torch.float16, r)[0]
    check(x, [0.3, 0.6, 0.9, 0.5], [1.0, 1.0, 0.8, 0.0], [0, 50, 0, 0], [1.0, 1.0, 0.9, 1.0], rows=[33999, 33999, 33999, 33999])
    del x
    torch.cuda.empty_cache()
