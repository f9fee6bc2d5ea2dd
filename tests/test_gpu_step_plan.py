"""The plan of a step against a plain form that takes one request after another."""
import random

import pytest

torch = pytest.importorskip("torch")

import serving_ref as S  # noqa: E402
from fishai_engine import paged  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE = 16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def world(lens, max_pages, spare, seed=0):
    """table, free stack and its height for sequences of these lengths"""
    rng = random.Random(seed)
    per = [-(-n // PAGE) for n in lens]
    ids = list(range(sum(per) + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for p in per:
        table.append(ids[at: at + p] + [0] * (max_pages - p))
        at += p
    return table, ids[at:] + [0] * at, spare, len(ids)


def kv_of(table, n_pages):
    pages = torch.zeros(1, n_pages, 2, 1, PAGE, 8, dtype=torch.float16, device="cuda")
    return paged.PagedKV(pages, i32(table))


def run(kv, add, lens, free, n_free, rows, seqs=None, keep=None, in_place=True, slots=True, last=True, stream=0, n_pages=None):
    n = len(add)
    t = dict(lens=i32(lens), free=i32(free), n_free=i32([n_free]), q_start=i32([9] * (n + 1)), kv_len=i32([9] * n), pos=i32([9] * rows),
             seq=i32([9] * rows), slot=i32([9] * rows), last=i32([9] * n), err=i32([0]))
    out = {} if in_place else dict(lengths_out=t["lens"].clone(), n_free_out=i32([0]))
    paged.plan_step(kv, i32(add), t["lens"], t["free"], t["n_free"], t["q_start"], t["kv_len"], t["pos"], t["seq"],
                    seqs=None if seqs is None else i32(seqs), keep=None if keep is None else i32(keep), slots=t["slot"] if slots else None,
                    last=t["last"] if last else None, err=t["err"], stream=stream, **out)
    return [t["q_start"], t["kv_len"], t["last"], t["pos"], t["seq"], t["slot"], kv.page_table, t["free"], out.get("lengths_out", t["lens"]),
            out.get("n_free_out", t["n_free"]), t["err"]]


def check(add, lens, rows, max_pages, spare, seqs=None, keep=None, seed=0, cap=None, **kw):
    table, free, n_free, n_pages = world([min(x, max_pages * PAGE) for x in lens], max_pages, spare, seed)
    free = free if cap is None else free[:cap]
    kv = kv_of(table, n_pages)
    want = S.plan(seqs, keep, add, rows, lens, table, free, n_free, n_pages)
    got = run(kv, add, lens, free, n_free, rows, seqs, keep, **kw)
    names = ("q_start", "kv_len", "last", "pos", "seq", "slot", "table", "free", "lens", "n_free", "err")
    for name, g, w in zip(names, got, want):
        if (name == "slot" and not kw.get("slots", True)) or (name == "last" and not kw.get("last", True)):
            continue
        w = [w] if name in ("n_free", "err") else w
        assert g.tolist() == w, name
    return want


@pytest.mark.parametrize("in_place", [True, False])
def test_decode_steps(in_place):
    for n in (1, 2, 7, 33, 64, 300, 600):
        lens = [(i * 37) % 200 for i in range(n)]
        check([1] * n, lens, n, 16, n, in_place=in_place)
        check([1] * n, lens, n + 5, 16, n, in_place=in_place)  # padded rows


@pytest.mark.parametrize("seed", range(12))
def test_all_kinds_of_requests(seed):
    rng = random.Random(seed)
    n, m, most = rng.choice([3, 40, 200, 513, 1500]), rng.randint(0, 30), rng.choice([3, 20, 130])
    lens = [rng.randint(0, most * PAGE) for _ in range(n + m)]
    seqs = list(range(n + m))
    rng.shuffle(seqs)
    seqs = seqs[:n]
    keep = [rng.choice([lens[q], lens[q], 0, rng.randint(0, lens[q])]) for q in seqs]
    add = [min(most * PAGE - k, rng.choice([0, 1, 1, 5, rng.randint(0, 400)])) for k in keep]
    total, need = sum(add), sum(max(0, -(-(k + a) // PAGE) - -(-lens[q] // PAGE)) for q, k, a in zip(seqs, keep, add))
    check(add, lens, total + 3, most, need, seqs, keep, seed)                       # just enough pages
    check(add, lens, max(1, total * 2 // 3), most, need, seqs, keep, seed, slots=False)   # too few rows
    check(add, lens, total + 9, most, need // 2, seqs, keep, seed, last=False)      # too few pages
    check(add, lens, total, most, 0, seqs, keep, seed)


def test_nothing_and_little():
    check([], [5, 6], 4, 2, 3)
    check([], [5, 6], 0, 2, 3)
    check([0], [0], 1, 1, 0)
    check([16], [0], 16, 1, 1)
    check([17], [0], 17, 1, 2)   # beyond the table
    check([1], [16], 1, 1, 1)    # beyond the table
    check([1], [16], 1, 2, 1)
    check([1], [15], 1, 1, 0)
    check([3, 0], [40, 40], 3, 4, 0, keep=[1, 0])  # pages come back; none needed


def test_pages_that_come_back_are_given_out_in_the_same_call():
    # 4 pages come back; the first request grows from 1 page to 4 and the third from none to 2: 5 would be needed
    want = check([40, 0, 20], [10, 64, 0], 60, 4, 0, keep=[10, 0, 0])
    assert want[10] == paged.FLAG_FULL and want[9] == 1
    want = check([40, 0, 16], [10, 64, 0], 60, 4, 0, keep=[10, 0, 0])  # 4 needed
    assert want[10] == 0 and want[9] == 0


def test_a_request_that_does_not_fit_and_those_behind_it():
    want = check([4, 100, 4, 0], [10, 0, 20, 30], 50, 8, 50, keep=[10, 0, 20, 5])
    assert want[0] == [0, 4, 4, 4, 4] and want[10] == paged.FLAG_FULL and want[8] == [14, 0, 20, 5]
    check([4, 60, 4], [16, 0, 20], 100, 8, 2)
    check([2 ** 20] * 50, [0] * 50, 2 ** 20, 2 ** 17, 2 ** 16 + 7)


def test_sums_beyond_32_bits_do_not_wrap():
    n, most = 140, 2 ** 21  # 140 x 2^25 tokens and 140 x 2^21 pages
    lens = [0] * n
    table = torch.zeros(n, most, dtype=torch.int32, device="cuda")
    kv = paged.PagedKV(torch.zeros(1, 4, 2, 1, PAGE, 8, dtype=torch.float16, device="cuda"), table)
    got = run(kv, [1] + [2 ** 25] * (n - 1), lens, [0, 1, 2, 3], 4, 100)
    assert got[0].tolist() == [0] + [1] * n and got[10].tolist() == [paged.FLAG_FULL]
    assert got[1].tolist() == [1] + [0] * (n - 1) and got[9].tolist() == [3] and int(table[0, 0]) == 3


@pytest.mark.parametrize("kw", [dict(seqs=[0, 3, 1]), dict(seqs=[0, -1, 1]), dict(seqs=[1, 0, 1]), dict(seqs=[2, 2, 2]), dict(keep=[10, 21, 30]),
                                dict(keep=[10, -1, 30]), dict(lens=[10, 2000, 30]), dict(lens=[10, -5, 30]), dict(add=[1, 45, 2]),
                                dict(add=[1, -1, 1]), dict(add=[1, 2 ** 31 - 1, 1], lens=[10, 0, 30])], ids=str)
def test_bad_requests_are_left_out_and_flagged(kw):
    args = dict(add=[1, 2, 3], lens=[10, 20, 30], keep=None, seqs=None)
    args.update(kw)
    want = check(args["add"], args["lens"], 80, 4, 9, args["seqs"], args["keep"])
    assert want[10] & paged.FLAG_RANGE


def test_a_stack_that_does_not_fit_its_array():
    want = check([0, 1], [64, 10], 4, 4, 2, keep=[0, 10], cap=5)  # four pages come back, room for three
    assert want[10] == paged.FLAG_RANGE and want[8] == [64, 10]
    check([0, 1], [64, 10], 4, 4, 2, keep=[0, 10], cap=6)
    table, free, n_free, n_pages = world([10], 4, 3)
    got = run(kv_of(table, n_pages), [20], [10], free[:3], 7, 20)  # a height beyond the array
    assert got[10].tolist() == [paged.FLAG_RANGE] and got[0].tolist() == [0, 0] and got[9].tolist() == [7] and got[8].tolist() == [10]


def test_bad_pages_are_flagged():
    table, free, n_free, n_pages = world([40, 10], 4, 3)
    free[n_free - 1] = n_pages
    kv = kv_of(table, n_pages)
    got = run(kv, [1, 30], [40, 10], free, n_free, 40)
    assert got[10].tolist() == [paged.FLAG_PAGE]
    table[0][2] = n_pages + 5
    got = run(kv_of(table, n_pages), [0, 1], [40, 10], free, n_free, 40, keep=[0, 10])
    assert got[10].tolist() == [paged.FLAG_PAGE]


def test_captured_and_replayed():
    """a graph that plans a decode step over and over, in place"""
    n, max_pages = 20, 8
    lens = [(i * 7) % 40 for i in range(n)]
    table, free, n_free, n_pages = world(lens, max_pages, 100)
    kv = kv_of(table, n_pages)
    t = dict(lens=i32(lens), free=i32(free), n_free=i32([n_free]), q=i32([0] * (n + 1)), kv=i32([0] * n), pos=i32([0] * n), seq=i32([0] * n), err=i32([0]))
    add = i32([1] * n)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        paged.plan_step(kv, add, t["lens"], t["free"], t["n_free"], t["q"], t["kv"], t["pos"], t["seq"], err=t["err"], stream=st.cuda_stream)
    for step in range(50):
        want = S.plan(None, None, [1] * n, n, lens, table, free, n_free, n_pages)
        graph.replay()
        torch.cuda.synchronize()
        table, free, lens, n_free = want[6], want[7], want[8], want[9]
        assert t["pos"].tolist() == want[3] and t["lens"].tolist() == lens and kv.page_table.tolist() == table and int(t["n_free"]) == n_free
    assert int(t["err"]) == 0


def test_two_calls_at_once_on_pools_of_their_own():
    """streams side by side: nothing is shared between calls"""
    rng = random.Random(3)
    cases = []
    for i in range(8):
        n = [5, 300, 20, 700][i % 4]
        lens = [rng.randint(0, 100) for _ in range(n)]
        add = [rng.randint(0, 40) for _ in range(n)]
        table, free, n_free, n_pages = world(lens, 10, 3 * n, i)
        cases.append((kv_of(table, n_pages), add, lens, free, n_free, sum(add) + 3, S.plan(None, None, add, sum(add) + 3, lens, table, free, n_free, n_pages)))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for st, (kv, add, lens, free, n_free, rows, _) in zip(streams, cases):
        with torch.cuda.stream(st):
            got.append(run(kv, add, lens, free, n_free, rows, stream=st.cuda_stream))
    torch.cuda.synchronize()
    for g, c in zip(got, cases):
        for a, w in zip(g, c[6]):
            assert a.tolist() == (w if isinstance(w, list) else [w])


@pytest.mark.parametrize("n", [4096])
def test_the_most_requests(n):
    rng = random.Random(4)
    lens = [rng.randint(0, 60) for _ in range(n + 100)]
    seqs = list(range(n + 100))
    rng.shuffle(seqs)
    keep = [rng.choice([lens[q], lens[q], lens[q] // 2, 0]) for q in seqs[:n]]
    add = [min(64 - k, rng.choice([0, 1, 1, 17])) for k in keep]
    check(add, lens, sum(add), 4, 4 * n, seqs[:n], keep)
