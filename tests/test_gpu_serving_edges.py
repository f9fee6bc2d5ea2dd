"""Calls of the operators around a serving step that their documentation allows and their own files do not make."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
import test_gpu_sinks as A  # noqa: E402
import test_gpu_step_plan as P  # noqa: E402
from fishai_engine import _lib as L  # noqa: E402
from fishai_engine import paged  # noqa: E402

pytestmark = pytest.mark.gpu
i32 = P.i32


# ------------------------------------------------------------------ the plan with lengths of its own to write
@pytest.mark.parametrize("kw", [dict(seqs=[0, 3, 1]), dict(seqs=[0, 7, 1]), dict(seqs=[0, -1, 1]), dict(seqs=[1, 0, 1]), dict(seqs=[2, 2, 2]),
                                dict(keep=[10, 21, 30]), dict(keep=[10, -1, 30]), dict(lens=[10, 2000, 30, 8]), dict(lens=[10, -5, 30, 8]),
                                dict(add=[1, 45, 2]), dict(add=[1, -1, 1]), dict(cap=1), dict(), dict(rows=3), dict(spare=0)], ids=str)
@pytest.mark.parametrize("n_more", [0, 300])
def test_lengths_of_requests_that_are_left_out(kw, n_more):
    """lengths_out holds junk before the call: what is named has its length after it, the old one where the request was refused"""
    a = dict(add=[1, 2, 3], lens=[10, 20, 30, 8], keep=None, seqs=[0, 1, 2], rows=80, cap=None, spare=9)
    a.update(kw)
    add, lens = a["add"] + [1] * n_more, a["lens"] + [5] * n_more
    seqs, keep = a["seqs"] + list(range(4, 4 + n_more)), a["keep"] and a["keep"] + [5] * n_more
    if a["cap"]:  # two pages come back, and the stack has room for one
        keep = [0] * 3 + [5] * n_more
    table, free, n_free, n_pages = P.world([max(0, min(x, 64)) for x in lens], 4, a["spare"])
    free = free[: n_free + a["cap"]] if a["cap"] else free
    want = S.plan(seqs, keep, add, a["rows"] + n_more, lens, table, free, n_free, n_pages)
    kv, n, rows = P.kv_of(table, n_pages), len(add), a["rows"] + n_more
    out, err = i32([-77] * len(lens)), i32([0])
    arrays = [i32([9] * m) for m in (n + 1, n, rows, rows)]
    before = i32(lens)
    paged.plan_step(kv, i32(add), before, i32(free), i32([n_free]), *arrays, seqs=i32(seqs), keep=None if keep is None else i32(keep),
                    lengths_out=out, n_free_out=i32([0]), err=err)
    named = {q for q in seqs if 0 <= q < len(lens)}
    assert out.tolist() == [m if q in named else -77 for q, m in enumerate(want[8])]
    assert before.tolist() == lens and arrays[1].tolist() == want[1] and int(err) == want[10]


def test_a_shared_prefix_that_no_request_is_cut_into():
    """two sequences with the same two pages in front: they grow, are cut down to the prefix and grow again, and the pages stay"""
    lens = [50, 39, 0]
    table, free, n_free, n_pages = P.world(lens, 6, 9)
    table[1][:2] = table[0][:2]  # the second one's own first two pages are nobody's now
    prefix = set(table[0][:2])
    kv, t, f, n = P.kv_of(table, n_pages), i32(lens), i32(free), i32([n_free])
    for keep, add in (([50, 39, 0], [1, 1, 20]), ([40, 33, 20], [3, 30, 1]), ([32, 32, 0], [0, 0, 60]), ([32, 32, 60], [17, 40, 1])):
        err, out = i32([0]), [i32([9] * m) for m in (4, 3, 100, 100)]
        want = S.plan(None, keep, add, 100, lens, table, free, n_free, n_pages)
        table, free, lens, n_free = want[6], want[7], want[8], want[9]
        paged.plan_step(kv, i32(add), t, f, n, *out, keep=i32(keep), err=err)
        assert int(err) == want[10] == 0
        assert kv.page_table.tolist() == table and f.tolist() == free and t.tolist() == lens and int(n) == n_free
        assert not prefix & set(free[:n_free]) and table[0][:2] == table[1][:2] and not prefix & set(table[2][: -(-lens[2] // 16)])


# ------------------------------------------------------------------ which slots of a page are read
@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 65, 300])
def test_only_slots_that_are_seen_are_read(t, hd, n):
    """every other slot holds NaN, every other page is a bad one: edges of the cache, of the window and of the first positions
    at every place of a page"""
    for q in (1, 5, 40):
        for window, sinks in ((0, 0), (1, 0), (7, 0), (16, 0), (17, 0), (1, 1), (3, 5), (16, 16), (15, 17), (2, 40)):
            if q <= n:
                A.check([q, q], [n, max(q, n - 3)], 4, 2, hd, R.TYPES[t], window, sinks, seed=n)


# ------------------------------------------------------------------ the entry with first positions, and none of them
@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("window", [0, 1, 30, 10 ** 6])
def test_no_first_positions_through_their_entry(t, window):
    """Python takes the other entry for these; from C both give the same bits"""
    qs, kvs = [1, 40, 200, 0], [300, 90, 250, 8]
    pages, table = R.make_cache(kvs, 1, 2, 64, R.TYPES[t], 3)
    start, n = [0, 1, 41, 241, 241], 241
    q = A.randn(4, n, 8 * 64, dtype=R.TYPES[t])
    want = A.call(pages, table, q, start, kvs, window, 0)
    kv, out, err = paged.PagedKV(pages, table), torch.full_like(q, 7.0), i32([0])
    ws = torch.empty(paged.workspace_bytes(64), dtype=torch.uint8, device="cuda")
    starts, lens = i32(start), i32(kvs)
    L.check(L.lib().fa_attn_chunks_sinks(kv._ref, 0, q.data_ptr(), 8 * 64, 8, 4, starts.data_ptr(), lens.data_ptr(), None, n, 200, 0.0, window, 0,
                                         out.data_ptr(), 8 * 64, ws.data_ptr(), ws.numel(), err.data_ptr(), None))
    assert torch.equal(out, want) and int(err) == 0
    exact, tol = S.attention(pages, table, q, start, kvs, 8, 0.0, window, 0)
    assert bool(((out.double().view_as(exact) - exact).abs() <= tol).all())


def test_numbers_of_numpy_and_err_by_place():
    """the same bits and flags as with Python's own numbers, named"""
    lens = np.array([1, 33, 7])
    start = [0] + np.cumsum(lens).tolist()
    pages, table = R.make_cache([50, 40, 90], 2, 2, 64, torch.float16, 9)
    table[2, 1] = pages.shape[1]  # a bad page
    q = A.randn(1, 41, 4 * 64, dtype=torch.float16)
    kv, ws = paged.PagedKV(pages, table), torch.empty(paged.workspace_bytes(64), dtype=torch.uint8, device="cuda")
    args = (i32(start), i32([50, 40, 90]))
    a, b, ea, eb = torch.zeros_like(q), torch.zeros_like(q), i32([0]), i32([0])
    paged.attention(kv, 1, q, *args, a, 33, ws, window=60, err=ea, sinks=4)
    paged.attention(kv, np.int32(1), q, *args, b, np.max(lens), ws, None, 0.0, np.uint32(60), eb, 0, np.int64(4))
    assert torch.equal(a, b) and int(ea) == int(eb) == paged.FLAG_PAGE
