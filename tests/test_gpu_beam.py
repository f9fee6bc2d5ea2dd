"""The paged operators as they are used together: shared pages of a model's
cache, and beam search (batched decode, selection, reordering of the pages)."""
import math
import os

import numpy as np
import pytest

import oracle as O
from fishai_engine import _lib as L
from fishai_engine import beam, paged, synth
from fishai_engine.model import ModelWeights
from fishai_engine.sampling import Sampler, SamplerConfig

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def path(tmp_path_factory):
    return synth.write_preset("tiny-q8_0", str(tmp_path_factory.mktemp("beam") / "tiny.gguf"))


@pytest.fixture(scope="module")
def dev(path):
    m = ModelWeights.load_from_gguf(path)
    # the same bits at every call: the default sums of split products vary in their last bits
    L.check(L.lib().fa_debug_set(m._h, L.DEBUG_FIXED_ORDER_SUMS, 1))
    yield m
    m.close()


def contents(kv, seq):
    return [kv.get(layer, seq) for layer in range(kv.n_layers())]


def equal(a, b):
    return all(np.array_equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))


def fill(dev, kv, lens, seed=0):
    rng = np.random.default_rng(seed)
    for s, n in enumerate(lens):
        if n:
            dev.prefill(rng.integers(3, dev.config.vocab_size, n).tolist(), 0, kv, seq=s, want_logits=False)


@pytest.mark.parametrize("dtype", [L.KV_F16, L.KV_F32])
def test_fork_shares_and_diverges(dev, dtype):
    kv = dev.new_kv_cache(96, dtype=dtype, n_seq=4)
    fill(dev, kv, [37, 20, 0, 48])
    a, d = contents(kv, 0), contents(kv, 3)
    before = kv.pages_used()
    kv.fork(0, 1)       # over a sequence of its own
    kv.fork(0, 2)       # into an empty one
    kv.fork(0, 0)
    assert kv.pages_used() == (before[0] - 2 + 1 + 1, 24)  # 2 pages of sequence 1 go, two partly filled ones come
    assert [kv.seq_len_with_dim(0, kv.kv_dim, s) for s in range(4)] == [37, 37, 37, 48]
    assert equal(contents(kv, 1), a) and equal(contents(kv, 2), a) and equal(contents(kv, 3), d)
    # each goes on by itself: the others keep their positions
    dev.prefill([5, 6, 7], 37, kv, seq=1, want_logits=False)
    dev.prefill([9] * 20, 37, kv, seq=2, want_logits=False)
    assert equal(contents(kv, 0), a)
    one, two = contents(kv, 1), contents(kv, 2)
    n = 37 * kv.kv_dim
    assert equal([(k[:n], v[:n]) for k, v in one], a) and equal([(k[:n], v[:n]) for k, v in two], a)
    assert not np.array_equal(one[0][0][n:], two[0][0][n: n + 3 * kv.kv_dim])
    # a copy decodes as the original does
    kv2 = dev.new_kv_cache(96, dtype=dtype, n_seq=2)
    fill(dev, kv2, [37])
    want = dev.forward([11], 37, kv2, seq=0)
    kv2.clear()
    got = dev.forward([11], 37, kv, seq=0)
    assert np.array_equal(got, want)
    kv.clear(0)
    assert equal(contents(kv, 1), one) and equal(contents(kv, 2), two)
    kv.clear()
    assert kv.pages_used() == (0, 24)


def test_fork_chains_and_clears_keep_every_page_in_order(dev):
    """random operations against plain copies on the host"""
    kv = dev.new_kv_cache(64, dtype=L.KV_F16, n_seq=5)
    rng = np.random.default_rng(1)
    fill(dev, kv, [30, 17, 33, 16, 5], 3)
    want = [contents(kv, s) for s in range(5)]
    for step in range(60):
        op = rng.integers(0, 6)
        s, d = int(rng.integers(0, 5)), int(rng.integers(0, 5))
        n = kv.seq_len_with_dim(0, kv.kv_dim, s)
        if op == 0:
            kv.fork(s, d)
            want[d] = want[s]
        elif op == 1:
            m = int(rng.integers(1, 6))
            parents = [int(x) for x in rng.integers(0, m, m)]
            kv.reorder(parents)
            want[:m] = [want[p] for p in parents]
        elif op == 2:
            m = int(rng.integers(0, n + 1))
            kv.truncate(s, m)
            want[s] = [(k[: m * kv.kv_dim], v[: m * kv.kv_dim]) for k, v in want[s]]
        elif op == 3 and n:
            keep = sorted(rng.choice(n, int(rng.integers(1, n + 1)), replace=False).tolist())
            kv.compact(s, keep)
            want[s] = [tuple(x.reshape(n, -1)[keep].reshape(-1) for x in kvp) for kvp in want[s]]
        elif op == 4:
            kv.clear(s)
            want[s] = [(k[:0], v[:0]) for k, v in want[s]]
        elif n < 55:
            m = int(rng.integers(1, min(9, 64 - n)))
            dev.prefill([int(x) for x in rng.integers(3, 1000, m)], n, kv, seq=s, want_logits=False)
            new = contents(kv, s)
            assert equal([(k[: n * kv.kv_dim], v[: n * kv.kv_dim]) for k, v in new], want[s]), step
            want[s] = new
        for q in range(5):
            assert equal(contents(kv, q), want[q]), (step, op, s, d, q)
    used, total = kv.pages_used()
    assert used <= total == 20


def test_share_refusals(dev):
    kv = dev.new_kv_cache(32, dtype=L.KV_F16, n_seq=2)
    fill(dev, kv, [20, 3])
    for bad in (lambda: kv.fork(2, 0), lambda: kv.fork(0, 2), lambda: kv.reorder([0, 0, 0]), lambda: kv.reorder([0, 2]),
                lambda: kv.truncate(0, 21), lambda: kv.truncate(2, 0), lambda: kv.compact(0, [3, 3]), lambda: kv.compact(0, [5, 2]),
                lambda: kv.compact(0, [20]), lambda: kv.compact(2, [])):
        with pytest.raises(L.FishaiError) as e:
            bad()
        assert e.value.code == L.ERR_INVALID
    kv.reorder([])
    kv.compact(1, [])
    assert kv.seq_len_with_dim(0, kv.kv_dim, 1) == 0


def test_operators_on_a_models_cache(dev):
    """rope_append and attention on the pages of a KVCache give what the model's own step does"""
    cfg = dev.config
    kv = dev.new_kv_cache(64, dtype=L.KV_F16, n_seq=2)
    fill(dev, kv, [21, 40], 5)
    pk = paged.PagedKV.of(kv)
    assert (pk.n_seq, pk.n_layers, pk.head_dim, pk.n_kv_heads) == (2, cfg.n_layers, cfg.head_dim, cfg.n_kv_heads)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    H, KVH, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = torch.randn(3, (H + 2 * KVH) * hd, device="cuda", generator=g)
    q, k, v = rows[:, : H * hd], rows[:, H * hd: (H + KVH) * hd], rows[:, (H + KVH) * hd:]
    out, err = torch.empty(3, H * hd, dtype=torch.float16, device="cuda"), i32([0])
    rope = paged.Rope(hd, base=cfg.rope_base)
    paged.rope_append(pk, 1, rope, q, k, v, i32([40, 21, 22]), i32([1, 0, 0]), out, err=err)
    att = torch.empty_like(out)
    ws = torch.empty(paged.workspace_bytes(hd), dtype=torch.uint8, device="cuda")
    paged.attention(pk, 1, out, i32([0, 1, 3]), i32([41, 23]), att, max_q=2, workspace=ws, seqs=i32([1, 0]), err=err)
    assert int(err) == 0
    f, _ = rope.freqs()
    pos = np.array([40, 21, 22])
    ang = pos[:, None] * np.array(f)
    def turned(x, n):
        x = x.double().cpu().numpy().reshape(3, n, hd // 2, 2)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        return np.stack((x[..., 0] * c - x[..., 1] * s, x[..., 0] * s + x[..., 1] * c), -1).reshape(3, n, hd)
    kt, vt = turned(k, KVH), v.double().cpu().numpy().reshape(3, KVH, hd)
    qh = out.double().cpu().numpy().reshape(3, H, hd)
    for t, (seq, n) in enumerate([(1, 41), (0, 22), (0, 23)]):
        ck, cv = (x.reshape(-1, KVH, hd).astype(np.float64) for x in kv.get(1, seq))
        mine = [0] if seq == 1 else [1, 2][: n - 21]
        ck, cv = (np.concatenate([c, np.float16(x[mine]).astype(np.float64)]) for c, x in ((ck, kt), (cv, vt)))
        assert len(ck) == n
        for h in range(H):
            s = ck[:, h // (H // KVH)] @ qh[t, h] / math.sqrt(hd)
            p = np.exp(s - s.max())
            want = p @ cv[:, h // (H // KVH)] / p.sum()
            # q, k, v and the result are f16 (half a step 2^-11 each), weights too; |v| < 5
            size = p @ np.abs(cv[:, h // (H // KVH)]) / p.sum()
            assert np.all(np.abs(att[t].double().cpu().numpy().reshape(H, hd)[h] - want) <= 2 ** -11 * (np.abs(want) + 6 * size) + 1e-6)


def search(dev, prompt, nb, max_new, eos, kv_dtype):
    """beam search made of the public pieces: batched decode with its logits, beam.select, KVCache.reorder"""
    V = dev.config.vocab_size
    kv = dev.new_kv_cache(len(prompt) + max_new, dtype=kv_dtype, n_seq=nb)
    if len(prompt) > 1:
        dev.prefill(prompt[:-1], 0, kv, seq=0, want_logits=False)
    for r in range(1, nb):
        kv.fork(0, r)
    smp = Sampler(SamplerConfig.greedy(), V, seeds=[0] * nb)
    scores = torch.full((1, nb), -math.inf, device="cuda")
    scores[0, 0] = 0.0
    done = torch.zeros(1, nb, dtype=torch.int32, device="cuda")
    par, tok = torch.empty_like(done), torch.empty_like(done)
    ws = torch.empty(beam.workspace_bytes(1, nb, V, nb), dtype=torch.uint8, device="cuda")
    hyp, cur = [[] for _ in range(nb)], [prompt[-1]] * nb
    for s in range(max_new):
        _, lg = dev.decode_batch(kv, cur, [len(prompt) - 1 + s] * nb, smp, 1, want_logits=True)
        beam.select(torch.from_numpy(lg[0]).cuda(), scores, done, scores, par, tok, done, workspace=ws,
                    eos=-1 if eos is None else eos)
        torch.cuda.synchronize()
        p, cur = par[0].tolist(), tok[0].tolist()
        hyp = [hyp[p[r]] + [cur[r]] for r in range(nb)]
        kv.reorder(p)
        if bool((done != 0).all()):
            break
    out = []
    for h, sc in zip(hyp, scores[0].tolist()):
        out.append((h[: h.index(eos) + 1] if eos in h else h, sc))
    return out


@pytest.mark.parametrize("kv_dtype", [L.KV_F16, L.KV_F32])
@pytest.mark.parametrize("nb,n_prompt,max_new", [(1, 5, 6), (4, 1, 5), (5, 30, 20), (16, 17, 8)])
def test_generate_beams_is_the_search_of_its_pieces(dev, kv_dtype, nb, n_prompt, max_new):
    prompt = np.random.default_rng(n_prompt).integers(3, dev.config.vocab_size, n_prompt).tolist()
    want = sorted(search(dev, prompt, nb, max_new, None, kv_dtype), key=lambda h: -h[1] / len(h[0]))
    got = dev.generate_beams(prompt, nb, max_new, kv_dtype=kv_dtype)
    assert [g[0] for g in got] == [w[0] for w in want]
    assert [g[1] for g in got] == [w[1] for w in want]
    assert len({tuple(g[0]) for g in got}) == nb  # all different


def test_generate_beams_ends_at_eos_and_ranks_by_length(dev):
    prompt = np.random.default_rng(9).integers(3, dev.config.vocab_size, 12).tolist()
    free = dev.generate_beams(prompt, 4, 8)
    eos = free[0][0][2]  # a token that the best hypothesis would pass through
    for penalty in (0.0, 1.0, 2.0):
        got = dev.generate_beams(prompt, 4, 8, eos=eos, length_penalty=penalty)
        want = sorted(search(dev, prompt, 4, 8, eos, L.KV_F16), key=lambda h: -h[1] / len(h[0]) ** penalty)
        assert [g[0] for g in got] == [w[0] for w in want]
        assert any(g[0][-1] == eos for g in got)
        assert all(eos not in g[0][:-1] for g in got)


def test_generate_beams_scores_are_the_oracles(dev, path):
    """each hypothesis' score is its sum of log-probabilities under the oracle: logits differ by at most 1e-2 of the largest
    (the 16-bit bar of the batched decode), twice that in a log-probability, per token"""
    ref = O.Model(path, threads=os.cpu_count() or 4)
    prompt = np.random.default_rng(4).integers(3, dev.config.vocab_size, 9).tolist()
    for ids, score in dev.generate_beams(prompt, 3, 5):
        kv = ref.kv(32)
        total, room = 0.0, 0.0
        for i, t in enumerate(prompt + ids[:-1]):
            lg = np.asarray(ref.forward([t], i, kv, algo=1), np.float64).reshape(-1)
            if i >= len(prompt) - 1:
                nxt = ids[i - len(prompt) + 1]
                m = lg.max()
                total += lg[nxt] - m - math.log(np.exp(lg - m).sum())
                room += 2e-2 * np.abs(lg).max()
        assert abs(total - score) <= room


def test_generate_beams_refusals(dev):
    for bad in (dict(n_beams=0), dict(n_beams=65), dict(max_new=0), dict(prompt_tokens=[]), dict(prompt_tokens=[10 ** 6]),
                dict(length_penalty=math.nan), dict(kv_dtype=2)):
        with pytest.raises(L.FishaiError) as e:
            dev.generate_beams(**{**dict(prompt_tokens=[5], n_beams=2, max_new=2), **bad})
        assert e.value.code == L.ERR_INVALID
    with pytest.raises(L.FishaiError):
        dev.new_kv_cache(16, dtype=L.KV_BF16)


@pytest.mark.parametrize("penalty", [31.0, -1e4, math.inf])
def test_generate_beams_refuses_penalties_without_a_rank(dev, penalty):
    """length^penalty would leave the range of f64: score / it could be 0 / 0"""
    with pytest.raises(L.FishaiError) as e:
        dev.generate_beams([5], 2, 2, length_penalty=penalty)
    assert e.value.code == L.ERR_INVALID
    assert len(dev.generate_beams([5], 2, 2, length_penalty=math.copysign(30.0, penalty))) == 2
