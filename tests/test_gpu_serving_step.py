"""The operators of a serving step as they are used together: a scheduler's loop over a small attention layer, plan, rotary
append with three axes, attention with a window and first positions, logits, sampling, and the drawn ids fed back."""
import random

import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from fishai_engine import paged, sampling  # noqa: E402

pytestmark = pytest.mark.gpu
HEADS, KVH, HD, VOCAB, WINDOW, SINKS = 8, 2, 64, 977, 40, 5
WIDTH = (HEADS + 2 * KVH) * HD


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Loop:
    """Fixed buffers for up to n requests and `rows` rows a step, as a captured step needs them."""

    def __init__(self, n, rows, max_pages, n_pages, dtype, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.n, self.rows = n, rows
        self.embed = rand(VOCAB, WIDTH).to(dtype)          # stands for all in front of the attention: a token's q, k, v
        self.head = (rand(HEADS * HD, VOCAB) / 4).to(dtype)
        self.pages = torch.zeros(1, n_pages, 2, KVH, 16, HD, dtype=dtype, device="cuda")
        self.table = torch.zeros(n, max_pages, dtype=torch.int32, device="cuda")
        self.kv = paged.PagedKV(self.pages, self.table)
        self.free = torch.randperm(n_pages, device="cuda", generator=g).int()
        self.n_free, self.lens, self.err = i32([n_pages]), i32([0] * n), i32([0])
        z = lambda k: torch.zeros(k, dtype=torch.int32, device="cuda")  # noqa: E731
        self.add, self.keep, self.q_start, self.kv_len, self.last = z(n), z(n), z(n + 1), z(n), z(n)
        self.pos, self.seq, self.slots, self.tokens, self.ids = z(rows), z(rows), z(rows), z(rows), z(n)
        self.axes = torch.zeros(3, rows, dtype=torch.int32, device="cuda")
        self.rope = paged.Rope(HD, layout="half", axes=[12, 10, 10], axis_order="turns")
        self.out = torch.zeros(rows, HEADS * HD, dtype=dtype, device="cuda")
        self.ws = torch.empty(paged.workspace_bytes(HD), dtype=torch.uint8, device="cuda")
        self.u = torch.zeros(n, device="cuda")
        self.temperature = torch.full((n,), 0.8, device="cuda")
        self.top_k, self.top_p = i32([40] * n), torch.full((n,), 0.9, device="cuda")
        self.min_p, self.logprobs = torch.full((n,), 0.02, device="cuda"), torch.zeros(n, device="cuda")
        self.logits = torch.zeros(rows, VOCAB, dtype=dtype, device="cuda")

    def plan(self, stream, keep):
        paged.plan_step(self.kv, self.add, self.lens, self.free, self.n_free, self.q_start, self.kv_len, self.pos, self.seq,
                        keep=self.keep if keep else None, slots=self.slots, last=self.last, err=self.err, stream=stream)

    def compute(self, max_q, stream):
        """everything behind the plan; text in all axes but for a shift, as behind pictures"""
        for a in range(3):
            torch.add(self.pos, 3 * a, out=self.axes[a])
        self.qkv = self.embed[self.tokens.clamp(0, VOCAB - 1)]
        q, k, v = self.qkv[:, : HEADS * HD], self.qkv[:, HEADS * HD: (HEADS + KVH) * HD], self.qkv[:, (HEADS + KVH) * HD:]
        self.q = torch.zeros_like(self.out)
        paged.rope_append(self.kv, 0, self.rope, q, k, v, self.axes, self.seq, self.q, slots=self.pos, err=self.err, stream=stream)
        paged.attention(self.kv, 0, self.q, self.q_start, self.kv_len, self.out, max_q=max_q, workspace=self.ws, window=WINDOW, sinks=SINKS,
                        err=self.err, stream=stream)
        torch.matmul(self.out, self.head, out=self.logits)
        sampling.sample_logits(self.logits, self.u, self.ids, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p, min_p=self.min_p,
                               rows=self.last, logprobs=self.logprobs, err=self.err, stream=stream)


def steps(n, count, seed):
    """what a scheduler asks for: prompts in parts, single tokens, drafts taken back, ends and new prompts"""
    rng = random.Random(seed)
    lens, left = [0] * n, [rng.randint(1, 150) for _ in range(n)]
    for _ in range(count):
        keep, add = list(lens), []
        for i in range(n):
            if lens[i] > 120 and rng.random() < 0.3:  # ends; the next one's prompt
                keep[i], left[i] = 0, rng.randint(1, 90)
            if left[i]:
                add.append(min(left[i], rng.choice([7, 33, 64])))
                left[i] -= add[-1]
            else:
                back = min(keep[i], rng.choice([0, 0, 0, 2]))
                keep[i] -= back
                add.append(back + 1)
            lens[i] = keep[i] + add[-1]
        yield keep, add, list(lens)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
def test_a_schedulers_loop(t):
    n, dtype = 7, R.TYPES[t]
    loop = Loop(n, 320, 40, 7 * 18, dtype)
    rng = random.Random(5)
    table, free, n_free, lens = loop.table.tolist(), loop.free.tolist(), int(loop.n_free), [0] * n
    for step, (keep, add, want_lens) in enumerate(steps(n, 25, 1)):
        loop.keep.copy_(i32(keep))
        loop.add.copy_(i32(add))
        loop.u.copy_(torch.rand(n))
        loop.tokens.copy_(torch.randint(0, VOCAB, (320,), dtype=torch.int32))
        loop.plan(0, True)
        # the ids that were drawn go on where a sequence grows by one
        want = S.plan(None, keep, add, 320, lens, table, free, n_free, 7 * 18)
        starts, table, free, lens, n_free = want[0], want[6], want[7], want[8], want[9]
        assert want[10] == 0 and lens == want_lens
        for got, w in ((loop.q_start, want[0]), (loop.kv_len, want[1]), (loop.last, want[2]), (loop.pos, want[3]), (loop.seq, want[4]),
                       (loop.slots, want[5]), (loop.table, table), (loop.free, free), (loop.lens, lens)):
            assert got.tolist() == w
        single = [i for i in range(n) if add[i] == 1]
        if step and single:
            loop.tokens[[starts[i] for i in single]] = loop.ids[single].clamp_min(0)
        loop.out.fill_(7.0)
        loop.compute(max(add), 0)
        assert int(loop.err) == 0
        total = starts[-1]
        assert bool((loop.out[total:] == 7.0).all())  # padded rows
        # the cache holds what was appended at the slots of the plan
        flat = loop.pages[0].permute(0, 3, 1, 2, 4).reshape(-1, 2, KVH * HD)
        assert torch.equal(flat[loop.slots[:total].long(), 1], loop.qkv[:total, (HEADS + KVH) * HD:])
        want_out, tol = S.attention(loop.pages, loop.table, loop.q, starts, lens, HEADS, 0.0, WINDOW, SINKS)
        assert bool(((loop.out.double().view_as(want_out) - want_out).abs() <= tol)[:total].all())
        for i in range(n):
            ids, logp = S.sample(loop.logits[want[2][i]], float(loop.u[i]), float(loop.temperature[i]), 40, float(loop.top_p[i]), float(loop.min_p[i]))
            assert int(loop.ids[i]) in ids
            assert abs(float(loop.logprobs[i]) - logp[int(loop.ids[i])]) <= 2.0 ** -24 * abs(logp[int(loop.ids[i])]) + 1e-12


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_a_captured_decode_step_gives_the_same_bits(t):
    """a graph of a whole step, replayed in place, beside the same calls without one"""
    n, dtype = 5, R.TYPES[t]
    loops = [Loop(n, 8, 30, 5 * 12, dtype, seed=3) for _ in range(2)]
    stream = torch.cuda.Stream()

    def step(loop, at):
        loop.plan(at, False)
        loop.tokens[: n].copy_(loop.ids)
        loop.compute(1, at)

    for loop in loops:
        loop.add.fill_(1)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step(loop, stream.cuda_stream)  # the libraries' first calls are outside the capture
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(loops[0], stream.cuda_stream)
    torch.manual_seed(0)
    for _ in range(150):
        u = torch.rand(n)
        for loop in loops:
            loop.u.copy_(u)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step(loops[1], stream.cuda_stream)
        torch.cuda.synchronize()
        a, b = loops
        for name in ("ids", "logprobs", "lens", "table", "free", "pages", "out", "err"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert int(a.err) == 0 and a.lens.tolist() == [151] * n
