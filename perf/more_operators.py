"""The operators around the paged serving path's steps, as cases to be measured: the plan of a step (pages taken and given
back, positions and slots of its rows), rotary positions with several axes, attention with a sliding window beside a few first
positions that stay visible, and sampling from given random numbers.

`run` computes them from elementary torch operations; with `own` set it calls fishai_engine's kernels instead.

Pages are [layer][page][k | v][kv head][16 positions][head_dim]; page_table[sequence][i] holds positions 16 i .. 16 i + 15.
"""
import math
import random
import sys

import numpy as np
import torch

own = False

PAGE = 16
NONE = -1  # no sequence, no slot, no row
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    big = {"heads": 32, "kv_heads": 8, "head_dim": 128}  # the 8B shape
    return [
        # a decode step of eight sequences, some pages full: latency
        {"name": "plan decode of 8", "op": "plan", "requests": 8, "seqs": 16, "most": 512, "prompts": 0.0, "longest": 1, "tight": False},
        # a scheduling step of a busy server: prompts and parts of them beside single tokens, drafts taken back, ends
        {"name": "plan mixed 512", "op": "plan", "requests": 512, "seqs": 640, "most": 8192, "prompts": 0.1, "longest": 2048,
         "tight": False},
        # one token behind an image: three axes, the f32 sums of a decode step into an f16 cache; latency
        {"name": "axes one token", "op": "rope", **big, "in": "f32", "type": "f16", "tokens": 1, "seqs": 1, "axes": 3, "rot": 128,
         "layout": "half", "order": "blocks", "freqs": "shared", "scaling": "none", "start": 1900},
        # prompts with pictures of three requests in one call
        {"name": "axes prompts of 8192", "op": "rope", **big, "in": "bf16", "type": "bf16", "tokens": 8192, "seqs": 3, "axes": 3, "rot": 128,
         "layout": "half", "order": "turns", "freqs": "shared", "scaling": "none", "start": 7},
        # a stream that runs on and on: one token over the end of a long cache; latency and split work
        {"name": "sinks one token", "op": "attn", **big, "type": "f16", "chunks": 1, "q_min": 1, "q_max": 1, "kv_min": 65536,
         "kv_max": 65536, "window": 4096, "sinks": 4},
        # 64 such streams, caches of every length
        {"name": "sinks batch of 64", "op": "attn", **big, "type": "bf16", "chunks": 64, "q_min": 1, "q_max": 1, "kv_min": 100,
         "kv_max": 16384, "window": 1024, "sinks": 4},
        # one to three tokens of five short sequences over the f32 cache of the tiny shape
        {"name": "sinks tiny f32", "op": "attn", "heads": 8, "kv_heads": 2, "head_dim": 64, "type": "f32", "chunks": 5,
         "q_min": 1, "q_max": 3, "kv_min": 1, "kv_max": 512, "window": 48, "sinks": 3},
        # one scheduling step: prompts, parts of prompts and single tokens together
        {"name": "sinks mixed chunks", "op": "attn", **big, "type": "bf16", "chunks": 8, "q_min": 1, "q_max": 1024, "kv_min": 900,
         "kv_max": 8192, "window": 2000, "sinks": 33},
        # a chunk of 2048 tokens deep in a long prompt
        {"name": "sinks chunk of 2048", "op": "attn", **big, "type": "f16", "chunks": 1, "q_min": 2048, "q_max": 2048,
         "kv_min": 16384, "kv_max": 16384, "window": 4096, "sinks": 64},
        # one request's next token; latency
        {"name": "sample one row", "op": "sample", "rows": 1, "vocab": 128256, "type": "f32", "kind": "all"},
        # a decode step of 64 requests with settings of their own
        {"name": "sample batch of 64", "op": "sample", "rows": 64, "vocab": 128256, "type": "f32", "kind": "all"},
        # many requests without cuts, logits in 16 bits (many of them equal)
        {"name": "sample 200 plain bf16", "op": "sample", "rows": 200, "vocab": 32000, "type": "bf16", "kind": "temperature"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["plan", "plan", "rope", "rope", "attn", "attn", "attn", "attn", "sample", "sample", "sample"])
        kv = rng.choice([1, 2, 4, 8, 8])
        hd = rng.choice([64, 128, 128])
        rep = rng.choice([1, 2, 4, 4, 7, 8])
        kind = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
        if op == "plan":
            n = _log(rng, 1, 2000)
            c = {"op": op, "requests": n, "seqs": n + rng.randint(0, 64), "most": _log(rng, 20, 8192), "prompts": rng.choice([0.0, 0.1, 0.5]),
                 "longest": _log(rng, 1, 2048), "tight": rng.random() < 0.3}
            if n * c["longest"] * c["prompts"] > 200000:
                continue
        elif op == "rope":
            n, axes = _log(rng, 1, 8192), rng.choice([2, 3, 3, 4])
            c = {"op": op, "heads": kv * rep, "kv_heads": kv, "head_dim": hd, "in": rng.choice(["f32", "f16", "bf16"]), "type": kind,
                 "tokens": n, "seqs": rng.randint(1, min(n, 64)), "axes": axes, "rot": rng.choice([hd, hd, hd // 2, 24]),
                 "layout": rng.choice(["interleaved", "half"]), "order": rng.choice(["blocks", "turns"]),
                 "freqs": rng.choice(["shared", "shared", "own"]), "scaling": rng.choice(["none", "none", "linear", "ntk"]),
                 "start": _log(rng, 1, 200000)}
        elif op == "attn":
            q = rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 1, 2048)])
            n = rng.choice([1, _log(rng, 1, 64)])
            kv_max = max(q, _log(rng, 1, 32768))
            c = {"op": op, "heads": kv * rep, "kv_heads": kv, "head_dim": hd, "type": kind, "chunks": n, "q_min": rng.randint(1, q), "q_max": q,
                 "kv_min": rng.randint(1, kv_max), "kv_max": kv_max, "window": _log(rng, 1, 8192), "sinks": rng.choice([1, 4, 16, _log(rng, 1, 1000)])}
            if kind == "f32":  # the f32 cache is the reference's own values, not the fast path
                c.update(q_min=min(c["q_min"], 32), q_max=min(q, 32))
            if n * kv_max * kv * hd > 2 ** 29 or n * c["heads"] * c["q_max"] * _span(c) > 2 ** 29 or n * _span(c) * kv * hd > 2 ** 28:
                continue
        else:
            c = {"op": op, "rows": _log(rng, 1, 256), "vocab": rng.choice([32000, 128256, _log(rng, 50, 200000)]),
                 "type": rng.choice(["f32", "f32", "f16", "bf16"]), "kind": rng.choice(["all", "all", "temperature", "top_k", "top_p", "min_p"])}
        if _cost(c) <= top:
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / (1.6e15 if c.get("type") != "f32" else 3e13))


# ------------------------------------------------------------------ what a case is made of, the same for every seed
def _requests(c):
    """(length, kept positions, new tokens) of each request, and the rows of the step."""
    r = random.Random(c["requests"] * 7919 + c["most"] * 31 + c["longest"])
    got = []
    for i in range(c["requests"]):
        have = r.randint(1, c["most"] - 1)
        x = r.random()
        if x < c["prompts"]:  # a prompt, or a part of one behind what is there
            have = 0 if r.random() < 0.5 else have
            got.append((have, have, min(r.randint(1, c["longest"]), c["most"] - have)))
        elif x < c["prompts"] + 0.05 and i:  # ended: its pages are free
            got.append((have, 0, 0))
        elif x < c["prompts"] + 0.2 and i:  # drafts that were refused, and the next ones
            back = min(have, r.randint(1, 5))
            got.append((have, have - back, min(5, c["most"] - have + back)))
        else:
            got.append((have, have, 1))
    total = sum(g[2] for g in got)
    return got, max(1, total * 3 // 4) if c["tight"] else -(-total // 8) * 8  # rows are padded; a tight step has too few


def _sizes(c):
    """The chunks' lengths and their caches' lengths: one of the largest, the others spread down to the smallest."""
    r = random.Random(c["chunks"] * 7919 + c["kv_max"] * 31 + c["q_max"])
    n = c["chunks"]
    kv = [c["kv_max"]] + [r.randint(c["kv_min"], c["kv_max"]) for _ in range(n - 1)]
    q = [c["q_max"]] + [r.randint(c["q_min"], c["q_max"]) if r.random() < 0.5 else c["q_min"] for _ in range(n - 1)]
    return [min(a, b) for a, b in zip(q, kv)], kv


def _span(c):
    """Most positions that the tokens of a chunk see."""
    return min(c["kv_max"], c["window"] + c["q_max"] - 1 + c["sinks"])


def _seen(q, kv, window, sinks):
    """How many (query, position) pairs a chunk of q tokens sees, and how many positions of its cache any of them sees."""
    p = np.arange(kv - q, kv)
    low = np.maximum(0, p - window + 1)
    return int((p - low + 1 + np.minimum(sinks, low)).sum()), int(kv - low[0] + min(sinks, low[0]))


def _shares(c):
    """Pairs of the turned elements for each axis, the first the rest."""
    half, n = c["rot"] // 2, c["axes"]
    each = half * 3 // (4 * n) if n > 2 else half // n
    each = max(1, each)
    return [half - (n - 1) * each] + [each] * (n - 1)


def work(c):
    if c["op"] == "plan":
        got, rows = _requests(c)
        moved = sum(abs(-(-(k + a) // PAGE) - -(-n // PAGE)) for n, k, a in got)
        return {"bytes": 4 * (8 * c["requests"] + 3 * rows + 2 * moved), "flops": 0}
    t = _SIZE[c["type"]]
    if c["op"] == "rope":
        n = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
        return {"bytes": n * (_SIZE[c["in"]] + t), "flops": 6 * n}
    if c["op"] == "attn":
        q, kv = _sizes(c)
        both = [_seen(a, b, c["window"], c["sinks"]) for a, b in zip(q, kv)]
        rows = 2 * sum(q) * c["heads"] * c["head_dim"]
        return {"bytes": t * (rows + 2 * c["kv_heads"] * c["head_dim"] * sum(p[1] for p in both)),
                "flops": 4 * c["heads"] * c["head_dim"] * sum(p[0] for p in both)}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * t + c["rows"] * 28, "flops": 4 * n}


# ------------------------------------------------------------------ inputs
def _whole(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(per, order):
    """Shuffled pages for sequences of so many each; behind a sequence's end any page."""
    ids = list(range(sum(per) + 1))
    order.shuffle(ids)
    at, table = 0, []
    for p in per:
        table.append(ids[at: at + p] + [ids[-1]] * (max(max(per), 1) - p))
        at += p
    return _whole(table), len(ids)


def _positions(n, axes, start):
    """Axes of n positions: runs of text, in which all axes count together, and pictures of some frames, rows and columns."""
    r = random.Random(n * 31 + axes)
    got, p = [], start
    while len(got) < n:
        for _ in range(r.randint(4, 40)):
            got.append([p] * axes)
            p += 1
        f, h, w = r.choice([(1, 14, 20), (1, 24, 24), (4, 10, 16)])
        for i in range(f * h * w):
            at = (i // (h * w), i // w % h, i % w, i % (h * w))
            got.append([p + at[a] for a in ((1, 2) if axes == 2 else range(axes))])
        p += max(f, h, w)
    return got[:n]


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    order = random.Random(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, device="cuda", generator=g)  # noqa: E731
    s = {"case": dict(c)}
    if c["op"] == "plan":
        return _prepare_plan(c, s, order)
    if c["op"] == "sample":
        n, v = c["rows"], c["vocab"]
        x = 2 * rand(n, v)
        peaks = min(v, 40)  # a few tokens stand out, as they do where a text goes on
        x.scatter_add_(1, (uniform(n, peaks) * v).long().clamp_max(v - 1), 9 * uniform(n, peaks) + 2)
        s["logits"] = x.to(_TYPES[c["type"]])
        s["u"] = uniform(n)
        t = 0.6 + 0.8 * uniform(n)
        if c["kind"] == "all":
            t = torch.where(uniform(n) < 0.1, 0.0, t)  # some requests are greedy
        s["temperature"] = t
        some = lambda x, off: torch.where(uniform(n) < 0.25, off, x)  # noqa: E731  some requests leave a cut out
        s["top_k"] = some((20 + 80 * uniform(n)).int(), torch.zeros(n, dtype=torch.int32, device="cuda")) if c["kind"] in ("all", "top_k") else None
        s["top_p"] = some(0.8 + 0.19 * uniform(n), 1.0) if c["kind"] in ("all", "top_p") else None
        s["min_p"] = some(0.1 * uniform(n), 0.0) if c["kind"] in ("all", "min_p") else None
        s["ids"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(n, device="cuda")
        return s
    if c["op"] == "rope":
        n, m = c["tokens"], c["seqs"]
        each = [n // m + (i < n % m) for i in range(m)]
        per = [-(-(20 + e) // PAGE) for e in each]
        at = [_positions(e, c["axes"], c["start"] + 11 * i) for i, e in enumerate(each)]
        s["pos"] = _whole([p for a in at for p in a]).t().contiguous()
        s["seq"] = _whole([i for i in range(m) for _ in range(each[i])])
        s["slot"] = _whole([j for e in each for j in range(3, 3 + e)])
        # the rows of a fused projection: q | k | v, one row a token
        wide = (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
        qd, kd = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        rows = rand(n, wide).to(_TYPES[c["in"]])
        s["q"], s["k"], s["v"] = rows[:, :qd], rows[:, qd: qd + kd], rows[:, qd + kd:]
        s["out"] = torch.empty(n, qd, dtype=_TYPES[c["type"]], device="cuda")
        layers, s["layer"] = 2, 1
    else:
        q, kv = _sizes(c)
        per = [-(-k // PAGE) for k in kv]
        s["q"] = rand(sum(q), c["heads"] * c["head_dim"]).to(_TYPES[c["type"]])
        s["out"] = torch.empty_like(s["q"])
        s["start"] = _whole([sum(q[:i]) for i in range(len(q) + 1)])
        s["kv_len"] = _whole(kv)
        s["work"] = torch.empty(96 << 20, dtype=torch.uint8, device="cuda")
        layers, s["layer"] = 1, 0
    s["table"], pages = _table(per, order)
    s["pages"] = torch.empty(layers, pages, 2, c["kv_heads"], PAGE, c["head_dim"], dtype=_TYPES[c["type"]], device="cuda").normal_(generator=g)
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


def _prepare_plan(c, s, order):
    got, rows = _requests(c)
    n, m = c["requests"], c["seqs"]
    names = list(range(m))
    order.shuffle(names)
    r = random.Random(m)
    lens = [0] * m
    for i, q in enumerate(names):
        lens[q] = got[i][0] if i < n else r.randint(0, c["most"])  # the step leaves some sequences alone
    most = -(-c["most"] // PAGE)
    per = [-(-x // PAGE) for x in lens]
    need = sum(max(0, -(-(k + a) // PAGE) - -(-h // PAGE)) for h, k, a in got)
    total = sum(per) + need + 7
    ids = list(range(total))
    order.shuffle(ids)
    table, at = [], 0
    for p in per:
        table.append(ids[at: at + p] + [0] * (most - p))
        at += p
    s["table"] = _whole(table)
    s["free"] = _whole(ids[at:] + [0] * at)  # a stack: the free pages, then room for those that come back
    s["n_free"], s["n_free_out"] = _whole([total - at]), _whole([0])
    s["seqs"] = _whole(names[:n])
    s["keep"], s["add"] = _whole([k for _, k, _ in got]), _whole([a for _, _, a in got])
    s["lens"] = _whole(lens)
    s["lens_out"] = s["lens"].clone()
    s["rows"] = rows
    s["pages"] = torch.zeros(1, total, 2, 1, PAGE, 8, dtype=torch.float16, device="cuda")
    s["out"] = {k: torch.empty(v, dtype=torch.int32, device="cuda") for k, v in
                {"q_start": n + 1, "kv_len": n, "positions": rows, "row_seqs": rows, "slots": rows, "last": n}.items()}
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


ROPE_BASE, ROPE_FACTOR = 1000000.0, 8.0


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"plan": _plan, "rope": _rope, "attn": _attn, "sample": _sample}[op](s)


# ------------------------------------------------------------------ the plain forms
def _plan(s):
    q, keep, add, table, lens = s["seqs"].long(), s["keep"].long(), s["add"].long(), s["table"], s["lens"]
    pages = lambda x: (x + PAGE - 1) // PAGE  # noqa: E731
    have, want = pages(lens[q].long()), pages(keep + add)
    n_free = s["n_free"].long()
    room = n_free + (have - want).clamp_min(0).sum()
    taken = (add.cumsum(0) <= s["rows"]) & ((want - have).clamp_min(0).cumsum(0) <= room)
    now = torch.where(taken, keep + add, keep)
    length = torch.where(taken, add, 0)
    end = pages(now)
    each = torch.arange(table.shape[1], device="cuda")
    # pages behind the new ends go to the stack, the missing ones come from its top
    back = (each >= end[:, None]) & (each < have[:, None])
    at = n_free + back.flatten().cumsum(0) - 1
    free = s["free"]
    freed = back.sum()
    mine = table[q]
    ids = torch.where(back.flatten(), at, len(free))  # entries that stay go to a spare place
    wide = torch.cat((free, free[:1]))
    wide[ids] = mine.flatten()
    free.copy_(wide[:-1])
    new = (each >= have[:, None]) & (each < end[:, None])
    top = n_free + freed - new.flatten().cumsum(0)
    mine = torch.where(new, free[top.clamp(0, len(free) - 1)].view_as(new), mine)
    table[q] = mine
    s["lens_out"].copy_(lens)
    s["lens_out"][q] = now.int()
    s["n_free_out"].copy_((n_free + freed - new.sum()).int())
    o = s["out"]
    o["q_start"][0] = 0
    o["q_start"][1:] = length.cumsum(0).int()
    o["kv_len"].copy_(now.int())
    o["last"].copy_(torch.where(length > 0, o["q_start"][1:] - 1, NONE))
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    who = torch.bucketize(row, o["q_start"][1:], right=True)
    live = who < len(q)
    who = who.clamp_max(len(q) - 1)
    pos = keep[who] + row - o["q_start"][who]
    o["positions"].copy_(torch.where(live, pos, 0))
    o["row_seqs"].copy_(torch.where(live, q[who], NONE))
    page = mine[who, (pos // PAGE).clamp(0, table.shape[1] - 1)]
    o["slots"].copy_(torch.where(live, page * PAGE + pos % PAGE, NONE))
    return [o[k] for k in ("q_start", "kv_len", "positions", "row_seqs", "slots", "last")] + [s["table"], free, s["lens_out"], s["n_free_out"]]


def _axis_of(c):
    """The axis of each pair."""
    shares, half = _shares(c), c["rot"] // 2
    i = torch.arange(half, device="cuda")
    if c["order"] == "blocks":
        return torch.bucketize(i, torch.tensor(shares, device="cuda").cumsum(0), right=True)
    a = i % c["axes"]  # in turns, as long as the axis has pairs left; the rest is of the first axis
    return torch.where(i // c["axes"] < torch.tensor(shares, device="cuda")[a], a, 0)


def _rope(s):
    c = s["case"]
    axis = _axis_of(c)
    i, rot = torch.arange(len(axis), device="cuda").double(), torch.tensor(float(c["rot"]), device="cuda", dtype=torch.float64)
    if c["freqs"] == "own":  # the pair's number among those of its axis
        mine = axis[None] == torch.arange(c["axes"], device="cuda")[:, None]
        i = (mine.cumsum(1) - 1).gather(0, axis[None])[0].double()
        rot = 2.0 * mine.sum(1).double()[axis]
    base = ROPE_BASE
    if c["scaling"] == "ntk":
        base = base * ROPE_FACTOR ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if c["scaling"] == "linear":
        f = f / ROPE_FACTOR
    a = s["pos"].t().double()[:, axis] * f
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    s["out"].copy_(_turn(c, s["q"], cos, sin).flatten(1))
    seq, slot = s["seq"].long(), s["slot"].long()
    page, at = s["table"].long()[seq, slot // PAGE], slot % PAGE
    pages = s["pages"][s["layer"]]
    pages[page, 0, :, at] = _turn(c, s["k"], cos, sin).to(pages.dtype)
    pages[page, 1, :, at] = s["v"].float().view(len(seq), -1, c["head_dim"]).to(pages.dtype)
    return s["out"], pages


def _turn(c, x, cos, sin):
    rot = c["rot"]
    y = x.float().reshape(x.shape[0], -1, c["head_dim"]).clone()
    r = y[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["layout"] == "interleaved" else (r[..., : rot // 2], r[..., rot // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    y[..., :rot] = torch.stack((u, v), -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat((u, v), -1)
    return y


def _attn(s):
    c = s["case"]
    hd, n, most = c["head_dim"], c["chunks"], c["q_max"]
    start, length = s["start"].long(), s["kv_len"].long()
    first = length - (start[1:] - start[:-1])  # position of a chunk's first token
    low = (first - c["window"] + 1).clamp_min(0)
    # the positions that a chunk's tokens see: the first ones, then the windows
    t = torch.cat((torch.arange(c["sinks"], device="cuda").expand(n, -1),
                   low[:, None] + torch.arange(min(c["kv_max"], c["window"] + most - 1), device="cuda")), 1)
    there = t < length[:, None]
    there[:, : c["sinks"]] &= t[:, : c["sinks"]] < low[:, None]
    at = torch.where(there, t, 0)
    page = s["table"].long().gather(1, at // PAGE)
    pages = s["pages"][s["layer"]]
    k, v = (pages[page, x, :, at % PAGE].permute(0, 2, 1, 3).float() for x in (0, 1))  # chunk, head, position, element
    i = torch.arange(most, device="cuda")
    live = i < (start[1:] - start[:-1])[:, None]
    row = torch.where(live, start[:-1, None] + i, 0)
    q = s["q"].float()[row].view(n, most, c["kv_heads"], -1, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (q @ k.transpose(-1, -2)) / math.sqrt(hd)
    own_pos = (first[:, None] + i)[..., None]  # a token's own position
    see = (t[:, None] <= own_pos) & ((t[:, None] > own_pos - c["window"]) | (t[:, None] < c["sinks"])) & there[:, None]
    see = see[:, None, None].expand(-1, -1, c["heads"] // c["kv_heads"], -1, -1).flatten(2, 3)
    x = x.masked_fill(~see, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    y = (x @ v) / x.sum(-1, keepdim=True).clamp_min(1e-30)
    y = y.view(n, c["heads"], most, hd).transpose(1, 2).flatten(2)
    s["out"][row[live]] = y[live].to(s["out"].dtype)
    return s["out"]


def _sample(s):
    """In 64 bits: which token is drawn, and which is cut, depends on which of two near sums is larger."""
    x = s["logits"].double()
    n, v = x.shape
    t = s["temperature"].double()[:, None]
    greedy = t == 0
    z = (x.amax(-1, keepdim=True) - x) / torch.where(greedy, 1.0, t)
    w = torch.where(z > 64 * math.log(2.0), 0.0, torch.exp(-z))
    order = x.sort(dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(v, device="cuda")
    kept = torch.ones_like(ws, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        kept &= (k == 0) | (rank < k)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        sums = (ws * kept).cumsum(-1)
        kept &= (p >= 1) | (rank == 0) | (sums - ws < p * sums[:, -1:])
    if s["min_p"] is not None:
        kept &= ws >= s["min_p"].double()[:, None]
    kept = torch.empty_like(kept).scatter_(1, order, kept)
    w = w * kept
    sums = w.cumsum(-1)
    ids = (sums > s["u"].double()[:, None] * sums[:, -1:]).int().argmax(-1)
    ids = torch.where(greedy[:, 0], order[:, 0], ids)
    got = (w.gather(1, ids[:, None]) / sums[:, -1:]).log()[:, 0]
    s["ids"].copy_(ids)
    s["logprobs"].copy_(torch.where(greedy[:, 0], 0.0, got))
    return s["ids"], s["logprobs"]


# ------------------------------------------------------------------ the framework's calls
def _own(s, op):
    if "module" not in s:
        if "fishai-engine_b200" not in sys.path:
            sys.path.insert(0, "fishai-engine_b200")
        from fishai_engine import paged, sampling
        s["module"] = sampling if op == "sample" else paged
        if op != "sample":
            s["kv"] = paged.PagedKV(s["pages"], s["table"])
        if op == "rope":
            c = s["case"]
            s["rope"] = paged.Rope(c["head_dim"], rot_dim=c["rot"], base=ROPE_BASE, layout=c["layout"], scaling=c["scaling"], factor=ROPE_FACTOR,
                                   axes=_shares(c), axis_order=c["order"], axis_freqs=c["freqs"])
    m = s["module"]
    if op == "plan":
        o = s["out"]
        m.plan_step(s["kv"], s["add"], s["lens"], s["free"], s["n_free"], o["q_start"], o["kv_len"], o["positions"], o["row_seqs"],
                    seqs=s["seqs"], keep=s["keep"], lengths_out=s["lens_out"], n_free_out=s["n_free_out"], slots=o["slots"], last=o["last"],
                    err=s["err"])
        return [o[k] for k in ("q_start", "kv_len", "positions", "row_seqs", "slots", "last")] + [s["table"], s["free"], s["lens_out"],
                                                                                                s["n_free_out"]]
    if op == "rope":
        m.rope_append(s["kv"], s["layer"], s["rope"], s["q"], s["k"], s["v"], s["pos"], s["seq"], s["out"], slots=s["slot"], err=s["err"])
        return s["out"], s["pages"][s["layer"]]
    if op == "attn":
        c = s["case"]
        m.attention(s["kv"], s["layer"], s["q"], s["start"], s["kv_len"], s["out"], max_q=c["q_max"], window=c["window"], sinks=c["sinks"],
                    workspace=s["work"], err=s["err"])
        return s["out"]
    m.sample_logits(s["logits"], s["u"], s["ids"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                    logprobs=s["logprobs"])
    return s["ids"], s["logprobs"]


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(c, seed):
    if c["op"] == "sample" and c["rows"] * c["vocab"] > 30_000_000:
        return None
    s = prepare(c, seed)

    def plan():
        """One request after another."""
        table, lens, free, n_free = s["table"].tolist(), s["lens"].tolist(), s["free"].tolist(), int(s["n_free"])
        todo = list(zip(s["seqs"].tolist(), s["keep"].tolist(), s["add"].tolist()))
        pages = lambda x: math.ceil(x / PAGE)  # noqa: E731
        room = n_free + sum(max(0, pages(lens[q]) - pages(k + a)) for q, k, a in todo)
        left, starts, kv, last, takes = s["rows"], [0], [], [], []
        for q, k, a in todo:
            left -= a
            room -= max(0, pages(k + a) - pages(lens[q]))
            takes.append(left >= 0 and room >= 0)
            kv.append(k + a if takes[-1] else k)
            starts.append(starts[-1] + (a if takes[-1] else 0))
            last.append(starts[-1] - 1 if takes[-1] and a else NONE)
        for (q, _, _), m in zip(todo, kv):
            for e in range(pages(m), pages(lens[q])):
                free[n_free] = table[q][e]
                n_free += 1
        for (q, _, _), m in zip(todo, kv):
            for e in range(pages(lens[q]), pages(m)):
                n_free -= 1
                table[q][e] = free[n_free]
        pos, seq, slot = [], [], []
        for (q, k, a), yes in zip(todo, takes):
            for p in range(k, k + a if yes else k):
                pos.append(p)
                seq.append(q)
                slot.append(table[q][p // PAGE] * PAGE + p % PAGE)
        pad = s["rows"] - len(pos)
        for (q, _, _), m in zip(todo, kv):
            lens[q] = m
        return [_whole(v) for v in (starts, kv, pos + [0] * pad, seq + [NONE] * pad, slot + [NONE] * pad, last, table, free, lens, [n_free])]

    def rope():
        shares, rot, f, axis = _shares(c), c["rot"], [], []
        if c["order"] == "blocks":
            axis = [a for a, n in enumerate(shares) for _ in range(n)]
        else:
            axis = [0] * (rot // 2)
            for a in range(1, c["axes"]):
                for j in range(shares[a]):
                    axis[a + c["axes"] * j] = a
        for i, a in enumerate(axis):
            j, width = (i, rot) if c["freqs"] == "shared" else (axis[:i].count(a), 2 * axis.count(a))
            base = ROPE_BASE * (math.pow(ROPE_FACTOR, width / (width - 2.0)) if c["scaling"] == "ntk" else 1.0)
            f.append(math.pow(base, -2.0 * j / width) / (ROPE_FACTOR if c["scaling"] == "linear" else 1.0))
        angle = torch.stack([s["pos"][a].double() * x for a, x in zip(axis, f)], 1)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        half = rot // 2

        def rotated(x):
            x = x.double().reshape(len(x), -1, c["head_dim"])
            one = list(range(0, rot, 2)) if c["layout"] == "interleaved" else list(range(half))
            two = list(range(1, rot, 2)) if c["layout"] == "interleaved" else list(range(half, rot))
            z = torch.complex(x[..., one], x[..., two]) * turn
            y = x.clone()
            y[..., one], y[..., two] = z.real, z.imag
            return y

        pages = s["pages"][s["layer"]].double()
        k, v = rotated(s["k"]), s["v"].double().reshape(c["tokens"], -1, c["head_dim"])
        flat = pages.permute(0, 3, 1, 2, 4).reshape(-1, 2, c["kv_heads"], c["head_dim"]).clone()  # (page, position), k | v, head, element
        flat[s["table"][s["seq"].long(), (s["slot"] // PAGE).long()].long() * PAGE + s["slot"].long() % PAGE] = torch.stack((k, v), 1)
        pages = flat.view(-1, PAGE, 2, c["kv_heads"], c["head_dim"]).permute(0, 2, 3, 1, 4).contiguous()
        return rotated(s["q"]).reshape(c["tokens"], -1), pages

    def attn():
        hd, rep = c["head_dim"], c["heads"] // c["kv_heads"]
        q, kv = _sizes(c)
        out = torch.zeros(sum(q), c["heads"], hd, dtype=torch.float64, device="cuda")
        row = 0
        for n in range(c["chunks"]):
            ids = s["table"][n][: -(-kv[n] // PAGE)].long()
            mine = s["q"][row: row + q[n]].view(q[n], c["heads"], hd).double()
            gap = torch.arange(kv[n] - q[n], kv[n], device="cuda")[:, None] - torch.arange(kv[n], device="cuda")
            seen = (gap >= 0) & ((gap < c["window"]) | (torch.arange(kv[n], device="cuda") < c["sinks"]))
            use = seen.any(0).nonzero().flatten()
            for h in range(c["heads"]):
                k, v = (s["pages"][s["layer"], :, x, h // rep][ids].reshape(-1, hd)[use].double() for x in (0, 1))
                a = torch.einsum("id,td->it", mine[:, h], k) * hd ** -0.5
                out[row: row + q[n], h] = torch.softmax(a.masked_fill_(~seen[:, use], -math.inf), -1) @ v
            row += q[n]
        return out.flatten(1)

    def sample():
        """A row at a time, from the sorted candidates."""
        host = {k: (None if s[k] is None else s[k].cpu().numpy()) for k in ("u", "temperature", "top_k", "top_p", "min_p")}
        logits = s["logits"].double().cpu().numpy()
        ids, logs = [], []
        for r, x in enumerate(logits):
            best = int(x.argmax())
            t = float(host["temperature"][r])
            if t == 0:
                ids.append(best)
                logs.append(0.0)
                continue
            by_size = np.lexsort((np.arange(len(x)), -x))
            if host["top_k"] is not None and host["top_k"][r]:
                by_size = by_size[: host["top_k"][r]]
            w = np.exp((x[by_size] - x[best]) / t)
            w[(x[best] - x[by_size]) / t > 64 * math.log(2.0)] = 0
            if host["top_p"] is not None and host["top_p"][r] < 1:
                need, total, n = float(host["top_p"][r]) * math.fsum(w), np.cumsum(w), 1
                n += int(np.searchsorted(total, need))  # the first place where the sum is enough
                by_size, w = by_size[:n], w[:n]
            if host["min_p"] is not None:
                fine = w >= float(host["min_p"][r])
                by_size, w = by_size[fine], w[fine]
            by_id = np.argsort(by_size)
            total = np.cumsum(w[by_id])
            at = int(np.searchsorted(total, float(host["u"][r]) * total[-1], side="right"))
            ids.append(int(by_size[by_id][at]))
            logs.append(math.log(w[by_id][at] / total[-1]))
        return _whole(ids), torch.tensor(logs, dtype=torch.float64, device="cuda")

    return {"plan": plan, "rope": rope, "attn": attn, "sample": sample}[c["op"]]()
