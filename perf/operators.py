"""The operators of the paged serving path, as cases to be measured: rotary positions with the append to the pages,
attention of chunks of new tokens over the pages, page copies and compaction, and the beam search's selection.

`run` computes them from elementary torch operations; with `own` set it calls fishai_engine's kernels instead.

Pages are [layer][page][k | v][kv head][16 positions][head_dim]; page_table[sequence][i] holds positions 16 i .. 16 i + 15.
"""
import math
import random
import sys

import torch

own = False

PAGE = 16
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    big = {"heads": 32, "kv_heads": 8, "head_dim": 128}  # the 8B shape
    return [
        # one token of one sequence: the qkv sums of a decode step arrive in f32, the cache is f16; latency
        {"name": "rope one token", "op": "rope", **big, "in": "f32", "type": "f16", "tokens": 1, "seqs": 1, "rot": 128,
         "layout": "interleaved", "scaling": "none", "start": 2047},
        # a decode step of 64 sequences far into a stretched context, half of each head rotated
        {"name": "rope batch of 64", "op": "rope", **big, "in": "bf16", "type": "bf16", "tokens": 64, "seqs": 64, "rot": 64,
         "layout": "half", "scaling": "yarn", "start": 120000},
        # the prompts of three requests in one call
        {"name": "rope prompts of 8192", "op": "rope", **big, "in": "f16", "type": "f16", "tokens": 8192, "seqs": 3, "rot": 128,
         "layout": "interleaved", "scaling": "llama3", "start": 5},
        # decode of one sequence at the end of the model's context; latency and split work
        {"name": "attn one token", "op": "attn", **big, "type": "f16", "chunks": 1, "q_min": 1, "q_max": 1, "kv_min": 8192,
         "kv_max": 8192, "window": 0},
        # batched decode, caches of every length
        {"name": "attn batch of 64", "op": "attn", **big, "type": "f16", "chunks": 64, "q_min": 1, "q_max": 1, "kv_min": 37,
         "kv_max": 4096, "window": 0},
        # one to three tokens of five short sequences over the f32 cache of the tiny shape
        {"name": "attn tiny f32", "op": "attn", "heads": 8, "kv_heads": 2, "head_dim": 64, "type": "f32", "chunks": 5,
         "q_min": 1, "q_max": 3, "kv_min": 1, "kv_max": 512, "window": 0},
        # one scheduling step of a server: prompts, parts of prompts and single tokens together
        {"name": "attn mixed chunks", "op": "attn", **big, "type": "bf16", "chunks": 8, "q_min": 1, "q_max": 1024, "kv_min": 900,
         "kv_max": 4096, "window": 0},
        # the last chunk of 2048 tokens of a prompt that fills the context
        {"name": "attn chunk of 2048", "op": "attn", **big, "type": "f16", "chunks": 1, "q_min": 2048, "q_max": 2048,
         "kv_min": 8192, "kv_max": 8192, "window": 0},
        # 64 sequences forked: the last, partly filled page of each copied in every layer
        {"name": "pages fork of 64", "op": "fork", "kv_heads": 8, "head_dim": 128, "type": "f16", "layers": 32, "pages": 192,
         "pairs": 64},
        # four sequences of 2048 positions thinned out to about half
        {"name": "pages compact", "op": "compact", "kv_heads": 8, "head_dim": 128, "type": "f16", "layers": 32, "seqs": 4,
         "length": 2048, "keep": 0.5},
        # one request with four beams; latency
        {"name": "beam 1x4", "op": "beam", "batch": 1, "beams": 4, "vocab": 128256, "k": 4, "type": "f32"},
        # 32 requests with eight beams each, some beams finished
        {"name": "beam 32x8", "op": "beam", "batch": 32, "beams": 8, "vocab": 128256, "k": 8, "type": "f32"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["rope", "rope", "attn", "attn", "attn", "attn", "fork", "compact", "beam", "beam"])
        kv = rng.choice([1, 2, 4, 8, 8])
        hd = rng.choice([64, 128, 128])
        rep = rng.choice([1, 2, 4, 4, 7, 8])
        kind = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
        if op == "rope":
            n = _log(rng, 1, 8192)
            c = {"op": op, "heads": kv * rep, "kv_heads": kv, "head_dim": hd, "in": rng.choice(["f32", "f16", "bf16"]), "type": kind,
                 "tokens": n, "seqs": rng.randint(1, min(n, 64)), "rot": rng.choice([hd, hd, hd // 2, 24]),
                 "layout": rng.choice(["interleaved", "half"]), "scaling": rng.choice(["none", "linear", "ntk", "llama3", "yarn"]),
                 "start": _log(rng, 1, 500000)}
        elif op == "attn":
            q = rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 1, 2048)])
            n = rng.choice([1, _log(rng, 1, 64)])
            kv_max = max(q, _log(rng, 1, 8192))
            c = {"op": op, "heads": kv * rep, "kv_heads": kv, "head_dim": hd, "type": kind, "chunks": n, "q_min": rng.randint(1, q), "q_max": q,
                 "kv_min": rng.randint(1, kv_max), "kv_max": kv_max, "window": rng.choice([0, 0, _log(rng, 1, 4096)])}
            if kind == "f32":  # the f32 cache is the reference's own values, not the fast path
                c.update(q_min=min(c["q_min"], 32), q_max=min(q, 32))
        elif op == "fork":
            n = _log(rng, 1, 96)
            c = {"op": op, "kv_heads": kv, "head_dim": hd, "type": kind, "layers": rng.choice([2, 4, 32]), "pages": 2 * n + rng.randint(0, 64),
                 "pairs": n}
        elif op == "compact":
            c = {"op": op, "kv_heads": kv, "head_dim": hd, "type": kind, "layers": rng.choice([2, 4, 32]), "seqs": rng.randint(1, 6),
                 "length": _log(rng, 16, 2500), "keep": rng.uniform(0.1, 0.95)}
        else:
            c = {"op": op, "batch": _log(rng, 1, 32), "beams": rng.randint(1, 12), "vocab": rng.choice([32000, 128256, _log(rng, 50, 200000)]),
                 "type": rng.choice(["f32", "f32", "f16", "bf16"])}
            c["k"] = rng.randint(1, min(16, c["vocab"]))
        if _cost(c) <= top and not (op == "attn" and c["chunks"] * c["heads"] * c["q_max"] * (c["kv_max"] + 15) > 2 ** 30):
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / (1.6e15 if c["type"] != "f32" else 3e13))


def _sizes(c):
    """The chunks' lengths and their caches' lengths, the same for every seed: one of the largest, the others spread down to
    the smallest."""
    r = random.Random(c["chunks"] * 7919 + c["kv_max"] * 31 + c["q_max"])
    n = c["chunks"]
    kv = [c["kv_max"]] + [r.randint(c["kv_min"], c["kv_max"]) for _ in range(n - 1)]
    q = [c["q_max"]] + [r.randint(c["q_min"], c["q_max"]) if r.random() < 0.5 else c["q_min"] for _ in range(n - 1)]
    return [min(a, b) for a, b in zip(q, kv)], kv


def _pairs(q, kv, window):
    """How many (query, position) pairs a chunk of q tokens sees, and how many positions of its cache any of them sees."""
    first = kv - q  # position of the first token
    low = max(0, first - window + 1) if window else 0
    if window:
        full = max(0, min(q, kv - max(first, window - 1)))  # tokens that see a whole window
        part = q - full
        seen = full * window + part * (first + 1) + part * (part - 1) // 2
    else:
        seen = q * (first + 1) + q * (q - 1) // 2
    return seen, kv - low


def work(c):
    t = _SIZE[c["type"]]
    if c["op"] == "rope":
        n = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
        return {"bytes": n * (_SIZE[c["in"]] + t), "flops": 6 * n}
    if c["op"] == "attn":
        q, kv = _sizes(c)
        both = [_pairs(a, b, c["window"]) for a, b in zip(q, kv)]
        rows = 2 * sum(q) * c["heads"] * c["head_dim"]
        return {"bytes": t * (rows + 2 * c["kv_heads"] * c["head_dim"] * sum(p[1] for p in both)),
                "flops": 4 * c["heads"] * c["head_dim"] * sum(p[0] for p in both)}
    if c["op"] == "fork":
        return {"bytes": 2 * t * sum(_slots(c)) * c["layers"] * 2 * c["kv_heads"] * c["head_dim"], "flops": 0}
    if c["op"] == "compact":
        moved = sum(sum(i != p for i, p in enumerate(k)) for k in _keeps(c))
        return {"bytes": 2 * t * moved * c["layers"] * 2 * c["kv_heads"] * c["head_dim"], "flops": 0}
    n = c["batch"] * c["beams"] * c["vocab"]
    return {"bytes": n * t, "flops": 4 * n}


def _slots(c):
    """Positions that a fork copies of each page: mostly part of one, some whole."""
    r = random.Random(c["pairs"] * 31 + c["layers"])
    return [r.choice([16, r.randint(1, 15)]) for _ in range(c["pairs"])]


def _keeps(c):
    r = random.Random(c["length"] * 31 + c["seqs"])
    lengths = [c["length"]] + [r.randint(1, c["length"]) for _ in range(c["seqs"] - 1)]
    return [[p for p in range(n) if p < 4 or r.random() < c["keep"]] for n in lengths]  # the first few positions always stay


def _pages(c, layers, n, g):
    """The pages of a cache in use."""
    kv, hd, kind = c["kv_heads"], c["head_dim"], _TYPES[c["type"]]
    x = torch.empty(layers, n, 2, kv, PAGE, hd, dtype=kind, device="cuda")
    return x.normal_(generator=g)


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    order = random.Random(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": dict(c)}
    if c["op"] == "beam":
        rows = c["batch"] * c["beams"]
        s["logits"] = (3 * rand(rows, c["vocab"])).to(_TYPES[c["type"]])
        s["scores"] = -6 * torch.rand(c["batch"], c["beams"], device="cuda", generator=g)
        s["done"] = (torch.rand(c["batch"], c["beams"], device="cuda", generator=g) < 0.1).int()
        s["done"][:, 0] = 0  # a request with no open beam would have ended
        s["eos"], s["pad"] = 2, 0
        s["out"] = [torch.empty(c["batch"], c["k"], dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32, torch.int32)]
        s["work"] = torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
        return s
    if c["op"] == "fork":
        ids = list(range(c["pages"]))
        order.shuffle(ids)
        s["pages"] = _pages(c, c["layers"], c["pages"], g)
        s["table"] = whole(ids).view(1, -1)
        s["src"], s["dst"], s["slots"] = whole(ids[: c["pairs"]]), whole(ids[c["pairs"]: 2 * c["pairs"]]), whole(_slots(c))
        return s
    if c["op"] == "compact":
        keeps = _keeps(c)
        per = -(-c["length"] // PAGE)
        ids = list(range(per * c["seqs"]))
        order.shuffle(ids)
        s["pages"] = _pages(c, c["layers"], len(ids), g)
        s["table"] = whole(ids).view(c["seqs"], per)
        s["keep"] = whole([p for k in keeps for p in k])
        s["start"] = whole([sum(map(len, keeps[:i])) for i in range(len(keeps) + 1)])
        s["seq"] = whole(list(range(c["seqs"])))
        return s
    if c["op"] == "rope":
        n, m = c["tokens"], c["seqs"]
        each = [n // m + (i < n % m) for i in range(m)]
        per = [-(-(20 + e) // PAGE) for e in each]
        seq = [i for i in range(m) for _ in range(each[i])]
        slot = [j for e in each for j in range(3, 3 + e)]
        s["pos"] = whole([c["start"] + 97 * i + j for i, j in zip(seq, slot)])
        s["seq"], s["slot"] = whole(seq), whole(slot)
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
        s["start"] = whole([sum(q[:i]) for i in range(len(q) + 1)])
        s["kv_len"] = whole(kv)
        s["work"] = torch.empty(96 << 20, dtype=torch.uint8, device="cuda")
        layers, s["layer"] = 1, 0
    ids = list(range(sum(per) + 1))
    order.shuffle(ids)
    at, table = 0, []
    for p in per:
        table.append(ids[at: at + p] + [ids[-1]] * (max(per) - p))  # behind a sequence's end: any page
        at += p
    s["table"] = whole(table)
    s["pages"] = _pages(c, layers, len(ids), g)
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


ROPE_BASE, ROPE_FACTOR, ROPE_CONTEXT = 500000.0, 8.0, 8192


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"rope": _rope, "attn": _attn, "fork": _fork, "compact": _compact, "beam": _beam}[op](s)


# ------------------------------------------------------------------ the plain forms
def _angles(c, pos):
    """Angles in 64 bits: positions go to hundreds of thousands."""
    rot, base = c["rot"], ROPE_BASE
    i = torch.arange(0, rot, 2, device=pos.device, dtype=torch.float64)
    scale = 1.0
    if c["scaling"] == "ntk":
        base = base * ROPE_FACTOR ** (rot / (rot - 2))
    f = base ** (-i / rot)
    if c["scaling"] == "linear":
        f = f / ROPE_FACTOR
    elif c["scaling"] == "llama3":  # frequencies of long waves are stretched, of short ones kept, between the two blended
        t = (ROPE_CONTEXT * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)
        t = t.clamp(0, 1)
        f = f * t + f / ROPE_FACTOR * (1 - t)
    elif c["scaling"] == "yarn":
        at = lambda turns: rot * math.log(ROPE_CONTEXT / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        t = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / ROPE_FACTOR * t + f * (1 - t)
        scale = 0.1 * math.log(ROPE_FACTOR) + 1.0
    a = pos.double()[:, None] * f
    return (a.cos() * scale).float()[:, None], (a.sin() * scale).float()[:, None]


def _turn(c, x, cos, sin):
    rot = c["rot"]
    y = x.float().view(x.shape[0], -1, c["head_dim"]).clone()
    r = y[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["layout"] == "interleaved" else (r[..., : rot // 2], r[..., rot // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    y[..., :rot] = torch.stack((u, v), -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat((u, v), -1)
    return y


def _rope(s):
    c = s["case"]
    cos, sin = _angles(c, s["pos"])
    s["out"].copy_(_turn(c, s["q"], cos, sin).flatten(1))
    seq, slot = s["seq"].long(), s["slot"].long()
    page, at = s["table"].long()[seq, slot // PAGE], slot % PAGE
    pages = s["pages"][s["layer"]]
    pages[page, 0, :, at] = _turn(c, s["k"], cos, sin).to(pages.dtype)
    pages[page, 1, :, at] = s["v"].float().view(len(seq), -1, c["head_dim"]).to(pages.dtype)
    return s["out"], pages


def _attn(s):
    c = s["case"]
    hd, n, most = c["head_dim"], c["chunks"], c["q_max"]
    kv = s["pages"][s["layer"]][s["table"].long()].permute(2, 0, 3, 1, 4, 5).flatten(3, 4).float()  # k | v, chunk, head, position
    start, length = s["start"].long(), s["kv_len"].long()
    i = torch.arange(most, device="cuda")
    live = i < (start[1:] - start[:-1])[:, None]
    row = torch.where(live, start[:-1, None] + i, 0)
    q = s["q"].float()[row].view(n, most, c["kv_heads"], -1, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (q @ kv[0].transpose(-1, -2)) / math.sqrt(hd)
    at = (length - (start[1:] - start[:-1]))[:, None] + i  # a token's own position
    t = torch.arange(kv.shape[3], device="cuda")
    see = t <= at[..., None]
    if c["window"]:
        see &= t > at[..., None] - c["window"]
    see = see[:, None, None].expand(-1, -1, c["heads"] // c["kv_heads"], -1, -1).flatten(2, 3)
    x = x.masked_fill(~see, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    y = (x @ kv[1]) / x.sum(-1, keepdim=True).clamp_min(1e-30)
    y = y.view(n, c["heads"], most, hd).transpose(1, 2).flatten(2)
    s["out"][row[live]] = y[live].to(s["out"].dtype)
    return s["out"]


def _fork(s):
    pages, src, dst = s["pages"], s["src"].long(), s["dst"].long()
    copied = (torch.arange(PAGE, device="cuda") < s["slots"][:, None])[None, :, None, None, :, None]
    pages[:, dst] = torch.where(copied, pages[:, src], pages[:, dst])
    return pages


def _compact(s):
    pages, start, keep = s["pages"], s["start"].long(), s["keep"].long()
    n = torch.arange(len(keep), device="cuda")
    seq = torch.bucketize(n, start[1:], right=True)
    to = n - start[seq]
    table = s["table"].long()[s["seq"].long()]
    a, b = table[seq, keep // PAGE], table[seq, to // PAGE]
    pages[:, b, :, :, to % PAGE] = pages[:, a, :, :, keep % PAGE]
    return pages


def _beam(s):
    """In 64 bits: what is chosen depends on which of two near scores is larger."""
    c = s["case"]
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    x = (x - x.exp().sum(-1, keepdim=True).log()).view(c["batch"], c["beams"], -1)
    done = s["done"].bool()
    x = x.masked_fill(done[..., None], -math.inf)
    x[..., s["pad"]] = torch.where(done, 0.0, x[..., s["pad"]])
    x = x + s["scores"].double()[..., None]
    score, at = x.flatten(1).sort(dim=-1, descending=True, stable=True)
    score, at = score[:, : c["k"]], at[:, : c["k"]]
    parent, token = at // c["vocab"], at % c["vocab"]
    return score.float(), parent.int(), token.int(), (done.gather(1, parent) | (token == s["eos"])).int()


# ------------------------------------------------------------------ the framework's calls
def _own(s, op):
    if "kv" not in s and op != "beam":
        if "fishai-engine_b200" not in sys.path:
            sys.path.insert(0, "fishai-engine_b200")
        from fishai_engine import paged
        s["kv"] = paged.PagedKV(s["pages"], s["table"])
        s["paged"] = paged
        if op == "rope":
            c = s["case"]
            s["rope"] = paged.Rope(c["head_dim"], rot_dim=c["rot"], base=ROPE_BASE, layout=c["layout"], scaling=c["scaling"],
                                   factor=ROPE_FACTOR, context=ROPE_CONTEXT)
    if op == "rope":
        s["paged"].rope_append(s["kv"], s["layer"], s["rope"], s["q"], s["k"], s["v"], s["pos"], s["seq"], s["out"], slots=s["slot"],
                               err=s["err"])
        return s["out"], s["pages"][s["layer"]]
    if op == "attn":
        s["paged"].attention(s["kv"], s["layer"], s["q"], s["start"], s["kv_len"], s["out"], max_q=s["case"]["q_max"],
                             window=s["case"]["window"], workspace=s["work"], err=s["err"])
        return s["out"]
    if op == "fork":
        s["paged"].copy_pages(s["kv"], s["src"], s["dst"], slots=s["slots"])
        return s["pages"]
    if op == "compact":
        s["paged"].compact(s["kv"], s["seq"], s["keep"], s["start"])
        return s["pages"]
    if "beam" not in s:
        if "fishai-engine_b200" not in sys.path:
            sys.path.insert(0, "fishai-engine_b200")
        from fishai_engine import beam
        s["beam"] = beam
    s["beam"].select(s["logits"], s["scores"], s["done"], *s["out"], eos=s["eos"], pad=s["pad"], workspace=s["work"])
    return tuple(s["out"])


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(c, seed):
    s = prepare(c, seed)

    def freqs():
        """One frequency at a time, from the definitions of the scalings."""
        rot, got, m = c["rot"], [], 1.0
        for j in range(rot // 2):
            f = math.pow(ROPE_BASE, -2.0 * j / rot)
            if c["scaling"] == "linear":
                f /= ROPE_FACTOR
            elif c["scaling"] == "ntk":
                f = math.pow(ROPE_BASE * math.pow(ROPE_FACTOR, rot / (rot - 2.0)), -2.0 * j / rot)
            elif c["scaling"] == "llama3":
                wave = 2 * math.pi / f
                if wave > ROPE_CONTEXT / 1.0:
                    f /= ROPE_FACTOR
                elif wave >= ROPE_CONTEXT / 4.0:
                    t = (ROPE_CONTEXT / wave - 1.0) / 3.0
                    f = (1 - t) * f / ROPE_FACTOR + t * f
            elif c["scaling"] == "yarn":
                edge = [rot * math.log(ROPE_CONTEXT / (turns * 2 * math.pi)) / (2 * math.log(ROPE_BASE)) for turns in (32.0, 1.0)]
                lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
                t = min(1.0, max(0.0, (j - lo) / max(hi - lo, 0.001)))
                f = f / ROPE_FACTOR * t + f * (1 - t)
                m = 0.1 * math.log(ROPE_FACTOR) + 1.0
            got.append(f)
        return got, m

    def rope():
        f, m = freqs()
        angle = s["pos"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.full_like(angle, m), angle)[:, None]
        half, rot = c["rot"] // 2, c["rot"]

        def rotated(x):
            x = x.double().reshape(len(x), -1, c["head_dim"])
            first = list(range(0, rot, 2)) if c["layout"] == "interleaved" else list(range(half))
            second = list(range(1, rot, 2)) if c["layout"] == "interleaved" else list(range(half, rot))
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        pages = s["pages"][s["layer"]].double()
        k, v = rotated(s["k"]), s["v"].double().reshape(c["tokens"], -1, c["head_dim"])
        flat = pages.permute(0, 3, 1, 2, 4)  # page, position, k | v, head, dim
        flat = flat.reshape(-1, 2, c["kv_heads"], c["head_dim"]).clone()
        at = s["table"][s["seq"].long(), (s["slot"] // PAGE).long()].long() * PAGE + s["slot"].long() % PAGE
        flat[at] = torch.stack((k, v), 1)
        pages = flat.view(-1, PAGE, 2, c["kv_heads"], c["head_dim"]).permute(0, 2, 3, 1, 4).contiguous()
        return rotated(s["q"]).reshape(c["tokens"], -1), pages

    def attn():
        hd, rep = c["head_dim"], c["heads"] // c["kv_heads"]
        q, kv = _sizes(c)
        out = torch.zeros(sum(q), c["heads"], hd, dtype=torch.float64, device="cuda")
        table, row = s["table"].tolist(), 0
        for n in range(c["chunks"]):
            ids = torch.tensor(table[n][: -(-kv[n] // PAGE)], device="cuda")
            pages = s["pages"][s["layer"]].index_select(0, ids)
            mine = s["q"][row: row + q[n]].view(q[n], c["heads"], hd)
            for h in range(c["heads"]):
                k, v = (pages[:, x, h // rep].reshape(-1, hd)[: kv[n]].double() for x in (0, 1))
                a = torch.einsum("id,td->it", mine[:, h].double(), k) * hd ** -0.5
                gap = torch.arange(kv[n] - q[n], kv[n], device="cuda")[:, None] - torch.arange(kv[n], device="cuda")
                hidden = (gap < 0) if not c["window"] else (gap < 0) | (gap >= c["window"])
                out[row: row + q[n], h] = torch.softmax(a.masked_fill_(hidden, -math.inf), -1) @ v
            row += q[n]
        return out.flatten(1)

    def fork():
        pages = s["pages"].clone()
        for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), s["slots"].tolist()):
            pages[:, b, :, :, :n] = s["pages"][:, a, :, :, :n]
        return pages

    def compact():
        was, pages, table = s["pages"].clone(), s["pages"], s["table"].tolist()
        for n, keep in enumerate(_keeps(c)):
            for to, p in enumerate(keep):
                if to != p:
                    pages[:, table[n][to // PAGE], :, :, to % PAGE] = was[:, table[n][p // PAGE], :, :, p % PAGE]
        return pages

    def beam():
        got = ([], [], [], [])
        for b in range(c["batch"]):
            found = []
            for j in range(c["beams"]):
                old = float(s["scores"][b, j])
                if int(s["done"][b, j]):
                    found.append((old, j, s["pad"]))
                    continue
                x = s["logits"][b * c["beams"] + j].double()
                lse = float(torch.logsumexp(x, 0))
                edge = x.topk(c["k"]).values[-1]
                at = (x >= edge).nonzero().flatten().tolist()
                found += [(old + (v - lse), j, t) for v, t in zip(x[at].tolist(), at)]
            found = sorted(found, key=lambda f: (-f[0], f[1], f[2]))[: c["k"]]
            for out, values in zip(got, zip(*((f[0], f[1], f[2], int(bool(s["done"][b, f[1]]) or f[2] == s["eos"])) for f in found))):
                out.append(list(values))
        kinds = (torch.float64, torch.int32, torch.int32, torch.int32)
        return tuple(torch.tensor(g, dtype=d, device="cuda") for g, d in zip(got, kinds))

    return {"rope": rope, "attn": attn, "fork": fork, "compact": compact, "beam": beam}[c["op"]]()
