"""Plain 64-bit forms of the paged operators, and error bounds derived from the
arithmetic the kernels may use."""
import math
import random

import torch

PAGE = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    """largest relative error of one rounding to the type"""
    return torch.finfo(dtype).eps / 2


def make_cache(lens, n_layers, kvh, hd, dtype, seed, spare=3, junk=None):
    """pages with random K and V for sequences of the given lengths, shuffled,
    and their table; entries behind a sequence's end are page 0's number or
    junk.  Slots of no position hold NaN: whatever reads them shows it."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = random.Random(seed)
    per = [-(-n // PAGE) for n in lens]
    total = sum(per) + spare
    ids = list(range(total))
    rng.shuffle(ids)
    most = max(max(per), 1)
    table = torch.full((len(lens), most), 0 if junk is None else junk, dtype=torch.int64)
    pages = torch.full((n_layers, total, 2, kvh, PAGE, hd), float("nan"), dtype=dtype, device="cuda")
    at = 0
    for s, n in enumerate(lens):
        mine = ids[at: at + per[s]]
        at += per[s]
        table[s, : per[s]] = torch.tensor(mine, dtype=torch.int64)
        for j, page in enumerate(mine):
            m = min(PAGE, n - j * PAGE)
            pages[:, page, :, :, :m] = torch.randn(n_layers, 2, kvh, m, hd, device="cuda", generator=g).to(dtype)
    return pages, table.to(torch.int32).cuda()


def rows_of(pages, table, layer, seq, n):
    """K and V of the first n positions of a sequence: [n, kvh, hd] each"""
    ids = table[seq, : -(-n // PAGE)].long()
    x = pages[layer, ids].permute(1, 0, 3, 2, 4).reshape(2, -1, pages.shape[3], pages.shape[5])[:, :n]
    return x[0], x[1]


def attention(pages, table, layer, q, q_start, kv_len, seqs, heads, scale, window):
    """(output, bound): bound[row, head, dim] is an upper bound of what roundings
    may do.  With u the half step of the type and e = 2^-24 that of f32:
      a score is a sum of hd products in f32, off by at most (hd + 2) e
      |q|.|k| scale and by 3 e |score| in its scaling to base 2, so a weight
      exp(s) is off by that (twice: the maximum is subtracted) relatively, and
      by 4 e in exp itself; sums of n weights and of n products p v are off by
      n e more; p may be rounded to the type before its product (u); tensor
      cores may truncate rather than round their partial sums (a factor of 2);
      the result is rounded once (u |o|)."""
    hd, rep = pages.shape[5], heads // pages.shape[3]
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u, e = half_step(q.dtype), 2.0 ** -24
    sc = scale or hd ** -0.5
    start, lens = q_start.tolist(), kv_len.tolist()
    for c in range(len(lens)):
        a, b, n = start[c], start[c + 1], lens[c]
        if b == a or n == 0:
            continue
        k, v = rows_of(pages, table, layer, c if seqs is None else int(seqs[c]), n)
        k, v = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
        x = q[a:b].double().view(b - a, heads, hd)
        pos = torch.arange(n - (b - a), n, device=q.device)[:, None]
        t = torch.arange(n, device=q.device)[None]
        see = t <= pos
        if window:
            see = see & (t > pos - window)
        used = see.any(0)
        k, v = torch.where(used[:, None, None], k, 0), torch.where(used[:, None, None], v, 0)
        s = torch.einsum("ihd,thd->hit", x, k) * sc
        size = torch.einsum("ihd,thd->hit", x.abs(), k.abs()) * sc
        s = s.masked_fill(~see, -math.inf)
        m = s.amax(-1, keepdim=True).clamp_min(-1e300)
        p = torch.exp(s - m)
        w = p.sum(-1, keepdim=True)
        p = torch.where(w > 0, p / w.clamp_min(1e-300), 0)
        out[a:b] = torch.einsum("hit,thd->ihd", p, v)
        worst = torch.where(see, size, 0).amax(-1, keepdim=True)  # of a row's scores
        rel = 2 * (2 * (hd + 5) * e * worst) + (2 * n + 12) * e + (u if q.dtype != torch.float32 else 0)
        # numerator and denominator
        tol[a:b] = torch.einsum("hit,thd->ihd", p * rel, v.abs()) + out[a:b].abs() * (rel.permute(1, 0, 2) + u) + 1e-30
        if q.dtype == torch.float16:
            tol[a:b] += 2.0 ** -25  # the smallest step of f16
    return out, tol


def rope_rows(x, pos, freqs, scale, rot, layout, heads, hd):
    x = x.double().view(x.shape[0], heads, hd).clone()
    a = pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64, device=x.device)
    c, s = (a.cos() * scale)[:, None], (a.sin() * scale)[:, None]
    i0 = torch.arange(0, rot, 2) if layout == "interleaved" else torch.arange(rot // 2)
    i1 = i0 + 1 if layout == "interleaved" else i0 + rot // 2
    u, v = x[..., i0].clone(), x[..., i1].clone()
    x[..., i0], x[..., i1] = u * c - v * s, u * s + v * c
    size = x.abs()
    size[..., i0] = size[..., i1] = (u.abs() + v.abs()) * scale
    return x, size


def beam_select(logits, scores, done, k, eos, pad):
    """the definition, one request at a time"""
    nb, beams = scores.shape
    big = torch.finfo(torch.float32).max
    out = ([], [], [], [])
    for b in range(nb):
        found = []
        for j in range(beams):
            sc = float(scores[b, j])
            if not math.isfinite(sc):
                continue
            if done is not None and int(done[b, j]):
                found.append((sc, j, 0.0, pad))
                continue
            x = logits[b * beams + j].double()
            x = torch.where(x.isnan(), -math.inf, x).clamp_max(big)
            if bool((x == -math.inf).all()):
                continue
            m = x.max()
            lse = m + torch.log(torch.exp(x - m).sum())
            edge = x.topk(min(k, len(x))).values[-1]
            at = ((x >= edge) & (x != -math.inf)).nonzero().flatten()
            at = at[: 4 * k] if float(edge) == float(m) else at  # ties at the top: the lowest tokens are enough
            found += [(sc + (float(x[t]) - float(lse)), j, -float(x[t]), int(t)) for t in at]
        found.sort(key=lambda f: (-f[0], *f[1:]))  # of one beam by logit, which 64 bits of score may not tell apart
        found = found[:k]
        rows = [(s, j, t, int((done is not None and bool(done[b, j])) or t == eos)) for s, j, _, t in found]
        rows += [(-math.inf, i % beams, pad, 1) for i in range(len(rows), k)]
        for o, v in zip(out, zip(*rows)):
            o.append(list(v))
    return tuple(torch.tensor(o, dtype=d) for o, d in zip(out, (torch.float64, torch.int32, torch.int32, torch.int32)))
