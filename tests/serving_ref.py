"""Plain 64-bit forms of the operators around a serving step, and error bounds
derived from the arithmetic the kernels may use."""
import math

import torch

import paged_ref as R

PAGE = R.PAGE
half_step = R.half_step


def sees(n, q, window, sinks, device="cuda"):
    """[q, n]: which positions each of a chunk's tokens sees"""
    pos = torch.arange(n - q, n, device=device)[:, None]
    t = torch.arange(n, device=device)[None]
    return (t <= pos) & ((t > pos - window) | (t < sinks)) if window else t <= pos


def empty_gap(pages, table, qs, kvs, window, sinks):
    """What no token of a chunk sees: NaN in its slots, and no page at all where a whole page is unseen."""
    pages, table = pages.clone(), table.clone()
    for c, (q, n) in enumerate(zip(qs, kvs)):
        if not q or not n:
            continue
        used = sees(n, q, window, sinks, "cpu").any(0)
        for e in range(-(-n // PAGE)):
            mine = used[e * PAGE: (e + 1) * PAGE]
            for slot in (~mine).nonzero().flatten().tolist():
                pages[:, int(table[c, e]), :, :, slot] = float("nan")
            if not mine.any():
                table[c, e] = 10 ** 6
    return pages, table


def attention(pages, table, q, q_start, kv_len, heads, scale, window, sinks):
    """(output, bound) of layer 0, chunk c of sequence c; the bound as in paged_ref.attention: scores are sums of hd products
    in f32, weights and their sums in f32, the weights rounded to the type once for their product, the result once."""
    hd, rep = pages.shape[5], heads // pages.shape[3]
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u, e = half_step(q.dtype), 2.0 ** -24
    sc = scale or hd ** -0.5
    for c, n in enumerate(kv_len):
        a, b = q_start[c], q_start[c + 1]
        if b == a or n == 0:
            continue
        k, v = R.rows_of(pages, table.clamp_max(pages.shape[1] - 1), 0, c, n)
        k, v = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
        x = q[a:b].double().view(b - a, heads, hd)
        see = sees(n, b - a, window, sinks)
        used = see.any(0)
        k, v = torch.where(used[:, None, None], k, 0), torch.where(used[:, None, None], v, 0)
        s = torch.einsum("ihd,thd->hit", x, k) * sc
        size = torch.einsum("ihd,thd->hit", x.abs(), k.abs()) * sc
        s = s.masked_fill(~see, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
        w = p.sum(-1, keepdim=True)
        p = torch.where(w > 0, p / w.clamp_min(1e-300), 0)
        out[a:b] = torch.einsum("hit,thd->ihd", p, v)
        worst = torch.where(see, size, 0).amax(-1, keepdim=True)
        rel = 2 * (2 * (hd + 5) * e * worst) + (2 * n + 12) * e + (u if q.dtype != torch.float32 else 0)
        tol[a:b] = torch.einsum("hit,thd->ihd", p * rel, v.abs()) + out[a:b].abs() * (rel.permute(1, 0, 2) + u) + 1e-30
        if q.dtype == torch.float16:
            tol[a:b] += 2.0 ** -25  # the smallest step of f16
    return out, tol


def plan(seqs, keep, add, rows, lens, table, free, n_free, n_pages):
    """The plan of a step, one request after another, on lists; returns (q_start, kv_len, last, pos, row_seq, slot, table, free,
    lens, n_free, flags)."""
    FULL, RANGE, PAGE_ = 128, 32, 16
    up = lambda x: -(-x // PAGE)  # noqa: E731
    table, free, lens, flags = [list(t) for t in table], list(free), list(lens), 0
    n, most, cap = len(add), len(table[0]) * PAGE, len(free)
    seqs = list(range(n)) if seqs is None else seqs
    ok = []
    for q, a, i in zip(seqs, add, range(n)):
        fine = 0 <= q < len(lens) and seqs.count(q) == 1 and 0 <= lens[q] <= most
        k = (lens[q] if 0 <= q < len(lens) else 0) if keep is None else keep[i]
        fine = fine and 0 <= k <= lens[q] and 0 <= a and k + a <= most
        ok.append((fine, k))
        flags |= 0 if fine else RANGE
    room = n_free + sum(max(0, up(lens[q]) - up(k + a)) for q, a, (f, k) in zip(seqs, add, ok) if f)
    left, now, takes, put = rows, [], [], 0
    for q, a, (f, k) in zip(seqs, add, ok):
        if f:
            left -= a
            room -= max(0, up(k + a) - up(lens[q]))
        takes.append(f and left >= 0 and room >= 0)
        flags |= FULL if f and a and not takes[-1] else 0
        now.append(k + a if takes[-1] else k)
        put += max(0, up(lens[q]) - up(now[-1])) if f else 0
    bad = n_free > cap or n_free + put > cap
    if bad:
        flags |= RANGE
        ok, takes = [(False, 0)] * n, [False] * n
    high = n_free
    for q, m, (f, _) in zip(seqs, now, ok):
        for e in range(up(m), up(lens[q])) if f else ():
            free[high] = table[q][e]
            flags |= PAGE_ if not 0 <= table[q][e] < n_pages else 0
            high += 1
    for q, m, (f, _) in zip(seqs, now, ok):
        for e in range(up(lens[q]), up(m)) if f else ():
            high -= 1
            table[q][e] = free[high]
            flags |= PAGE_ if not 0 <= free[high] < n_pages else 0
    start, kv, last, pos, who, slot = [0], [], [], [], [], []
    for q, m, a, (f, k), t in zip(seqs, now, add, ok, takes):
        kv.append(m if f else 0)
        start.append(start[-1] + (a if t else 0))
        last.append(start[-1] - 1 if t and a else -1)
        for x in range(k, m) if t else ():
            pos.append(x)
            who.append(q)
            slot.append(table[q][x // PAGE] * PAGE + x % PAGE)
        if f:
            lens[q] = m
    pad = rows - len(pos)
    return start, kv, last, pos + [0] * pad, who + [-1] * pad, slot + [-1] * pad, table, free, lens, n_free if bad else high, flags


def sample(x, u, t=1.0, k=0, p=1.0, mp=0.0):
    """One row in 64 bits: (ids that may be drawn, {id: log-probability}).  More than one id only where u is within 1e-11
    of a border between two."""
    x = torch.where(x.isnan(), -math.inf, x.double()).clamp_max(torch.finfo(torch.float32).max) + 0.0
    top = x.max()
    if float(top) == -math.inf:
        return [-1], {-1: -math.inf}
    if t == 0:
        best = int((x == top).nonzero()[0])
        return [best], {best: 0.0}
    z = (top - x) / t
    w = torch.where(z > 64 * math.log(2), 0.0, torch.exp(-z))
    order = torch.sort(x, descending=True, stable=True).indices
    ws = w[order]
    n = int((ws > 0).sum())
    if k:
        n = min(n, k)
    sums = ws[:n].cumsum(0)
    if p < 1:
        n = max(1, int((sums - ws[:n] < p * sums[-1]).sum()))
    kept = order[:n]
    kept = kept[w[kept] >= mp].sort().values
    sums = w[kept].cumsum(0)
    at = u * float(sums[-1])
    slack = 1e-11 * float(sums[-1])
    lo, hi = int((sums <= at - slack).sum()), int((sums <= at + slack).sum())
    ids = kept[lo: min(hi, len(kept) - 1) + 1].tolist()
    return ids, {i: float((w[i] / sums[-1]).log()) for i in ids}
