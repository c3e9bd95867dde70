"""The paged operators from their definitions, in float64 on the host, one sequence and one head at
a time."""
from __future__ import annotations

import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half a subnormal step


def make_pool(rng, pages, page, heads, dim, dtype, layout="nhd", layers=0, fill=None):
    shape = (pages, page, heads, dim) if layout == "nhd" else (pages, heads, page, dim)
    shape = (layers,) + shape if layers else shape
    t = torch.randn(shape, generator=rng) if fill is None else torch.full(shape, fill)
    return t.to(dtype).cuda()


def make_table(rng, lengths, page, pages, width=None):
    """Randomly placed distinct pages for every sequence, -1 elsewhere."""
    need = [-(-n // page) for n in lengths]
    ids = torch.randperm(pages, generator=rng)[:sum(need)].to(torch.int32)
    table = torch.full((len(lengths), width or max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table


def offsets(rows):
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def row_first(pool, layout):
    return pool if layout == "nhd" else pool.transpose(-3, -2)


def cached(pool, layout, table, b, n, page):
    """Positions 0..n-1 of sequence b as [n, heads, dim] on the host, in float64."""
    at = torch.arange(n)
    p = table[b].long()[at // page]
    return row_first(pool.cpu(), layout)[p, at % page].double()


def rotate(x, pos, inv_freq, interleaved):
    """x [heads, dim] at position pos; inv_freq a list of radians per position."""
    y = x.clone()
    half = len(inv_freq)
    for i, f in enumerate(inv_freq):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = math.cos(pos * f), math.sin(pos * f)
        y[:, a] = x[:, a] * c - x[:, b] * s
        y[:, b] = x[:, b] * c + x[:, a] * s
    return y


def norm(x, w, eps):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def attention(q, k, v, seen, scale):
    """q [n, H, D], k and v [len, K, D] float64, seen [n, len] bool: out [n, H, D], lse [n, H], and
    the largest sum of |q k| scale, for tolerances."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out, lse = torch.zeros(n, H, v.shape[2], dtype=torch.float64), torch.full((n, H), -math.inf, dtype=torch.float64)
    most = 0.0
    for h in range(H):
        for i in range(n):
            at = seen[i].nonzero()[:, 0]
            if not len(at):
                continue
            s = (k[at, h // G] @ q[i, h]) * scale
            most = max(most, float((k[at, h // G].abs() @ q[i, h].abs()).max()) * abs(scale))
            p = torch.exp(s - s.max())
            out[i, h] = (p / p.sum()) @ v[at, h // G]
            lse[i, h] = s.max() + torch.log(p.sum())
    return out, lse, most


def tree_seen(parents, ctx):
    """[n, ctx + n] bool of a tree given by parents: the context, the ancestors and itself."""
    n = len(parents)
    seen = torch.zeros(n, ctx + n, dtype=torch.bool)
    seen[:, :ctx] = True
    for i in range(n):
        a = i
        while a >= 0:
            seen[i, ctx + a] = True
            a = parents[a]
    return seen


def mask_words(rows, words):
    """int32 words [T, words] of a list of per-row node lists."""
    out = torch.zeros(len(rows), words, dtype=torch.int64)
    for r, nodes in enumerate(rows):
        for j in nodes:
            out[r, j // 32] |= 1 << (j % 32)
    return out.to(torch.int32)


def random_parents(rng, n):
    return [-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=rng)) for i in range(1, n)]


def commit(tokens, parents, picks):
    """The accepted path of one tree."""
    path = [0]
    while True:
        nxt = [i for i in range(path[-1] + 1, len(tokens))
               if parents[i] == path[-1] and tokens[i] == picks[path[-1]]]
        if not nxt:
            return path
        path.append(nxt[0])


def beam(logits, scores, k, finished=None, pad=0):
    """One group, in float64: [(value, beam, token)] best first, padded."""
    found = []
    for b in range(logits.shape[0]):
        x, s = logits[b].double(), float(scores[b])
        if math.isnan(s) or s == math.inf:
            continue
        if finished is not None and finished[b]:
            if s > -math.inf:
                found.append((s, b, pad))
            continue
        if s == -math.inf or torch.isnan(x).any() or (x == math.inf).any():
            continue
        total = torch.logsumexp(x, 0)
        value = s + (x - total)
        for t in torch.argsort(-x, stable=True)[:k].tolist():
            if x[t] > -math.inf:
                found.append((float(value[t]), b, t))
    found.sort(key=lambda c: (-c[0], c[1], c[2]))
    found = found[:k]
    return found + [(-math.inf, -1, -1)] * (k - len(found))
