"""The serving operators over a paged K/V cache, case by case: appending rotated rows, the
attention of a tree of drafted tokens, the commit of the accepted path, and a beam step.

``run`` computes a case either in its plain form (elementary torch operations in 32 bits, in
64 where a far position's angle or the order of two candidates needs it) or, with ``own``
set, by the calls a user makes of ``potpori_b200.paged``. ``exact`` gives the same outputs
from the definitions in 64 bits.

Notation: B sequences, sequence b with rows[b] new rows (the nodes of its draft tree, or one
decoded token) that are the last rows[b] of its lengths[b] cached positions; pages of P
positions; H query heads over K cached heads of D dimensions.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
VOCAB = 151936


def listed():
    return [
        # One decoded token of the 0.6B geometry: the smallest append, all latency.
        {"name": "append 1 row", "op": "append", "batch": 1, "rows": 1, "length": 42, "heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "f32", "cache": "bf16", "layout": "nhd",
         "norm": True, "interleaved": False, "rotary": 128, "tree": False},
        # Draft trees of a batch, another rotation order and an odd page, positions by depth.
        {"name": "append trees 48x13", "op": "append", "batch": 48, "rows": 13, "length": 1031,
         "heads": 24, "kv_heads": 6, "dim": 64, "page": 24, "type": "f16", "cache": "f16",
         "layout": "hnd", "norm": False, "interleaved": True, "rotary": 32, "tree": True},
        # Four 2048-token prompts of the 4B geometry, F32 projections into a BF16 cache.
        {"name": "append prompts 4x2048", "op": "append", "batch": 4, "rows": 2048, "length": 2048,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "type": "f32", "cache": "bf16",
         "layout": "nhd", "norm": True, "interleaved": False, "rotary": 128, "tree": False},
        # The first token after a short prompt, F32 cache: all latency.
        {"name": "attend 1 row len 42 f32", "op": "attend", "batch": 1, "rows": 1, "length": 42,
         "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "cache": "f32", "layout": "nhd",
         "tree": False},
        # The verify chunk of the 4B workload (gamma + 1 = 8) after its 2048-token prompt.
        {"name": "attend chunk 8 len 2056", "op": "attend", "batch": 1, "rows": 8, "length": 2056,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16", "layout": "nhd",
         "tree": True},
        # Decode of a ragged batch: the cache is read once, HBM-bound.
        {"name": "attend 64x1 len 8192", "op": "attend", "batch": 64, "rows": 1, "length": 8192,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16", "layout": "nhd",
         "tree": False},
        # Wide trees over a batch: 244 query vectors share a cached head, compute counts.
        {"name": "attend trees 16x61 len 4096", "op": "attend", "batch": 16, "rows": 61,
         "length": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "cache": "f16",
         "layout": "hnd", "tree": True},
        # One long document with a tree: the cache split over the whole card.
        {"name": "attend tree 24 len 131072", "op": "attend", "batch": 1, "rows": 24,
         "length": 131072, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "cache": "bf16",
         "layout": "nhd", "tree": True},
        # The accepted path of one tree, 28 layers of the 0.6B geometry.
        {"name": "commit 8 nodes 28 layers", "op": "commit", "batch": 1, "rows": 8, "length": 49,
         "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16", "layout": "nhd", "layers": 28,
         "accept": 4},
        # A batch of trees, 36 layers of the 4B geometry.
        {"name": "commit 64x31 36 layers", "op": "commit", "batch": 64, "rows": 31, "length": 100,
         "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16", "layout": "hnd", "layers": 36,
         "accept": 9},
        # One prompt decoded with four beams.
        {"name": "beam 1x4 bf16", "op": "beam", "batch": 1, "beams": 4, "vocab": VOCAB,
         "type": "bf16", "length": 41, "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16",
         "layout": "nhd", "layers": 28},
        # A batch with eight beams each: the logits are read once.
        {"name": "beam 32x8 f32", "op": "beam", "batch": 32, "beams": 8, "vocab": VOCAB,
         "type": "f32", "length": 41, "kv_heads": 8, "dim": 128, "page": 16, "cache": "bf16",
         "layout": "nhd", "layers": 36},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "commit", "beam"])
    cache = rng.choice(["bf16", "bf16", "f16", "f32"])
    c = {"op": op, "cache": cache, "layout": rng.choice(["nhd", "hnd"]),
         "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128]), "dim": rng.choice([64, 80, 128, 128, 256]),
         "kv_heads": rng.choice([1, 2, 4, 5, 8])}
    if op == "append":
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 7])
        c["batch"] = _log_int(rng, 1, 64)
        c["rows"] = _log_int(rng, 1, max(1, 4096 // c["batch"]))
        c["length"] = c["rows"] + _log_int(rng, 1, 4096)
        c["type"] = rng.choice(["f32", c["cache"]])
        c["norm"] = rng.random() < 0.5
        c["interleaved"] = rng.random() < 0.3
        c["rotary"] = rng.choice([c["dim"], c["dim"] // 2])
        c["tree"] = rng.random() < 0.5
    elif op == "attend":
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 7, 8])
        c["batch"] = _log_int(rng, 1, 48)
        c["rows"] = _log_int(rng, 1, 64)
        # The scores are no more than those of the largest listed tree, the cache no more than
        # that of the listed batch.
        top = min(262144 // c["batch"], 12000000000 // (c["batch"] * c["rows"] * c["heads"] * c["dim"]))
        if c["dim"] > 128 or cache == "f32":
            top //= 4
        c["length"] = c["rows"] + _log_int(rng, 1, max(2, min(65536, top)))
        c["tree"] = c["rows"] > 1 and rng.random() < 0.8
    elif op == "commit":
        c["batch"] = _log_int(rng, 1, 64)
        c["rows"] = _log_int(rng, 2, 64)
        c["length"] = c["rows"] + _log_int(rng, 1, 100)
        c["layers"] = rng.choice([1, 7, 28])
        c["accept"] = rng.randint(0, 10)
    else:
        c["batch"] = _log_int(rng, 1, 24)
        c["beams"] = _log_int(rng, 1, 8)
        c["vocab"] = _log_int(rng, 1000, VOCAB)
        c["type"] = rng.choice(["f32", "bf16", "f16"])
        c["length"] = _log_int(rng, 1, 90)
        c["layers"] = rng.choice([1, 7, 28])
        c["dim"] = min(c["dim"], 128)
    return c


# ---- the shape of a case: lengths, rows and trees follow from the case alone ----------------


def _lengths(c):
    """Ragged lengths: the first is the longest, the others down to about half of it."""
    n, lo = c["length"], c.get("rows", 1)
    return [max(lo, n - (b * 7919) % max(1, n // 2)) for b in range(c["batch"] * c.get("beams", 1))]


def _rows(c):
    if c["rows"] > 256:
        return [max(1, c["rows"] - (b * 641) % max(1, c["rows"] // 2)) for b in range(c["batch"])]
    return [c["rows"] if not b % 3 else max(1, c["rows"] - b % 5) for b in range(c["batch"])]


def _parents(c, b, n):
    """A draft tree: node 0 is the current token, every other node hangs on one of the few
    nodes before it."""
    if not c.get("tree", True):
        return [i - 1 for i in range(n)]
    r = random.Random(1000 * b + n)
    return [-1] + [r.randint(max(0, i - 5), i - 1) for i in range(1, n)]


def _path(parents, depth):
    """The path that the targets' picks will take: the last child each time."""
    path = [0]
    while len(path) <= depth:
        below = [i for i in range(len(parents)) if parents[i] == path[-1]]
        if not below:
            break
        path.append(below[-1])
    return path


def _accept(c, b):
    return max(0, c["accept"] - b % 4)


def _element(t):
    return 4 if t == "f32" else 2


def work(c):
    e = _element(c["cache"])
    if c["op"] == "append":
        t = sum(_rows(c))
        n = t * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": n * (_element(c["type"]) + e), "flops": 6 * n}
    if c["op"] == "attend":
        rows, lens = _rows(c), _lengths(c)
        cached = 2 * sum(lens) * c["kv_heads"] * c["dim"] * e
        flops = sum(4 * r * n * c["heads"] * c["dim"] for r, n in zip(rows, lens))
        return {"bytes": cached + 2 * sum(rows) * c["heads"] * c["dim"] * e, "flops": flops}
    row = c["kv_heads"] * c["dim"] * e * 2 * c["layers"]
    if c["op"] == "commit":
        moved = sum(sum(k != p for k, p in enumerate(_path(_parents(c, b, n), _accept(c, b))))
                    for b, n in enumerate(_rows(c)))
        return {"bytes": 2 * moved * row + 16 * sum(_rows(c)), "flops": 0}
    n = c["batch"] * c["beams"] * c["vocab"]
    part = sum(n % c["page"] for n in _lengths(c)) * (c["beams"] - 1) / c["beams"] / 2
    return {"bytes": n * _element(c["type"]) + 2 * part * row, "flops": 4 * n}


# ---- inputs ---------------------------------------------------------------------------------


def _table(c, lens, extra, gen):
    """Page table of the sequences over randomly placed pages, unused entries -1, and `extra`
    more pages."""
    P = c["page"]
    need = [-(-n // P) for n in lens]
    ids = torch.randperm(sum(need) + extra, generator=gen)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, ids[at:], sum(need) + extra


def _pool(c, pages, gen, layers=0):
    shape = ((pages, c["page"], c["kv_heads"], c["dim"]) if c["layout"] == "nhd" else
             (pages, c["kv_heads"], c["page"], c["dim"]))
    shape = (layers,) + shape if layers else shape
    out = torch.empty(shape, dtype=TYPES[c["cache"]], device="cuda")
    return out.normal_(generator=gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = dict(case)
    cpu = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lengths(c)
    s = {"case": c}
    extra = c["batch"] * c["beams"] if c["op"] == "beam" else 2
    table, spare, pages = _table(c, lens, extra, cpu)
    s["table"], s["lengths"] = table.cuda(), _ints(lens)
    layers = c.get("layers", 0)
    s["k"], s["v"] = _pool(c, pages, gen, layers), _pool(c, pages, gen, layers)
    s["max_length"] = max(lens)
    if c["op"] == "beam":
        B, W = c["batch"], c["beams"]
        s["spare"] = spare.to(torch.int32).cuda().reshape(B, W)
        s["table"], s["lengths"] = s["table"].reshape(B, W, -1), s["lengths"].reshape(B, W)
        s["logits"] = (torch.empty(B, W, c["vocab"], device="cuda").normal_(generator=gen) * 3).to(TYPES[c["type"]])
        s["scores"] = -20 + 2 * torch.empty(B, W, device="cuda").normal_(generator=gen)
        return s
    rows = _rows(c)
    trees = [_parents(c, b, n) for b, n in enumerate(rows)]
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    T = cu[-1]
    s["cu_rows"], s["max_rows"] = _ints(cu), max(rows)
    if c["op"] == "commit":
        tokens = torch.randint(0, VOCAB, (T,), generator=cpu)
        picks = torch.randint(0, VOCAB, (T,), generator=cpu)
        for b, tree in enumerate(trees):
            path = _path(tree, _accept(c, b))
            for a, d in zip(path, path[1:]):
                picks[cu[b] + a] = tokens[cu[b] + d]
        s["tokens"], s["picks"] = tokens.to(torch.int32).cuda(), picks.to(torch.int32).cuda()
        s["parents"] = _ints([p for t in trees for p in t])
        return s
    if c["op"] == "append":
        H, K, D = c["heads"], c["kv_heads"], c["dim"]
        qkv = torch.empty(T, (H + 2 * K) * D, device="cuda").normal_(generator=gen).to(TYPES[c["type"]])
        # The three parts of a fused projection's rows.
        s["q"] = qkv[:, :H * D].unflatten(1, (H, D))
        s["k_new"] = qkv[:, H * D:(H + K) * D].unflatten(1, (K, D))
        s["v_new"] = qkv[:, (H + K) * D:].unflatten(1, (K, D))
        r = c["rotary"]
        s["inv_freq"] = 1e6 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
        s["q_norm"] = s["k_norm"] = s["positions"] = None
        if c["norm"]:
            s["q_norm"] = 1 + 0.1 * torch.empty(D, device="cuda").normal_(generator=gen)
            s["k_norm"] = 1 + 0.1 * torch.empty(D, device="cuda").normal_(generator=gen)
        if c["tree"]:
            pos = []
            for b, tree in enumerate(trees):
                depth = []
                for p in tree:
                    depth.append(depth[p] + 1 if p >= 0 else 0)
                pos += [lens[b] - rows[b] + d for d in depth]
            s["positions"] = _ints(pos)
        return s
    s["q"] = (2 * torch.empty(T, c["heads"], c["dim"], device="cuda").normal_(generator=gen)).to(TYPES[c["cache"]])
    s["mask"] = None
    if c["tree"]:
        words = -(-max(rows) // 32)
        mask = []
        for tree in trees:
            seen = []
            for i, p in enumerate(tree):
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
                mask.append([(seen[i] >> 32 * w) & 0xFFFFFFFF for w in range(words)])
        s["mask"] = torch.tensor(mask, dtype=torch.int64).to(torch.int32).cuda()
    return s


# ---- one pass -------------------------------------------------------------------------------


def run(s):
    return _run_own(s) if own else PLAIN[s["case"]["op"]](s)


def _run_own(s):
    from potpori_b200.paged import PagedBatch, PagedCache, beam_select
    c = s["case"]
    if "cache" not in s:  # the handles that a user's program keeps: pointers and strides only
        s["cache"] = PagedCache(s["k"], s["v"], layout=c["layout"])
        if c["op"] != "beam":
            s["batch"] = PagedBatch(s["table"], s["lengths"], s["cu_rows"], max_rows=s["max_rows"],
                                    max_length=s["max_length"])
    cache = s["cache"]
    if c["op"] == "append":
        q = cache.append(s["batch"], s["k_new"], s["v_new"], q=s["q"], inv_freq=s["inv_freq"],
                         positions=s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
                         interleaved=c["interleaved"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["op"] == "attend":
        return {"out": cache.tree_attention(s["batch"], s["q"], mask=s["mask"])}
    if c["op"] == "commit":
        path, accepted, correction, lengths = cache.tree_commit(s["batch"], s["tokens"], s["parents"], s["picks"])
        return {"path": path, "accepted": accepted, "correction": correction, "lengths": lengths,
                "k": s["k"], "v": s["v"]}
    scores, beams, tokens = beam_select(s["logits"], s["scores"], c["beams"])
    table, lengths, taken = cache.beam_reorder(s["table"], s["lengths"], beams, s["spare"])
    return {"scores": scores, "beams": beams, "tokens": tokens, "table": table, "lengths": lengths,
            "taken": taken, "k": s["k"], "v": s["v"]}


def _positions_first(pool, layout):
    """The pool as [(layers,) pages, positions, heads, dims]."""
    return pool if layout == "nhd" else pool.transpose(-3, -2)


def _row_places(s):
    """Sequence, row inside it, and cache index of every new row."""
    cu, lens = s["cu_rows"].long(), s["lengths"].long()
    t = torch.arange(_total(s), device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    i = t - cu[seq]
    return seq, i, lens[seq] - (cu[seq + 1] - cu[seq]) + i


def _total(s):
    return next(s[n].shape[0] for n in ("q", "tokens") if n in s)


def _plain_append(s):
    c = s["case"]
    P, r = c["page"], c["rotary"]
    seq, _, index = _row_places(s)
    pos = index if s["positions"] is None else s["positions"].long()
    angle = pos.double()[:, None] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        if c["interleaved"]:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = x[..., :r // 2], x[..., r // 2:r]
            y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((y, x[..., r:]), -1).to(s["k"].dtype)

    page, at = s["table"].long()[seq, index // P], index % P
    _positions_first(s["k"], c["layout"])[page, at] = rotated(s["k_new"], s["k_norm"])
    _positions_first(s["v"], c["layout"])[page, at] = s["v_new"].to(s["v"].dtype)
    return {"q": rotated(s["q"], s["q_norm"]), "k": s["k"], "v": s["v"]}


def _plain_attend(s):
    c = s["case"]
    B, n, K, D, P = c["batch"], s["max_rows"], c["kv_heads"], c["dim"], c["page"]
    G = c["heads"] // K
    seq, i, _ = _row_places(s)
    lens = s["lengths"].long()
    rows = s["cu_rows"].long().diff()
    j = torch.arange(s["max_length"], device=lens.device)
    page = s["table"].long()[:, j // P].clamp(min=0)
    k = _positions_first(s["k"], c["layout"])[page, j % P].float()
    v = _positions_first(s["v"], c["layout"])[page, j % P].float()
    q = torch.zeros(B, n, K, G, D, device=lens.device)
    q[seq, i] = s["q"].float().unflatten(1, (K, G))
    node = j - (lens - rows)[:, None]  # [B, L]: negative for the context
    drafted = (node >= 0) & (node < rows[:, None])
    if s["mask"] is None:
        seen = node[:, None] <= torch.arange(n, device=lens.device)[:, None]
    else:
        mask = torch.zeros(B, n, s["mask"].shape[1], dtype=torch.int32, device=lens.device)
        mask[seq, i] = s["mask"]
        at = node.clamp(0, 32 * mask.shape[2] - 1)
        word = mask.gather(2, (at // 32)[:, None].expand(B, n, -1))
        seen = (word >> (at % 32)[:, None].int() & 1) != 0
    seen = (node < 0)[:, None] | drafted[:, None] & seen
    score = torch.einsum("bnkgd,blkd->bkgnl", q, k) * (1 / math.sqrt(D))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("bkgnl,blkd->bnkgd", p, v) / total.movedim(3, 1)
    out = torch.where(total.movedim(3, 1) > 0, out, 0.0)
    return {"out": out[seq, i].flatten(1, 2).to(s["q"].dtype)}


def _plain_commit(s):
    c = s["case"]
    B, n, P = c["batch"], s["max_rows"], c["page"]
    seq, i, _ = _row_places(s)
    lens, rows = s["lengths"].long(), s["cu_rows"].long().diff()
    parent = torch.full((B, n), -1, device=lens.device)
    token, pick = parent.clone(), parent.clone()
    parent[seq, i], token[seq, i], pick[seq, i] = s["parents"].long(), s["tokens"].long(), s["picks"].long()
    node = torch.arange(n, device=lens.device)
    # A node follows when it is the first child of its parent that carries the parent's pick.
    match = (parent >= 0) & (token == pick.gather(1, parent.clamp(min=0)))
    twin = match[:, None] & (parent[:, None] == parent[..., None]) & (node[None] < node[:, None])
    follows = (match & ~twin.any(-1)) | (node == 0)
    # Ancestors of every node, itself among them, by squaring: paths up to 64 long.
    reach = torch.eye(n, device=lens.device) + (parent[..., None] == node)
    reach = torch.bmm(reach, reach).clamp(max=1)
    reach = torch.bmm(reach, reach).clamp(max=1)
    reach = torch.bmm(reach, reach).clamp(max=1)
    reach = torch.bmm(reach, reach).clamp(max=1)
    reach = torch.bmm(reach, reach).clamp(max=1)
    reach = torch.bmm(reach, reach).clamp(max=1) > 0
    taken = (follows[:, None] | ~reach).all(-1) & reach[..., 0]
    count = taken.sum(-1)
    order = torch.where(taken, node, n + node).sort(-1).values
    path = torch.where(node < count[:, None], order, -1)
    correction = pick.gather(1, path.gather(1, (count - 1)[:, None]))[:, 0]
    # Row path[d] of the tree goes to the d-th position after the context.
    base = (lens - rows)[:, None]
    live = path >= 0
    src, dst = (base + path.clamp(min=0))[live], (base + node)[live]
    b = torch.arange(B, device=lens.device)[:, None].expand(B, n)[live]
    table = s["table"].long()
    for_src, for_dst = (table[b, src // P], src % P), (table[b, dst // P], dst % P)
    k, v = _positions_first(s["k"], c["layout"]), _positions_first(s["v"], c["layout"])
    k[:, for_dst[0], for_dst[1]] = k[:, for_src[0], for_src[1]]
    v[:, for_dst[0], for_dst[1]] = v[:, for_src[0], for_src[1]]
    return {"path": path.int(), "accepted": (count - 1).int(), "correction": correction.int(),
            "lengths": (lens - rows + count).int(), "k": s["k"], "v": s["v"]}


def _plain_beam(s):
    c = s["case"]
    B, W, V, P = c["batch"], c["beams"], c["vocab"], c["page"]
    logits = s["logits"].float()
    # The best W of every beam by (logit, lowest token): one integer key holds both.
    bits = logits.view(torch.int32).long()
    rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = (rank << 32) + (2**32 - 1 - torch.arange(V, device=logits.device))
    token = 2**32 - 1 - (key.topk(W, -1).values & (2**32 - 1))
    top = logits.amax(-1, keepdim=True).double()
    total = top + (logits.double() - top).exp().sum(-1, keepdim=True).log()
    value = s["scores"].double()[..., None] + (logits.gather(-1, token).double() - total)
    value, at = value.flatten(1).sort(stable=True, dim=-1, descending=True)
    value, at = value[:, :W], at[:, :W]
    beam, token = at // W, token.flatten(1).gather(1, at)
    # States: the parent's pages; its last page, when only part full, stays with the first
    # child and is copied into the spare page of every other.
    table = s["table"].gather(1, beam[..., None].expand(-1, -1, s["table"].shape[2]))
    lengths = s["lengths"].gather(1, beam)
    order = torch.arange(W, device=beam.device)
    again = ((beam[:, None] == beam[..., None]) & (order < order[:, None])).any(-1)
    taken = again & (lengths % P > 0)
    last = (lengths // P).long().clamp(max=table.shape[2] - 1)
    source = table.gather(2, last[..., None])[..., 0]
    table = table.scatter(2, last[..., None], torch.where(taken, s["spare"], source)[..., None])
    inside = torch.arange(P, device=beam.device) < (lengths % P)[..., None]
    b, w, at = (inside & taken[..., None]).nonzero(as_tuple=True)
    src, dst = source[b, w].long(), s["spare"][b, w].long()
    k, v = _positions_first(s["k"], c["layout"]), _positions_first(s["v"], c["layout"])
    k[:, dst, at] = k[:, src, at]
    v[:, dst, at] = v[:, src, at]
    return {"scores": value.float(), "beams": beam.int(), "tokens": token.int(), "table": table,
            "lengths": lengths, "taken": taken.int(), "k": s["k"], "v": s["v"]}


PLAIN = {"append": _plain_append, "attend": _plain_attend, "commit": _plain_commit, "beam": _plain_beam}


# ---- the definitions in 64 bits -------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "commit":
        return None  # moves rows and counts: nothing is computed
    if c["op"] == "beam":
        out = torch.empty(c["batch"], c["beams"], dtype=torch.float64)
        for b in range(c["batch"]):
            logp = torch.log_softmax(s["logits"][b].double(), -1) + s["scores"][b].double()[:, None]
            out[b] = logp.flatten().topk(c["beams"]).values.cpu()
        return {"scores": out, "beams": None, "tokens": None, "table": None, "lengths": None,
                "taken": None, "k": None, "v": None}
    lens, rows, P = _lengths(c), _rows(c), c["page"]
    starts = [sum(rows[:b]) for b in range(len(rows))]
    heads_last = c["layout"] == "hnd"
    if c["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        k, v = (k.permute(0, 2, 1, 3).contiguous(), v.permute(0, 2, 1, 3).contiguous()) if heads_last else (k, v)
        flat_k, flat_v = k.view(-1, *k.shape[2:]), v.view(-1, *v.shape[2:])
        q_all = torch.empty(sum(rows), c["heads"], c["dim"], dtype=torch.float64, device="cuda")
        half = c["rotary"] // 2
        for b, n in enumerate(rows):
            sl = slice(starts[b], starts[b] + n)
            at = torch.arange(lens[b] - n, lens[b], device="cuda")
            pos = at if s["positions"] is None else s["positions"][sl]
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                               pos.double()[:, None, None] * s["inv_freq"])

            def turned(x, w):
                x = x[sl].double()
                if w is not None:
                    x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
                x = x.clone()
                first = slice(0, 2 * half, 2) if c["interleaved"] else slice(0, half)
                second = slice(1, 2 * half, 2) if c["interleaved"] else slice(half, 2 * half)
                z = torch.complex(x[..., first], x[..., second]) * turn
                x[..., first], x[..., second] = z.real, z.imag
                return x

            slot = s["table"][b].long()[at // P] * P + at % P
            flat_k[slot], flat_v[slot] = turned(s["k_new"], s["k_norm"]), s["v_new"][sl].double()
            q_all[sl] = turned(s["q"], s["q_norm"])
        back = (lambda x: x.permute(0, 2, 1, 3)) if heads_last else (lambda x: x)
        return {"q": q_all, "k": back(k), "v": back(v)}
    out = torch.empty(sum(rows), c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    G = c["heads"] // c["kv_heads"]
    for b, n in enumerate(rows):
        at = torch.arange(lens[b], device="cuda")
        page = s["table"][b].long()[at // P]
        tree = _parents(c, b, n)
        hidden = torch.zeros(n, lens[b], dtype=torch.bool)
        hidden[:, lens[b] - n:] = True
        for i in range(n):
            a = i
            while a >= 0:
                hidden[i, lens[b] - n + a] = False
                a = tree[a]
        hidden = hidden.cuda()
        for h in range(c["kv_heads"]):
            k = (s["k"][page, h, at % P] if heads_last else s["k"][page, at % P, h]).double()
            v = (s["v"][page, h, at % P] if heads_last else s["v"][page, at % P, h]).double()
            q = s["q"][starts[b]:starts[b] + n, h * G:(h + 1) * G].double()
            w = torch.matmul(q, k.T) / math.sqrt(c["dim"])
            w = torch.softmax(w.masked_fill(hidden[:, None], -math.inf), -1)
            out[starts[b]:starts[b] + n, h * G:(h + 1) * G] = torch.matmul(w, v)
    return {"out": out}
