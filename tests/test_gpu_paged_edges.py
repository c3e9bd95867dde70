"""The paged operators where their arithmetic or their rules are at the edge: small probabilities,
sums whose parts cancel, infinities that a row sees, rows past the arrays, many rows, many sequences.

Bounds of the attention's error are taken per output from sum_j p_j |v_j|, which is what a relative error
of the weights or of the sums acts on, so a lost share of the softmax shows.
"""
import math

import pytest
import torch

import paged_reference as ref
from paged_reference import EPS, TINY
from potpori_b200 import _lib
from potpori_b200._lib import PPError

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FAR = 1 << 20  # a host's bound on the lengths that sends more than 8 vectors a head to the tcgen05 kernel


def rng_of(seed):
    return torch.Generator().manual_seed(seed)


def make(rng, lengths, rows, page, heads, dim, dtype, bound=None):
    from potpori_b200.paged import PagedBatch, PagedCache

    pages = sum(-(-n // page) for n in lengths) + 2
    table = ref.make_table(rng, lengths, page, pages)
    k = ref.make_pool(rng, pages, page, heads, dim, dtype)
    v = ref.make_pool(rng, pages, page, heads, dim, dtype)
    batch = PagedBatch(table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), ref.offsets(rows).cuda(),
                       max_rows=max(rows), max_length=bound or max(lengths))
    return PagedCache(k, v), batch, table


def fill(pool, table, b, values):
    """Positions 0.. of sequence b take values [n, heads, dim]."""
    at = torch.arange(len(values), device="cuda")
    page = pool.shape[1]
    pool[table[b].cuda().long()[at // page], at % page] = values.to(pool.dtype).cuda()


def exact(q, k, v, seen, scale):
    """q [n, H, D], k and v [len, K, D], seen [n, len] or None (all), float64 on the device: out, lse, and
    what errors act on: sum p |v|, sum |v| / sum of exp(s - max) [n, H, D], the largest sum |q k| scale."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out, lse = torch.zeros(n, H, D, dtype=torch.float64, device="cuda"), torch.zeros(n, H, dtype=torch.float64, device="cuda")
    weight, floor, most = torch.zeros_like(out), torch.zeros_like(out), 0.0
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        s = q[:, h] @ kh.T * scale
        most = max(most, float((q[:, h].abs() @ kh.abs().T).max()) * abs(scale))
        if seen is not None:
            s = s.masked_fill(~seen, -math.inf)
        top = s.max(-1, keepdim=True).values
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        out[:, h], weight[:, h] = p @ vh / total, p @ vh.abs() / total
        floor[:, h] = vh.abs().sum(0) / total
        lse[:, h] = (top + torch.log(total))[:, 0]
    return out, lse, weight, floor, most


def bound_of(dtype, terms, dim, steps):
    """What an output may be off by. A score is an F32 sum of dim products, scaled and taken from the maximum
    (3 roundings of its magnitude), which moves a weight and its share; exponentials 2^-21; a weight's
    second 16-bit part leaves out 2^-16 of a BF16 weight, 2^-22 of an F16 one, but an F16 part has steps
    of 2^-24, half of which is 2^-38 where weights are taken at 2^13; `steps` additions one after the other
    each cut or round at 2^-23. Then the output's rounding."""
    out, _, weight, floor, most = terms
    rel = 2 * (dim + 3) * 2.0 ** -24 * most + 2.0 ** -20 + steps * 2.0 ** -23 + {F32: 0, BF16: 2.0 ** -16, F16: 2.0 ** -22}[dtype]
    return out.abs() * EPS[dtype] + TINY[dtype] + rel * weight + (2.0 ** -38 * floor if dtype == F16 else 0)


# (type, heads a cached head, host's bound): the F32, the narrow and the tcgen05 kernel. 12 vectors a head and
# FAR take the tcgen05 kernel, 1 vector the narrow one.
KERNELS = [(F32, 1, None), (BF16, 1, None), (F16, 1, None), (BF16, 12, FAR), (F16, 12, FAR)]


@pytest.mark.parametrize("dt,G,bound", KERNELS)
@pytest.mark.parametrize("sink_v", [0.0, 3.0])
@pytest.mark.parametrize("length", [200, 131072])
@pytest.mark.parametrize("spread", [0.0, 0.5])
def test_small_probabilities_count(gpu, dt, G, bound, sink_v, length, spread):
    """One key 17.5 nats above all the others, whose weights are 2^-25 of its own: they are what the
    output consists of where that key's V is zero."""
    rng = rng_of(50)
    cache, batch, table = make(rng, [length], [1], 64, 1, 64, dt, bound=bound)
    k = torch.zeros(length, 1, 64)
    k[:, 0, 0] = spread * torch.randn(length, generator=rng)
    k[5, 0, 0] = 17.5
    v = 256 + 32 * torch.randn(length, 1, 64, generator=rng)
    v[5] = sink_v
    fill(cache.k, table, 0, k)
    fill(cache.v, table, 0, v)
    q = torch.zeros(1, G, 64, dtype=dt, device="cuda")
    q[:, :, 0] = 1.0
    lse = torch.empty(1, G, device="cuda")
    got = cache.tree_attention(batch, q, scale=1.0, lse=lse)
    cache.check()
    terms = exact(q.double(), k.to(dt).double().cuda(), v.to(dt).double().cuda(), None, 1.0)
    # At 131072 the tiles of 64 (32) keys are cut over at least 148 CTAs: at most 14 (28) of them in a CTA, 8 additions
    # each (32 in the F32 kernel), and at most 740 partials; at 200 there are 4 (7).
    steps = (28 * 32 + 740) if length > 200 else 7 * 32
    off = (got.double() - terms[0]).abs()
    tol = bound_of(dt, terms, 1, steps)  # one product a score, the rest are zeros
    assert (off <= tol).all(), (float((off / tol).max()), float((off / terms[0].abs()).max()))
    assert ((lse.double() - terms[1]).abs() <= (steps + 64) * 2.0 ** -24 + 2.0 ** -20 + terms[1].abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("dt,G,bound", KERNELS)
@pytest.mark.parametrize("scale", [1.0, -1.0, 2.0 ** -4, 2.0 ** -10])
@pytest.mark.parametrize("step", [0.0, 1.0])
def test_scores_of_many_digits(gpu, dt, G, bound, scale, step):
    """Scores near 2^26, where F32 values are 4 or 8 apart, equal or rising with the position: outputs are means of
    V with weights of some kind, never infinite. Equal scores give the plain mean."""
    rng = rng_of(58)
    n = 300
    cache, batch, table = make(rng, [n], [1], 16, 1, 64, dt, bound=bound)
    k = torch.zeros(n, 1, 64)
    k[:, 0, 0], k[:, 0, 1] = 30720.0, step * torch.arange(n)
    v = 1 + torch.rand(n, 1, 64, generator=rng)
    fill(cache.k, table, 0, k)
    fill(cache.v, table, 0, v)
    q = torch.zeros(1, G, 64, dtype=dt, device="cuda")
    q[:, :, 0], q[:, :, 1] = 2048.0, 16.0
    lse = torch.empty(1, G, device="cuda")
    got = cache.tree_attention(batch, q, scale=scale, lse=lse).double()
    v = v.to(dt).double().cuda()
    slack = 2 * EPS[dt] + 2.0 ** -14
    assert (got >= v.min() * (1 - slack)).all() and (got <= v.max() * (1 + slack)).all() and torch.isfinite(lse).all()
    if step == 0:
        assert ((got[0] - v.mean(0)).abs() <= v.mean(0) * slack).all()


@pytest.mark.parametrize("dt,G,bound", KERNELS)
@pytest.mark.parametrize("dims", [64, 1])
def test_weights_whose_values_cancel(gpu, dt, G, bound, dims):
    """V alternates between +1000 and -1000 and neighbours have nearly equal scores, so that the output is
    a small difference of the weights: those must be good to far more than the output's type. With one
    dim of the queries in use the scores are exact and the bound is the weights' own: one rounded part of
    either 16-bit type would not meet it."""
    rng = rng_of(51)
    n = 70
    cache, batch, table = make(rng, [n], [1], 16, 1, 64, dt, bound=bound)
    q = torch.randn(1, G, 64, generator=rng).to(dt)
    q[..., dims:] = 0
    k = torch.randn(n // 2, 1, 64, generator=rng).repeat_interleave(2, 0) + 0.01 * torch.randn(n, 1, 64, generator=rng)
    v = torch.where(torch.arange(n)[:, None, None] % 2 == 0, 1000.0, -1000.0).expand(n, 1, 64)
    fill(cache.k, table, 0, k)
    fill(cache.v, table, 0, v)
    got = cache.tree_attention(batch, q.cuda())
    terms = exact(q.double().cuda(), k.to(dt).double().cuda(), v.to(dt).double().cuda(), None, 0.125)
    # Additions one after the other: F32 every key's of 3 tiles, else two for every 16 keys and the warps' four.
    off, tol = (got.double() - terms[0]).abs(), bound_of(dt, terms, dims, 3 * 32 if dt == F32 else 16)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("dt,G,bound", [(F32, 2, None), (BF16, 1, None), (F16, 1, None), (BF16, 8, FAR), (F16, 8, FAR)])
@pytest.mark.parametrize("length", [20000, 150])
def test_shares_of_a_split_cache(gpu, dt, G, bound, length):
    """V around 1: a share of the softmax that a split or a join lost or counted twice is a bias."""
    rng = rng_of(52)
    rows, lengths = [24, 3], [length, length // 3]
    cache, batch, table = make(rng, lengths, rows, 64, 1, 128, dt, bound=bound)
    parents = [ref.random_parents(rng, n) for n in rows]
    seen = [ref.tree_seen(p, lengths[b] - rows[b]) for b, p in enumerate(parents)]
    bits = [s[i, lengths[b] - rows[b]:].nonzero()[:, 0].tolist() for b, s in enumerate(seen) for i in range(rows[b])]
    q = torch.randn(27, G, 128, generator=rng).to(dt).cuda()
    ks = [torch.randn(n, 1, 128, generator=rng) for n in lengths]
    vs = [1 + 0.25 * torch.randn(n, 1, 128, generator=rng) for n in lengths]
    for b in range(2):
        fill(cache.k, table, b, ks[b])
        fill(cache.v, table, b, vs[b])
    got = cache.tree_attention(batch, q, mask=ref.mask_words(bits, 1).cuda())
    cache.check()
    t = 0
    for b, n in enumerate(rows):
        terms = exact(q[t:t + n].double(), ks[b].to(dt).double().cuda(), vs[b].to(dt).double().cuda(), seen[b].cuda(), 128 ** -0.5)
        # In a CTA: all tiles of a short cache, of a long one its share over at least 100 CTAs; then the partials.
        steps = 7 * 32 if length == 150 else 10 * 32 + 740
        off, tol = (got[t:t + n].double() - terms[0]).abs(), bound_of(dt, terms, 128, steps)
        assert (off <= tol).all(), (b, float((off / tol).max()))
        t += n


@pytest.mark.parametrize("dt,heads,bound", [(F32, 2, None), (BF16, 2, None), (F16, 2, None), (BF16, 16, FAR), (F16, 16, FAR)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("ctx", [0, 3000])
def test_seen_nonfinite_nodes(gpu, dt, heads, bound, bad, ctx):
    """A node's V that is not finite gives its own value to every row that sees the node, whichever
    keys the row sees beside it, and nothing to the others."""
    rng = rng_of(53)
    n = 40
    cache, batch, table = make(rng, [ctx + n], [n], 16, 2, 128, dt, bound=bound)
    q = torch.randn(n, heads, 128, generator=rng).to(dt).cuda()
    # Row i sees node i alone, the multiples of five node 21 too, and all of the context.
    bits = [[i] + ([21] if i % 5 == 0 else []) for i in range(n)]
    mask = ref.mask_words(bits, 2).cuda()
    want = cache.tree_attention(batch, q, mask=mask)
    p, at = int(table[0, (ctx + 21) // 16]), (ctx + 21) % 16
    cache.v[p, at, 0, 3:90:5] = bad
    got = cache.tree_attention(batch, q, mask=mask)
    sees = torch.tensor([21 in x for x in bits]).cuda()
    hit = torch.zeros(128, dtype=torch.bool, device="cuda")
    hit[3:90:5] = True
    first = heads // 2
    assert torch.equal(got[~sees], want[~sees]) and torch.equal(got[:, first:], want[:, first:])
    mine = got[sees][:, :first]
    assert torch.equal(mine[..., ~hit], want[sees][:, :first][..., ~hit])
    mine = mine[..., hit]
    assert torch.isnan(mine).all() if math.isnan(bad) else (mine == bad).all()


@pytest.mark.parametrize("dt,heads,bound", [(F32, 2, None), (BF16, 2, None), (F16, 2, None), (BF16, 16, FAR), (F16, 16, FAR)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("index", [0, 70, 3071, 3099])
@pytest.mark.parametrize("masked", [False, True])
def test_nonfinite_context(gpu, dt, heads, bound, bad, index, masked):
    """A V of the context that is not finite reaches every row, wherever its position lies: before the
    tree's first tile or in it, next to the first node."""
    rng = rng_of(59)
    n, ctx = 12, 3100
    cache, batch, table = make(rng, [ctx + n], [n], 16, 2, 128, dt, bound=bound)
    q = torch.randn(n, heads, 128, generator=rng).to(dt).cuda()
    mask = ref.mask_words([[i] for i in range(n)], 1).cuda() if masked else None
    want = cache.tree_attention(batch, q, mask=mask)
    p, at = int(table[0, index // 16]), index % 16
    cache.v[p, at, 0, 3:90:5] = bad
    got = cache.tree_attention(batch, q, mask=mask)
    hit = torch.zeros(128, dtype=torch.bool, device="cuda")
    hit[3:90:5] = True
    first = heads // 2
    assert torch.equal(got[:, first:], want[:, first:]) and torch.equal(got[:, :first][..., ~hit], want[:, :first][..., ~hit])
    mine = got[:, :first][..., hit]
    assert (torch.isnan(mine) if math.isnan(bad) else torch.isnan(mine) | (mine == bad)).all()


@pytest.mark.parametrize("vector", [True, False])
def test_append_rows_past_the_arrays(gpu, vector):
    """cu_rows that reaches past the row arrays, or before them, and lengths that do not fit: append leaves
    the sequence out whole, its rows of q_out too, and marks it; the others are written."""
    from potpori_b200.paged import PagedBatch

    rng = rng_of(54)
    cache, batch, table = make(rng, [40, 40, 40], [2, 2, 2], 16, 2, 64, BF16)
    wide = torch.randn(6, 4 + 2, 64 + (0 if vector else 1), generator=rng).bfloat16().cuda()
    rows = [wide.flatten(1)[:, a:a + h * 64].unflatten(1, (h, 64)) for a, h in ((0, 2), (128, 2), (256, 2))]
    q, k, v = rows
    freq = (1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).cuda()
    before = cache.k.clone(), cache.v.clone()
    whole = cache.append(batch, k, v, q=q, inv_freq=freq)
    cache.check()
    after = cache.k.clone(), cache.v.clone()
    cases = [([0, 2, 4, 8], [40, 40, 40], 2), ([0, 2, 4, 2 ** 31 - 1], [40, 40, 40], 2), ([-2, 2, 4, 6], [40, 40, 40], 0),
             ([0, 2, 4, 6], [40, 1, 40], 1), ([0, 2, 4, 6], [40, 49, 40], 1), ([0, 2, 4, 6], [40, -3, 40], 1)]
    for cu, lengths, left in cases:
        cache.k.copy_(before[0])
        cache.v.copy_(before[1])
        b = PagedBatch(batch.page_table, torch.tensor(lengths, dtype=torch.int32).cuda(),
                       torch.tensor(cu, dtype=torch.int32).cuda(), 8, 40)
        out = torch.full((6, 2, 64), 7.0, dtype=BF16, device="cuda")
        cache.append(b, k, v, q=q, inv_freq=freq, out=out)
        with pytest.raises(PPError):
            cache.check()
        for pool, old, new in ((cache.k, before[0], after[0]), (cache.v, before[1], after[1])):
            for s in range(3):
                pages = table[s].long().cuda()
                assert torch.equal(pool[pages], (old if s == left else new)[pages]), (cu, lengths, s)
        for s in range(3):
            rows_of = slice(2 * s, 2 * s + 2)
            assert (out[rows_of] == 7.0).all() if s == left else torch.equal(out[rows_of], whole[rows_of]), (cu, lengths, s)


def test_check_tells_beams_from_pages(gpu):
    """The error word that beam_select shares with a cache: a beam left out is not reported as a bad page."""
    from potpori_b200.paged import PagedBatch, beam_select

    rng = rng_of(55)
    cache, batch, table = make(rng, [20], [2], 16, 2, 64, BF16)
    logits = torch.zeros(1, 2, 100, device="cuda")
    logits[0, 1, 7] = math.nan
    scores = torch.zeros(1, 2, device="cuda")
    beam_select(logits, scores, 2, err=cache.err)
    with pytest.raises(PPError) as e:
        cache.check()
    assert e.value.status == _lib.PP_E_NONFINITE and "beam" in str(e.value) and "page" not in str(e.value)
    cache.check()
    k = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    cache.append(PagedBatch(torch.full_like(batch.page_table, -1), batch.lengths, batch.cu_rows, 2, 20), k, k)
    beam_select(logits, scores, 2, err=cache.err)
    with pytest.raises(PPError) as e:
        cache.check()
    assert e.value.status == _lib.PP_E_INVALID and "beam" in str(e.value) and "page" in str(e.value)
    cache.check()


def test_shard_refuses_f16_parameters(gpu):
    """PP_F16 is the paged operators' alone: a shard's loader knows F32 and BF16."""
    import ctypes

    import numpy as np

    from potpori_b200.config import QwenConfig
    from potpori_b200.shard import Shard

    cfg = QwenConfig(layers=2, hidden=256, intermediate=512, head_dim=128, n_heads=4, n_kv_heads=2, vocab_size=64,
                     rms_norm_eps=1e-6, rope_theta=1e6)
    shard = Shard(cfg, (0, 2), 8, 2)
    name = b"model.layers.0.mlp.gate_proj.weight"
    data = np.zeros(512 * 256, np.uint16)
    L, p = _lib.load(), data.ctypes.data_as(ctypes.c_void_p)
    for dtype in (_lib.PP_F16, 3):
        assert L.pp_shard_set_tensor(shard.handle, name, dtype, p, data.size) == _lib.PP_E_INVALID
        assert "parameters are PP_F32 or PP_BF16" in _lib.last_error(shard.handle)
    assert L.pp_shard_set_tensor(shard.handle, name, _lib.PP_BF16, p, data.size) == _lib.PP_OK


@pytest.mark.parametrize("dt,G,bound", [(F32, 2, None), (BF16, 1, None), (BF16, 4, FAR), (F16, 2, FAR)])
@pytest.mark.parametrize("rows,lengths", [([300], [300]), ([300, 77], [700, 1100]), ([520], [3000]), ([1], [9])])
def test_prompt_rows(gpu, dt, G, bound, rows, lengths):
    """A chain of many rows, with and without context, alone and beside others."""
    rng = rng_of(56)
    cache, batch, table = make(rng, lengths, rows, 16, 2, 64, dt, bound=bound)
    T = sum(rows)
    q = torch.randn(T, 2 * G, 64, generator=rng).to(dt).cuda()
    got = cache.tree_attention(batch, q, lse=(lse := torch.empty(T, 2 * G, device="cuda")))
    cache.check()
    t = 0
    for b, n in enumerate(rows):
        k, v = (ref.cached(p, "nhd", table, b, lengths[b], 16).cuda() for p in (cache.k, cache.v))
        seen = torch.ones(n, lengths[b], dtype=torch.bool, device="cuda").tril(lengths[b] - n)
        terms = exact(q[t:t + n].double(), k, v, seen, 0.125)
        steps = -(-lengths[b] // 16) * 16 + 740  # no more than every key's, however it is cut
        off, tol = (got[t:t + n].double() - terms[0]).abs(), bound_of(dt, terms, 64, steps)
        assert (off <= tol).all(), (b, float((off / tol).max()))
        assert ((lse[t:t + n].double() - terms[1]).abs() <= (steps + 2 * 64 * terms[4]) * 2.0 ** -24 + 2.0 ** -20 + terms[1].abs() * 2.0 ** -22).all()
        t += n


@pytest.mark.parametrize("sequences", [70, 210])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_sequences_of_many_vectors(gpu, sequences, dim):
    """The tcgen05 kernel with more sequences than a line is put in order for, and with more than the shared
    memory of two CTAs on an SM has room for."""
    rng = rng_of(57)
    rows = [int(torch.randint(0, 6, (1,), generator=rng)) for _ in range(sequences)]
    lengths = [n + int(torch.randint(0, 260, (1,), generator=rng)) for n in rows]
    cache, batch, table = make(rng, lengths, rows, 16, 1, dim, BF16, bound=FAR)
    T = sum(rows)
    parents = [ref.random_parents(rng, n) if n else [] for n in rows]
    seen = [ref.tree_seen(p, lengths[b] - rows[b]) for b, p in enumerate(parents)]
    bits = [s[i, lengths[b] - rows[b]:].nonzero()[:, 0].tolist() for b, s in enumerate(seen) for i in range(rows[b])]
    q = torch.randn(T, 12, dim, generator=rng).bfloat16().cuda()
    mask = ref.mask_words(bits, 1).cuda()
    got = cache.tree_attention(batch, q, mask=mask)
    cache.check()
    pools = cache.k.cpu().double(), cache.v.cpu().double()
    t = 0
    for b, n in enumerate(rows):
        if n:
            k, v = (ref.cached(p, "nhd", table, b, lengths[b], 16).cuda() for p in pools)
            terms = exact(q[t:t + n].double(), k, v, seen[b].cuda(), dim ** -0.5)
            off, tol = (got[t:t + n].double() - terms[0]).abs(), bound_of(BF16, terms, dim, 9 * 16 + 8)
            assert (off <= tol).all(), (b, float((off / tol).max()))
        t += n
    assert torch.equal(cache.tree_attention(batch, q, mask=mask), got)
