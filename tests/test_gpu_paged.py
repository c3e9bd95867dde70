"""The paged operators on the device against their definitions in float64 (paged_reference.py).

Tolerances are sums of what the arithmetic may round. A result of type T is off by at most half a
step of T (EPS) of its value; F32 work before that is bounded where it is used. What only moves or
compares is equal.
"""
import math

import pytest
import torch

import paged_reference as ref
from paged_reference import EPS, TINY
from potpori_b200._lib import PPError

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rng_of(seed):
    return torch.Generator().manual_seed(seed)


# The host's bound on the lengths chooses the kernel for 16-bit caches: the true one leaves these small
# calls to the narrow kernel, a far one sends more than 8 query vectors a head to the tcgen05 kernel.
FAR = 1 << 20


def make(rng, lengths, rows, page, heads, dim, dtype, layout="nhd", layers=0, spare=0, bound=None):
    from potpori_b200.paged import PagedBatch, PagedCache

    pages = sum(-(-n // page) for n in lengths) + 2 + spare
    table = ref.make_table(rng, lengths, page, pages)
    k = ref.make_pool(rng, pages, page, heads, dim, dtype, layout, layers)
    v = ref.make_pool(rng, pages, page, heads, dim, dtype, layout, layers)
    cache = PagedCache(k, v, layout)
    batch = PagedBatch(table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), ref.offsets(rows).cuda(),
                       max_rows=max(rows), max_length=bound or max(lengths))
    return cache, batch, table


# ---- append -------------------------------------------------------------------------------

APPEND = [
    # type, cache, layout, page, kv heads, q heads, dim, rotary, interleaved, norm, rows, lengths
    (F32, BF16, "nhd", 16, 8, 16, 128, 128, False, True, [1], [42]),
    (F32, F32, "hnd", 16, 2, 4, 128, 128, False, True, [3, 1, 5], [3, 40, 16]),
    (BF16, BF16, "nhd", 1, 3, 3, 64, 64, False, False, [2, 0, 4], [7, 0, 4]),
    (F16, F16, "hnd", 24, 2, 14, 80, 80, False, True, [13, 2], [49, 25]),
    (F16, F16, "nhd", 5, 1, 4, 64, 32, True, False, [4, 1, 1], [4, 6, 5]),
    (F32, F16, "nhd", 32, 2, 2, 256, 128, True, True, [2, 33], [100, 64]),
    (BF16, F32, "nhd", 16, 2, 2, 40, 16, False, True, [3], [17]),
    (F32, BF16, "nhd", 16, 2, 2, 128, 20, False, True, [3, 2], [17, 2]),   # odd rotation: the scalar kernel
    (F32, F32, "nhd", 16, 2, 2, 128, 6, True, False, [3, 2], [17, 2]),
    (F32, BF16, "nhd", 16, 2, 0, 128, 0, False, False, [5, 60], [21, 60]),  # no q, no rotation
]


@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("odd_stride", [False, True])
def test_append(gpu, case, odd_stride):
    dt, cdt, layout, page, K, H, D, rot, inter, normed, rows, lengths = APPEND[case]
    rng = rng_of(case)
    cache, batch, table = make(rng, lengths, rows, page, K, D, cdt, layout)
    before_k, before_v = cache.k.clone(), cache.v.clone()
    T, pad = sum(rows), 2  # two padding rows behind the last sequence
    width = (H + 2 * K) * D + (3 if odd_stride else 0)
    qkv = torch.randn(T + pad, width, generator=rng).to(dt).cuda()
    q = qkv[:, :H * D].unflatten(1, (H, D)) if H else None
    k = qkv[:, H * D:(H + K) * D].unflatten(1, (K, D))
    v = qkv[:, (H + K) * D:(H + 2 * K) * D].unflatten(1, (K, D))
    freq = [1e4 ** (-2 * i / rot) for i in range(rot // 2)]
    w = [(1 + 0.2 * torch.randn(D, generator=rng)) if normed else None for _ in range(2)]
    pos = torch.randint(-5, 2 ** 22, (T + pad,), generator=rng, dtype=torch.int32) if case % 2 else None
    out = torch.full((T + pad, H, D), 7.0, dtype=cdt, device="cuda") if H else None
    got = cache.append(batch, k, v, q=q, inv_freq=torch.tensor(freq, dtype=torch.float64).cuda() if rot else None,
                       positions=pos.cuda() if pos is not None else None,
                       q_norm=w[0].cuda() if normed else None, k_norm=w[1].cuda() if normed else None,
                       eps=1e-6, interleaved=inter, out=out)
    cache.check()
    assert (got is None) == (H == 0)
    want_k, want_v = before_k.cpu().double(), before_v.cpu()
    wk, wv = ref.row_first(want_k, layout), ref.row_first(want_v, layout)
    slack = torch.zeros_like(want_k)
    sk = ref.row_first(slack, layout)
    # F32 before the rounding: the norm is a sum of D squares, a square root, a division and two
    # products ((D / 2 + 4) roundings at most), the rotation two products and a sum of values no
    # larger than the row's largest times sqrt 2, and angles good to 2^-22 of a turn.
    f32 = ((D / 2 + 4) * 2.0 ** -24 if normed else 0.0) + 3 * 2.0 ** -24 + 2 * math.pi * 2.0 ** -22
    t = 0
    for b, n in enumerate(rows):
        for i in range(n):
            index = lengths[b] - n + i
            p, at = int(table[b, index // page]), index % page
            at_pos = index if pos is None else int(pos[t])
            y = ref.rotate(ref.norm(k[t].cpu().double(), w[1], 1e-6), at_pos, freq, inter)
            wk[p, at] = y
            sk[p, at] = y.abs() * EPS[cdt] + TINY[cdt] + f32 * 1.5 * y.abs().max()
            wv[p, at] = v[t].cpu().to(cdt)
            if H:
                z = ref.rotate(ref.norm(q[t].cpu().double(), w[0], 1e-6), at_pos, freq, inter)
                tol = z.abs() * EPS[cdt] + TINY[cdt] + f32 * 1.5 * z.abs().max()
                assert ((got[t].cpu().double() - z).abs() <= tol).all(), (b, i)
            t += 1
    assert torch.equal(cache.v.cpu(), want_v)
    assert ((cache.k.cpu().double() - want_k).abs() <= slack).all()
    if H:
        assert (got[T:] == 7.0).all()  # padding rows are not written


def test_append_in_place_and_layers(gpu):
    rng = rng_of(3)
    cache, batch, table = make(rng, [9, 20], [2, 3], 16, 2, 64, F16, layers=3)
    before = cache.k.clone(), cache.v.clone()
    q, k, v = (torch.randn(5, h, 64, generator=rng).half().cuda() for h in (4, 2, 2))
    freq = 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    want = cache.append(batch, k, v, q=q, inv_freq=freq.cuda(), layer=1).clone()
    got = cache.append(batch, k, v, q=q, inv_freq=freq.cuda(), layer=1, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    assert torch.equal(cache.k[0], before[0][0]) and torch.equal(cache.k[2], before[0][2])
    assert not torch.equal(cache.k[1], before[0][1])
    assert torch.equal(cache.v[1][int(table[1, 1]), 3], v[4])


def test_append_bad_pages(gpu):
    """Rows whose position has no valid page are left out and marked; the others are written."""
    from potpori_b200.paged import PagedBatch

    rng = rng_of(4)
    cache, batch, table = make(rng, [20, 20, 20], [2, 2, 2], 16, 2, 64, BF16)
    table[1, 1] = -1
    table[2, 1] = cache.pages
    lengths = torch.tensor([20, 20, 20], dtype=torch.int32)
    before = cache.k.clone()
    k = torch.randn(6, 2, 64, generator=rng).bfloat16().cuda()
    cache.append(PagedBatch(table.cuda(), lengths.cuda(), batch.cu_rows, 2, 20), k, k)
    with pytest.raises(PPError):
        cache.check()
    cache.check()  # the mark is cleared
    want = before.clone()
    want[int(table[0, 1]), 2:4] = k[:2]
    assert torch.equal(cache.k, want)
    for bad in ([33, 20, 20], [1, 20, 20]):  # past the table; shorter than its rows
        cache.append(PagedBatch(batch.page_table, torch.tensor(bad, dtype=torch.int32).cuda(), batch.cu_rows, 2, 20),
                     k, k)
        with pytest.raises(PPError):
            cache.check()


# ---- tree attention -----------------------------------------------------------------------

TREE = [
    # type, layout, page, kv heads, heads, dim, rows, lengths, masked
    (F32, "nhd", 16, 8, 16, 128, [1], [42], False),
    (F32, "hnd", 5, 2, 8, 64, [7, 0, 1, 13], [30, 0, 1, 200], True),
    (F32, "nhd", 32, 1, 3, 256, [9, 2], [9, 70], True),
    (F32, "nhd", 8, 2, 2, 40, [3], [33], True),
    (BF16, "nhd", 16, 2, 4, 128, [1, 1, 1], [1, 17, 700], False),
    (BF16, "nhd", 16, 2, 8, 128, [8], [1300], True),
    (BF16, "hnd", 24, 3, 3, 64, [5, 0, 33], [5, 9, 333], True),
    (BF16, "nhd", 64, 1, 7, 80, [9, 20], [100, 64], True),
    (BF16, "nhd", 128, 2, 4, 256, [1, 12], [300, 12], True),
    (F16, "nhd", 1, 2, 4, 128, [3, 1], [70, 129], False),
    (F16, "hnd", 32, 2, 8, 128, [61, 40], [500, 41], True),
    (F16, "hnd", 16, 1, 1, 72, [70], [75], False),
    (F16, "nhd", 48, 2, 16, 256, [30], [130], True),
    (BF16, "nhd", 16, 1, 64, 128, [2, 4], [65, 64], True),
]


def attention_tolerance(dtype, want, most, length, dim, vmax):
    """Scores are F32 sums of dim products (error dim 2^-24 of the sum of magnitudes), which moves a
    probability by as much and its share by twice that; the sums over the positions add 2^-24 each;
    the exponential 2^-21; the probabilities' second part (16-bit types) leaves out 2^-16. Then the
    rounding of the output."""
    work = 2 * dim * 2.0 ** -24 * most + length * 2.0 ** -24 + 2.0 ** -21 + (0 if dtype == F32 else 2.0 ** -16)
    return want.abs() * EPS[dtype] + TINY[dtype] + work * vmax


def check_attention(cache, table, layout, page, rows, lengths, seen, q, got, lse, scale):
    t = 0
    for b, n in enumerate(rows):
        if n:
            k = ref.cached(cache.k, layout, table, b, lengths[b], page)
            v = ref.cached(cache.v, layout, table, b, lengths[b], page)
            want, wl, most = ref.attention(q[t:t + n].cpu().double(), k, v, seen[b], scale)
            tol = attention_tolerance(cache.dtype, want, most, lengths[b], cache.head_dim, v.abs().max())
            off = (got[t:t + n].cpu().double() - want).abs()
            assert (off <= tol).all(), (b, float((off - tol).max()), float(off.max()))
            dl = (lse[t:t + n].cpu().double() - wl).abs()
            empty = torch.isinf(wl)
            assert torch.equal(empty, torch.isinf(lse[t:t + n].cpu())), b
            lim = 2 * cache.head_dim * 2.0 ** -24 * most + lengths[b] * 2.0 ** -24 + 2.0 ** -20 + wl.abs() * 2.0 ** -22
            assert (dl[~empty] <= lim[~empty]).all(), b
        t += n


@pytest.mark.parametrize("bound", [None, FAR])
@pytest.mark.parametrize("case", range(len(TREE)))
def test_tree_attention(gpu, case, bound):
    dt, layout, page, K, H, D, rows, lengths, masked = TREE[case]
    rng = rng_of(100 + case)
    cache, batch, table = make(rng, lengths, rows, page, K, D, dt, layout, bound=bound)
    T, pad = sum(rows), 3
    q = (2 * torch.randn(T + pad, H, D, generator=rng)).to(dt).cuda()
    parents = [ref.random_parents(rng, n) if masked else [i - 1 for i in range(n)] for n in rows]
    seen = [ref.tree_seen(p, lengths[b] - rows[b]) for b, p in enumerate(parents)]
    mask = None
    if masked:
        bits = [s[i, lengths[b] - rows[b]:].nonzero()[:, 0].tolist() for b, s in enumerate(seen) for i in range(rows[b])]
        mask = ref.mask_words(bits + [[0]] * pad, -(-max(rows) // 32)).cuda()
    out = torch.full_like(q, 7.0)
    lse = torch.full((T + pad, H), 7.0, device="cuda")
    got = cache.tree_attention(batch, q, mask=mask, out=out, lse=lse)
    cache.check()
    check_attention(cache, table, layout, page, rows, lengths, seen, q, got, lse, D ** -0.5)
    assert (got[T:] == 7.0).all() and (lse[T:] == 7.0).all()
    assert torch.equal(cache.tree_attention(batch, q, mask=mask)[:T], got[:T])


@pytest.mark.parametrize("bound", [None, FAR])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("heads", [2, 16])
@pytest.mark.parametrize("page", [16, 24])
def test_tree_attention_masks(gpu, dt, heads, bound, page):
    """Rows that see nothing, only the context, only others, every node; nodes past the mask."""
    rng = rng_of(7)
    rows, lengths = [6, 40, 3], [6, 90, 200]
    cache, batch, table = make(rng, lengths, rows, page, 2, 128, dt, bound=bound)
    T = sum(rows)
    nodes = [[int(j) for j in range(n) if torch.rand(1, generator=rng) < 0.3] for n in rows for _ in range(n)]
    nodes[0] = []            # no context either: an empty row
    nodes[3] = [5]           # only a later node
    nodes[10] = []           # only the context
    nodes[20] = list(range(32))
    mask = ref.mask_words(nodes, 1).cuda() if max(max(x, default=0) for x in nodes) < 32 else None
    if mask is None:
        nodes = [[j for j in x if j < 32] for x in nodes]
        mask = ref.mask_words(nodes, 1).cuda()  # one word: nodes 32..39 are unseen by all
    seen, t = [], 0
    for b, n in enumerate(rows):
        s = torch.zeros(n, lengths[b], dtype=torch.bool)
        s[:, :lengths[b] - n] = True
        for i in range(n):
            s[i, [lengths[b] - n + j for j in nodes[t]]] = True
            t += 1
        seen.append(s)
    # Bits past a sequence's nodes mean nothing.
    mask[0:6] |= ~0x3F
    q = (2 * torch.randn(T, heads, 128, generator=rng)).to(dt).cuda()
    lse = torch.empty(T, heads, device="cuda")
    got = cache.tree_attention(batch, q, mask=mask, lse=lse, scale=0.05)
    check_attention(cache, table, "nhd", page, rows, lengths, seen, q, got, lse, 0.05)
    assert (got[0] == 0).all() and (lse[0] == -math.inf).all()


@pytest.mark.parametrize("bound", [None, FAR])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("heads", [2, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("page", [16, 24])
def test_tree_attention_nonfinite_where_unseen(gpu, dt, heads, bad, bound, page):
    """Behind a sequence's last position, in pages of nobody, and in K and V of unseen nodes."""
    rng = rng_of(8)
    rows, lengths = [12, 5], [70, 131]
    cache, batch, table = make(rng, lengths, rows, page, 2, 128, dt, bound=bound)
    q = torch.randn(17, heads, 128, generator=rng).to(dt).cuda()
    parents = [ref.random_parents(rng, n) for n in rows]
    seen = [ref.tree_seen(p, lengths[b] - rows[b]) for b, p in enumerate(parents)]
    bits = [s[i, lengths[b] - rows[b]:].nonzero()[:, 0].tolist() for b, s in enumerate(seen) for i in range(rows[b])]
    mask = ref.mask_words(bits, 1).cuda()
    want = cache.tree_attention(batch, q, mask=mask)
    used = torch.zeros(cache.pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        at = torch.arange(n)
        used[table[b].long()[at // page], at % page] = True
    cache.k[~used.cuda()] = bad
    cache.v[~used.cuda()] = bad
    assert torch.equal(cache.tree_attention(batch, q, mask=mask), want)
    # Node 7 of sequence 0: rows that see it take its values, the others keep every bit.
    index = lengths[0] - rows[0] + 7
    p, at = int(table[0, index // page]), index % page
    cache.k[p, at, 0], cache.v[p, at, 0, 3:90:5] = bad, bad
    got = cache.tree_attention(batch, q, mask=mask)
    blind = torch.tensor([7 not in x for x in bits[:12]] + [True] * 5)
    assert torch.equal(got[blind.cuda()], want[blind.cuda()])
    first = heads // 2  # query heads of cached head 0
    assert torch.equal(got[:, first:], want[:, first:])
    assert torch.isnan(got[:12][~blind[:12].cuda()][:, :first]).all()
    cache.k[p, at, 0] = 0.25
    got = cache.tree_attention(batch, q, mask=mask)
    hit = torch.zeros(128, dtype=torch.bool)
    hit[3:90:5] = True
    sees = got[:12][~blind[:12].cuda()][:, :first]
    assert (~torch.isfinite(sees[..., hit.cuda()])).all() and torch.isfinite(sees[..., ~hit.cuda()]).all()
    assert torch.equal(got[blind.cuda()], want[blind.cuda()])


@pytest.mark.parametrize("dt,heads,bound", [(F32, 1, None), (F32, 9, None), (BF16, 1, None), (BF16, 9, FAR)])
def test_tree_attention_score_ranges(gpu, dt, heads, bound):
    """Scores far from zero: all very negative, one that takes all, and equal ones."""
    rng = rng_of(9)
    cache, batch, table = make(rng, [150], [2], 16, 1, 64, dt, bound=bound)
    cache.k.zero_()
    cache.k[..., 0] = -200.0
    index = int(table[0, 3])
    cache.k[index, 5, 0, 0] = 200.0
    q = torch.zeros(2, heads, 64, dtype=dt, device="cuda")
    q[0, 0, 0], q[1, 0, 0] = 40.0, 1.0
    got = cache.tree_attention(batch, q, scale=1.0)
    assert torch.equal(got[0, 0], cache.v[index, 5, 0])
    q[:, 0, 0] = 0.0
    v = ref.cached(cache.v, "nhd", table, 0, 150, 16)[:, 0]
    got = cache.tree_attention(batch, q)
    tol = 150 * 2.0 ** -24 + 2.0 ** -15 * v.abs().max()
    assert ((got[1, 0].cpu().double() - v.mean(0)).abs() <= tol + v.mean(0).abs() * EPS[dt]).all()
    # Scores that rise by more than the kernels let pass without rescaling, tile after tile.
    for j in range(150):
        cache.k[int(table[0, j // 16]), j % 16, 0, 0] = j / 2.0
    q[:, :, 0] = 1.0
    got = cache.tree_attention(batch, q, scale=1.0)
    seen = ref.tree_seen([-1, 0], 148)
    want, _, most = ref.attention(q.cpu().double(), ref.cached(cache.k, "nhd", table, 0, 150, 16), v[:, None], seen, 1.0)
    assert ((got.cpu().double() - want).abs() <= attention_tolerance(dt, want, most, 150, 64, v.abs().max())).all()


@pytest.mark.parametrize("dt,heads,bound", [(F32, 2, None), (BF16, 2, None), (F16, 16, None), (F16, 16, FAR)])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-3])
def test_tree_attention_scales(gpu, dt, heads, bound, scale):
    """Any scale, its sign and zero among them."""
    rng = rng_of(15)
    rows, lengths, page = [5, 3], [140, 3], 16
    cache, batch, table = make(rng, lengths, rows, page, 2, 128, dt, bound=bound)
    q = (2 * torch.randn(8, heads, 128, generator=rng)).to(dt).cuda()
    lse = torch.empty(8, heads, device="cuda")
    seen = [ref.tree_seen([i - 1 for i in range(n)], lengths[b] - n) for b, n in enumerate(rows)]
    got = cache.tree_attention(batch, q, lse=lse, scale=scale)
    check_attention(cache, table, "nhd", page, rows, lengths, seen, q, got, lse, scale)


@pytest.mark.parametrize("dt,heads,bound,page", [(BF16, 4, 40, 16), (BF16, 4, 40, 8), (BF16, 10, FAR, 16), (F16, 10, FAR, 8),
                                                 (F32, 4, 40, 16)])
def test_tree_attention_bad_descriptors(gpu, dt, heads, bound, page):
    """A sequence whose lengths do not fit is left out, a bad page contributes nothing it could
    fault on, the rest of the batch is right."""
    from potpori_b200.paged import PagedBatch

    rng = rng_of(10)
    cache, batch, table = make(rng, [40, 40, 40], [2, 2, 2], page, 2, 128, dt, bound=bound)
    q = torch.randn(6, heads, 128, generator=rng).to(dt).cuda()
    want = cache.tree_attention(batch, q)
    for lengths in ([40, 49, 40], [40, 1, 40], [40, -3, 40]):
        out = torch.full_like(q, 7.0)
        b = PagedBatch(batch.page_table, torch.tensor(lengths, dtype=torch.int32).cuda(), batch.cu_rows, 2, bound)
        cache.tree_attention(b, q, out=out)
        with pytest.raises(PPError):
            cache.check()
        assert torch.equal(out[:2], want[:2]) and torch.equal(out[4:], want[4:]) and (out[2:4] == 7.0).all()
    for bad in (-1, cache.pages, 2 ** 30):
        t = table.clone()
        t[1, 1] = bad
        got = cache.tree_attention(PagedBatch(t.cuda(), batch.lengths, batch.cu_rows, 2, bound), q)
        with pytest.raises(PPError):
            cache.check()
        assert torch.equal(got[:2], want[:2]) and torch.equal(got[4:], want[4:])


@pytest.mark.parametrize("understated", [False, True])
def test_tree_attention_host_bounds(gpu, understated):
    """The host's bounds choose the kernels, not the results (but for rounding); they may even be
    too small."""
    from potpori_b200.paged import PagedBatch

    rng = rng_of(11)
    rows, lengths = [30, 4], [500, 77]
    cache, batch, table = make(rng, lengths, rows, 16, 2, 128, BF16)
    q = torch.randn(34, 8, 128, generator=rng).bfloat16().cuda()
    b = PagedBatch(batch.page_table, batch.lengths, batch.cu_rows, 1 if understated else 1000, 3 if understated else None)
    lse = torch.empty(34, 8, device="cuda")
    got = cache.tree_attention(b, q, lse=lse)
    seen = [ref.tree_seen([i - 1 for i in range(n)], lengths[i0] - n) for i0, n in enumerate(rows)]
    check_attention(cache, table, "nhd", 16, rows, lengths, seen, q, got, lse, 128 ** -0.5)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_tree_attention_far_offsets(gpu, dt):
    """Pages beyond 2^31 elements of the pool, and pools that interleave K and V."""
    from potpori_b200.paged import PagedBatch, PagedCache

    D, K, page = 128, 2, 16
    pages = 2 ** 31 // (page * K * D * 2) + 40
    pool = torch.zeros(pages, 2, page, K, D, dtype=dt, device="cuda")
    cache = PagedCache(pool[:, 0], pool[:, 1])
    assert pool.numel() > 2 ** 31
    rng = rng_of(12)
    table = torch.tensor([[pages - 1, 3, pages - 20]], dtype=torch.int32)
    batch = PagedBatch(table.cuda(), torch.tensor([41], dtype=torch.int32).cuda(), ref.offsets([41]).cuda(), 41, 41)
    k, v = (torch.randn(41, K, D, generator=rng).to(dt).cuda() for _ in range(2))
    cache.append(batch, k, v)
    q = torch.randn(41, 4, D, generator=rng).to(dt).cuda()
    seen = ref.tree_seen([i - 1 for i in range(41)], 0)
    want, _, most = ref.attention(q.cpu().double(), k.cpu().double(), v.cpu().double(), seen, D ** -0.5)
    tol = attention_tolerance(dt, want, most, 41, D, v.abs().max().cpu())
    for bound in (41, FAR):
        b = PagedBatch(batch.page_table, batch.lengths, batch.cu_rows, 41, bound)
        got = cache.tree_attention(b, q)
        cache.check()
        assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt,G", [(BF16, 1), (BF16, 8), (F16, 4), (F32, 2)])
def test_tree_attention_splits_agree(gpu, dt, G):
    """A long cache split over the whole card, twice: equal bits, and right on sampled rows."""
    rng = rng_of(13)
    rows, lengths, page = [24, 1], [20000, 6001], 64
    cache, batch, table = make(rng, lengths, rows, page, 1, 128, dt)
    parents = [ref.random_parents(rng, n) for n in rows]
    seen = [ref.tree_seen(p, lengths[b] - rows[b]) for b, p in enumerate(parents)]
    bits = [s[i, lengths[b] - rows[b]:].nonzero()[:, 0].tolist() for b, s in enumerate(seen) for i in range(rows[b])]
    mask = ref.mask_words(bits, 2).cuda()
    q = (2 * torch.randn(25, G, 128, generator=rng)).to(dt).cuda()
    lse = torch.empty(25, G, device="cuda")
    got = cache.tree_attention(batch, q, mask=mask, lse=lse)
    check_attention(cache, table, "nhd", page, rows, lengths, seen, q, got, lse, 128 ** -0.5)
    for _ in range(3):
        assert torch.equal(cache.tree_attention(batch, q, mask=mask), got)


@pytest.mark.parametrize("dt,heads,bound", [(BF16, 4, 40), (F16, 16, FAR), (F32, 4, 40)])
def test_rows_past_the_arrays(gpu, dt, heads, bound):
    """cu_rows that reaches past the row arrays, or before them: that sequence is left out, by the
    attention and by the commit."""
    from potpori_b200.paged import PagedBatch

    rng = rng_of(24)
    cache, batch, table = make(rng, [40, 40, 40], [2, 2, 2], 16, 2, 128, dt, bound=bound)
    q = torch.randn(6, heads, 128, generator=rng).to(dt).cuda()
    want = cache.tree_attention(batch, q)
    ints = torch.zeros(6, dtype=torch.int32).cuda()
    for cu, left in (([0, 2, 4, 8], slice(4, 6)), ([0, 2, 4, 2 ** 31 - 1], slice(4, 6)), ([-2, 2, 4, 6], slice(0, 2))):
        b = PagedBatch(batch.page_table, batch.lengths, torch.tensor(cu, dtype=torch.int32).cuda(), 8, bound)
        out = torch.full_like(q, 7.0)
        cache.tree_attention(b, q, out=out)
        with pytest.raises(PPError):
            cache.check()
        keep = torch.ones(6, dtype=torch.bool, device="cuda")
        keep[left] = False
        assert torch.equal(out[keep], want[keep]) and (out[left] == 7.0).all()
        path, accepted, correction, new_len = cache.tree_commit(b, ints, ints - 1, ints + 1)
        with pytest.raises(PPError):
            cache.check()
        off = left.start // 2
        assert [int(x) for x in (accepted[off], correction[off], new_len[off])] == [0, -1, 40]
        assert (path[off] == -1).all() and all(int(path[b, 0]) == 0 for b in range(3) if b != off)


@pytest.mark.parametrize("dt,G,bound", [(BF16, 1, None), (BF16, 4, FAR), (F16, 5, FAR), (F32, 2, None)])
@pytest.mark.parametrize("long", [3000, 260])
def test_tree_attention_ragged_batch(gpu, dt, G, bound, long):
    """Many short sequences around a long one: CTAs that take parts of several units, or (none much
    longer than the rest) whole units by falling length."""
    rng = rng_of(25)
    B = 30
    rows = [int(torch.randint(0, 21, (1,), generator=rng)) if dt != BF16 or G > 1 else 1 for _ in range(B)]
    lengths = [n + int(torch.randint(100, 240, (1,), generator=rng)) for n in rows]
    rows[17], lengths[17] = max(rows[17], 1), long
    cache, batch, table = make(rng, lengths, rows, 16, 4, 64, dt, bound=bound)
    parents = [ref.random_parents(rng, n) for n in rows]
    seen = [ref.tree_seen(p, lengths[b] - rows[b]) for b, p in enumerate(parents)]
    bits = [s[i, lengths[b] - rows[b]:].nonzero()[:, 0].tolist() for b, s in enumerate(seen) for i in range(rows[b])]
    mask = ref.mask_words(bits, 1).cuda()
    T = sum(rows)
    q = (2 * torch.randn(T, 4 * G, 64, generator=rng)).to(dt).cuda()
    lse = torch.empty(T, 4 * G, device="cuda")
    got = cache.tree_attention(batch, q, mask=mask, lse=lse)
    cache.check()
    check_attention(cache, table, "nhd", 16, rows, lengths, seen, q, got, lse, 64 ** -0.5)
    assert torch.equal(cache.tree_attention(batch, q, mask=mask), got)


def test_masks_without_words_are_refused(gpu):
    rng = rng_of(26)
    cache, batch, _ = make(rng, [20], [3], 16, 2, 64, BF16)
    q = torch.randn(3, 4, 64, generator=rng).bfloat16().cuda()
    for mask in (torch.zeros(3, 0, dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int32).cuda()):
        with pytest.raises(PPError):
            cache.tree_attention(batch, q, mask=mask)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 8, 12, 40])
def test_tree_attention_small_pages(gpu, page, dim):
    """Many vectors a head over pages that end inside a tile: by boxes of 8 rows, or row by row."""
    rng = rng_of(27 + page)
    rows, lengths = [40, 3], [333, 70]
    cache, batch, table = make(rng, lengths, rows, page, 2, dim, F16, "hnd", bound=FAR)
    parents = [ref.random_parents(rng, n) for n in rows]
    seen = [ref.tree_seen(p, lengths[b] - rows[b]) for b, p in enumerate(parents)]
    bits = [s[i, lengths[b] - rows[b]:].nonzero()[:, 0].tolist() for b, s in enumerate(seen) for i in range(rows[b])]
    q = torch.randn(43, 8, dim, generator=rng).half().cuda()
    lse = torch.empty(43, 8, device="cuda")
    got = cache.tree_attention(batch, q, mask=ref.mask_words(bits, 2).cuda(), lse=lse)
    cache.check()
    check_attention(cache, table, "hnd", page, rows, lengths, seen, q, got, lse, dim ** -0.5)


def test_large_batch(gpu):
    """More sequences than a CTA has threads, many without rows."""
    rng = rng_of(14)
    B = 700
    rows = [int(torch.randint(0, 3, (1,), generator=rng)) for _ in range(B)]
    lengths = [n + int(torch.randint(0, 40, (1,), generator=rng)) for n in rows]
    cache, batch, table = make(rng, lengths, rows, 8, 1, 64, F16)
    T = sum(rows)
    q, k, v = (torch.randn(T, h, 64, generator=rng).half().cuda() for h in (2, 1, 1))
    cache.append(batch, k, v)
    got = cache.tree_attention(batch, q, lse=(lse := torch.empty(T, 2, device="cuda")))
    cache.check()
    t = 0
    for b, n in enumerate(rows):
        for i in range(n):
            index = lengths[b] - n + i
            assert torch.equal(cache.v[int(table[b, index // 8]), index % 8], v[t])
            t += 1
    seen = [ref.tree_seen([i - 1 for i in range(n)], lengths[b] - n) for b, n in enumerate(rows)]
    check_attention(cache, table, "nhd", 8, rows, lengths, seen, q, got, lse, 64 ** -0.5)


# ---- commit -------------------------------------------------------------------------------


@pytest.mark.parametrize("dt,layout,page,layers,rows,lengths", [
    (BF16, "nhd", 16, 3, [8], [49]),
    (F32, "hnd", 5, 0, [1, 31, 0, 9], [1, 40, 3, 30]),
    (F16, "nhd", 1, 2, [64, 12], [64, 40]),
    (BF16, "hnd", 24, 1, [200], [230]),
])
def test_tree_commit(gpu, dt, layout, page, layers, rows, lengths):
    for seed in range(4):
        rng = rng_of(seed)
        cache, batch, table = make(rng, lengths, rows, page, 3, 40, dt, layout, layers)
        T = sum(rows)
        parents = [ref.random_parents(rng, n) if n else [] for n in rows]
        tokens = torch.randint(0, 3 if seed % 2 else 1000, (T,), generator=rng)
        picks = torch.randint(0, 3 if seed % 2 else 1000, (T,), generator=rng)
        cu = ref.offsets(rows).tolist()
        if seed % 2 == 0:  # a long path
            for b, n in enumerate(rows):
                for i in range(1, n):
                    picks[cu[b] + parents[b][i]] = tokens[cu[b] + i]
        flat = torch.tensor([p for x in parents for p in x], dtype=torch.int32)
        want_k, want_v = cache.k.clone(), cache.v.clone()
        ints = [x.to(torch.int32).cuda() for x in (tokens, flat, picks)]
        path, accepted, correction, new_len = cache.tree_commit(batch, *ints)
        cache.check()
        for b, n in enumerate(rows):
            if not n:
                assert path[b].tolist() == [-1] * max(rows)
                assert (int(accepted[b]), int(correction[b]), int(new_len[b])) == (0, -1, lengths[b])
                continue
            tk, pk = tokens[cu[b]:cu[b + 1]].tolist(), picks[cu[b]:cu[b + 1]].tolist()
            want = ref.commit(tk, parents[b], pk)
            assert path[b].tolist() == want + [-1] * (max(rows) - len(want))
            assert int(accepted[b]) == len(want) - 1 and int(correction[b]) == pk[want[-1]]
            assert int(new_len[b]) == lengths[b] - n + len(want)
            for pool in (want_k, want_v):
                rf = ref.row_first(pool, layout)
                rf = rf if layers else rf[None]
                place = lambda j: (int(table[b, j // page]), j % page)  # noqa: E731
                moved = [rf[:, place(lengths[b] - n + w)[0], place(lengths[b] - n + w)[1]].clone() for w in want]
                for d, row in enumerate(moved):
                    rf[:, place(lengths[b] - n + d)[0], place(lengths[b] - n + d)[1]] = row
        assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


def test_tree_commit_odd_trees(gpu):
    """Parents that are not before their node hang it on nothing; more nodes than max_rows and bad
    pages are refused where they occur."""
    from potpori_b200.paged import PagedBatch

    rng = rng_of(5)
    cache, batch, table = make(rng, [20, 20], [5, 5], 16, 2, 64, BF16)
    parents = torch.tensor([3, 0, 2, 7, -5] + [-1, 0, 1, 1, 3], dtype=torch.int32).cuda()
    tokens = torch.tensor([9, 9, 9, 9, 9] + [1, 2, 3, 3, 4], dtype=torch.int32).cuda()
    picks = torch.tensor([9, 9, 9, 9, 9] + [2, 3, 4, 4, 5], dtype=torch.int32).cuda()
    path, accepted, correction, new_len = cache.tree_commit(batch, tokens, parents, picks)
    assert path.tolist() == [[0, 1, -1, -1, -1], [0, 1, 2, -1, -1]]
    assert accepted.tolist() == [1, 2] and correction.tolist() == [9, 4] and new_len.tolist() == [17, 18]
    cache.check()
    before = cache.k.clone()
    b = PagedBatch(batch.page_table, batch.lengths, batch.cu_rows, 4, 20)
    path, accepted, _, new_len = cache.tree_commit(b, tokens, parents, picks)
    assert (path == -1).all() and accepted.tolist() == [0, 0] and new_len.tolist() == [20, 20]
    with pytest.raises(PPError):
        cache.check()
    t = table.clone()
    t[1, 1] = cache.pages
    parents[6:] = torch.tensor([-1, 0, 0, 3], dtype=torch.int32)  # the path 0, 2 must move
    tokens[7], picks[5] = 2, 2
    cache.tree_commit(PagedBatch(t.cuda(), batch.lengths, batch.cu_rows, 5, 20), tokens, parents, picks)
    with pytest.raises(PPError):
        cache.check()
    assert torch.equal(cache.k, before)


# ---- beams --------------------------------------------------------------------------------


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (2, 3, 5, 4), (1, 4, 151936, 4), (3, 8, 5001, 16), (2, 5, 4096, 17), (1, 33, 9000, 64),
    (1, 64, 300, 64), (1, 2, 600000, 3), (5, 2, 40000, 1),
])
def test_beam_select(gpu, dt, groups, beams, vocab, k):
    from potpori_b200.paged import beam_select

    rng = rng_of(vocab + k)
    for ties in (False, True):
        logits = 3 * torch.randn(groups, beams, vocab, generator=rng)
        if ties:
            logits = logits.round()
        logits = logits.to(dt)
        scores = -5 + torch.randn(groups, beams, generator=rng)
        if ties and beams > 1:
            logits[:, 1], scores[:, 1] = logits[:, 0], scores[:, 0]
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = [x.cpu() for x in beam_select(logits.cuda(), scores.cuda(), k, err=err)]
        assert int(err) == 0
        for g in range(groups):
            want = ref.beam(logits[g], scores[g], k)
            assert [(int(b), int(t)) for b, t in zip(got[1][g], got[2][g])] == [(b, t) for _, b, t in want], g
            for s, w in zip(got[0][g].tolist(), want):
                # lse: exponentials good to 2^-21 each, so log of their sum to 2^-20.
                assert s == w[0] or abs(s - w[0]) <= abs(w[0]) * 2.0 ** -24 + 2.0 ** -20


def test_beam_select_special_rows(gpu):
    """Unused, finished, masked and non-finite beams; too few candidates; odd strides."""
    from potpori_b200.paged import beam_select

    rng = rng_of(2)
    W, V, k = 8, 5000, 6
    pool = torch.randn(1, W, V + 7, generator=rng)
    logits = pool[..., :V]
    scores = -3 + torch.randn(1, W, generator=rng)
    finished = torch.zeros(1, W, dtype=torch.bool)
    scores[0, 0] = -math.inf           # not in use
    finished[0, 1] = True              # goes on as pad
    logits[0, 1] = math.nan            # and its logits are not looked at
    logits[0, 2] = -math.inf           # nothing allowed
    logits[0, 3, 1:] = -math.inf       # one token
    scores[0, 3] = 0.5
    logits[0, 4, 77] = math.nan        # left out
    logits[0, 5, 4999] = math.inf      # left out
    scores[0, 6] = math.nan            # left out
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = beam_select(pool.cuda()[..., :V], scores.cuda(), k, finished=finished.cuda(), pad=42, err=err)
    want = ref.beam(logits[0], scores[0], k, finished[0], 42)
    assert int(err) == 2
    assert got[1][0].tolist() == [w[1] for w in want] and got[2][0].tolist() == [w[2] for w in want]
    assert want[0][1:] == (3, 0) and abs(float(got[0][0, 0]) - 0.5) < 1e-6
    # Only two candidates in all.
    scores[0, 7] = -math.inf
    got = beam_select(pool.cuda()[..., :V], scores.cuda(), k, finished=finished.cuda(), pad=42)
    assert got[1][0].tolist() == [3, 1, -1, -1, -1, -1] and got[2][0].tolist()[:3] == [0, 42, -1]
    assert got[0][0, 2:].tolist() == [-math.inf] * 4
    # All logits equal: the lowest tokens of the best beam.
    flat = torch.zeros(2, 3, 9000, device="cuda")
    s = torch.tensor([[-1.0, -0.5, -0.5], [-2.0, -3.0, -4.0]], device="cuda")
    got = beam_select(flat, s, 20)
    assert got[1][0].tolist() == [1] * 20 and got[2][0].tolist() == list(range(20))
    assert got[1][1].tolist() == [0] * 20


@pytest.mark.parametrize("dt,layout,page,layers", [(BF16, "nhd", 16, 3), (F32, "hnd", 5, 0), (F16, "nhd", 1, 2)])
def test_beam_reorder(gpu, dt, layout, page, layers):
    rng = rng_of(6)
    g, old, new = 3, 4, 6
    lengths = torch.tensor([[16, 17, 31, 1], [0, 5, 20, 20], [33, 33, 33, 33]], dtype=torch.int32)
    flat = lengths.flatten().tolist()
    cache, _, table = make(rng, flat, [1] * 12, page, 2, 64, dt, layout, layers, spare=g * new)
    free = [i for i in range(cache.pages) if i not in set(table.flatten().tolist())][:g * new]
    spare = torch.tensor(free, dtype=torch.int32).view(g, new)
    table = table.view(g, old, -1)
    beams = torch.tensor([[1, 1, 3, 1, 0, 0], [2, 2, -1, 0, 3, 2], [0, 0, 0, 0, 0, 0]], dtype=torch.int32)
    want_k, want_v = cache.k.clone(), cache.v.clone()
    got_t, got_l, taken = (x.cpu() for x in cache.beam_reorder(table.cuda(), lengths.cuda(), beams.cuda(), spare.cuda()))
    cache.check()
    for a in range(g):
        for j in range(new):
            p = int(beams[a, j])
            if p < 0:
                assert got_t[a, j].tolist() == [-1] * table.shape[2] and got_l[a, j] == 0 and taken[a, j] == 0
                continue
            n = int(lengths[a, p])
            row = table[a, p].tolist()
            copies = p in beams[a, :j].tolist() and n % page != 0
            assert int(taken[a, j]) == int(copies) and int(got_l[a, j]) == n
            if copies:
                src, dst = row[n // page], int(spare[a, j])
                row[n // page] = dst
                for pool in (want_k, want_v):
                    rf = ref.row_first(pool, layout)
                    rf = rf if layers else rf[None]
                    rf[:, dst, :n % page] = rf[:, src, :n % page]
            assert got_t[a, j].tolist() == row
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


# ---- streams, graphs ----------------------------------------------------------------------


def test_streams_and_graphs(gpu):
    """Two streams at once, and two captured graphs replayed over new contents, against the same
    calls one by one."""
    rng = rng_of(20)
    rows, lengths = [9, 1, 4], [300, 1000, 4]
    setups = []
    for dt in (BF16, F16):
        cache, batch, table = make(rng, lengths, rows, 16, 2, 128, dt, layers=2)
        q, k, v = (torch.randn(14, h, 128, generator=rng).to(dt).cuda() for h in (8, 2, 2))
        par = torch.tensor([p for n in rows for p in ref.random_parents(rng, n)], dtype=torch.int32).cuda()
        tok = torch.randint(0, 3, (14,), generator=rng, dtype=torch.int32).cuda()
        pick = torch.randint(0, 3, (14,), generator=rng, dtype=torch.int32).cuda()
        logits = torch.randn(3, 4, 30000, generator=rng).cuda()
        scores = torch.randn(3, 4, generator=rng).cuda()
        setups.append((cache, batch, q, k, v, par, tok, pick, logits, scores))

    from potpori_b200.paged import beam_select

    def step(s):
        cache, batch, q, k, v, par, tok, pick, logits, scores = s
        q1 = cache.append(batch, k, v, q=q, layer=1)
        o = cache.tree_attention(batch, q1, layer=1)
        return [o, *beam_select(logits, scores, 4), *cache.tree_commit(batch, tok, par, pick)]

    start = [(s[0].k.clone(), s[0].v.clone()) for s in setups]

    def restore():
        for s, (k, v) in zip(setups, start):
            s[0].k.copy_(k)
            s[0].v.copy_(v)
        torch.cuda.synchronize()

    want = [step(s) for s in setups]
    want_k = [s[0].k.clone() for s in setups]
    restore()
    streams = [torch.cuda.Stream() for _ in setups]
    got = []
    for s, st in zip(setups, streams):
        with torch.cuda.stream(st):
            got.append(step(s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(s[0].k, k) for s, k in zip(setups, want_k))
    restore()
    graphs = []
    for s in setups:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s)
        graphs.append((graph, out))
    fresh = [torch.randn(14, 8, 128, generator=rng).to(s[2].dtype).cuda() for s in setups]
    for s, f in zip(setups, fresh):
        s[2].copy_(f)
    for _ in range(3):
        restore()
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
    captured = [[x.clone() for x in out] for _, out in graphs]
    restore()
    for s, c in zip(setups, captured):
        assert all(torch.equal(x, y) for x, y in zip(step(s), c))
