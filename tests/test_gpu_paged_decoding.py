"""The paged operators together, as a decoder uses them: speculation with draft trees and beam search
over a small transformer, against the same model in float64 that recomputes the whole sequence for
every token. Both must give the tokens of plain greedy decoding (of exhaustive beam search)."""
import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

LAYERS, H, K, D, V, HID = 2, 4, 2, 64, 97, 128
FREQ = [1e4 ** (-2 * i / D) for i in range(D // 2)]


class Model:
    """Norm-free residual attention layers with QK-norm and rotation; weights float64 on the host."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64) / math.sqrt(s[-1])  # noqa: E731
        self.embed = w(V, HID) * math.sqrt(HID)
        self.qkv = [w((H + 2 * K) * D, HID) for _ in range(LAYERS)]
        self.o = [w(HID, H * D) for _ in range(LAYERS)]
        self.qn = [1 + 0.1 * torch.randn(D, generator=g, dtype=torch.float64) for _ in range(LAYERS)]
        self.kn = [1 + 0.1 * torch.randn(D, generator=g, dtype=torch.float64) for _ in range(LAYERS)]
        self.head = w(V, HID) * 3

    def full(self, tokens):
        """Logits after every token, from scratch."""
        x = self.embed[torch.tensor(tokens)]
        n = len(tokens)
        seen = ref.tree_seen([i - 1 for i in range(n)], 0)
        for l in range(LAYERS):
            y = x @ self.qkv[l].T
            q, k, v = (t.unflatten(1, (-1, D)) for t in y.split((H * D, K * D, K * D), 1))
            q = torch.stack([ref.rotate(ref.norm(q[i], self.qn[l], 1e-6), i, FREQ, False) for i in range(n)])
            k = torch.stack([ref.rotate(ref.norm(k[i], self.kn[l], 1e-6), i, FREQ, False) for i in range(n)])
            x = x + ref.attention(q, k, v, seen, D ** -0.5)[0].flatten(1) @ self.o[l].T
        return x @ self.head.T


class Paged:
    """The same model on the device in F32, over one paged cache."""

    def __init__(self, model, dtype, page=8, pages=64):
        from potpori_b200.paged import PagedCache

        f = lambda t: t.float().cuda()  # noqa: E731
        self.embed, self.head = f(model.embed), f(model.head)
        self.qkv, self.o = [f(w) for w in model.qkv], [f(w) for w in model.o]
        self.qn, self.kn = [f(w) for w in model.qn], [f(w) for w in model.kn]
        self.freq = torch.tensor(FREQ, dtype=torch.float64).cuda()
        pool = torch.full((LAYERS, 2, pages, page, K, D), math.nan, dtype=dtype, device="cuda")
        self.cache = PagedCache(pool[:, 0], pool[:, 1])

    def forward(self, batch, tokens, positions=None, mask=None):
        x = self.embed[tokens.long()]
        for l in range(LAYERS):
            y = x @ self.qkv[l].T
            q, k, v = (t.unflatten(1, (-1, D)) for t in y.split((H * D, K * D, K * D), 1))
            q = self.cache.append(batch, k, v, q=q, inv_freq=self.freq, positions=positions, q_norm=self.qn[l],
                                  k_norm=self.kn[l], layer=l)
            a = self.cache.tree_attention(batch, q, mask=mask, layer=l)
            x = x + a.float().flatten(1) @ self.o[l].T
        return x @ self.head.T


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("quality", [1.0, 0.6, 0.0])
def test_speculation_with_trees(gpu, quality):
    """Trees drawn around the greedy continuation (each true token is drafted with probability
    `quality`, beside wrong ones): the committed tokens are those of greedy decoding, whatever was
    drafted, and the cache stays contiguous."""
    from potpori_b200.paged import PagedBatch

    model = Model(1)
    rng = torch.Generator().manual_seed(5)
    prompts, new = [[3, 14, 15, 92, 65], [27, 18, 28]], 16
    truth = []
    for p in prompts:
        t = list(p)
        for _ in range(new + 8):
            t.append(int(model.full(t)[-1].argmax()))
        truth.append(t)
    # F32: its error is far below the gaps between the best and the second logit here.
    gaps = [g for t in truth for g in model.full(t).topk(2).values.diff().abs().flatten().tolist()]
    assert min(gaps) > 1e-4
    dev = Paged(model, torch.float32)
    table = torch.randperm(64, generator=rng)[:16].view(2, 8).to(torch.int32).cuda()
    # Prompts: chains.
    rows = [len(p) for p in prompts]
    batch = PagedBatch(table, ints(rows), ref.offsets(rows).cuda(), max(rows), 64)
    logits = dev.forward(batch, ints([t for p in prompts for t in p]))
    ends = ref.offsets(rows)[1:].long() - 1
    current = logits[ends].argmax(-1).tolist()
    done = [[c] for c in current]
    lengths = list(rows)
    steps = 0
    while min(map(len, done)) < new:
        trees = []
        for b in range(2):
            tokens, parents, spine = [done[b][-1]], [-1], 0
            for d in range(4):
                true = truth[b][len(prompts[b]) + len(done[b]) + d]
                for _ in range(int(torch.randint(0, 2, (1,), generator=rng))):  # a wrong sibling before it
                    tokens.append((true + 1 + int(torch.randint(0, V - 2, (1,), generator=rng))) % V)
                    parents.append(spine)
                if torch.rand(1, generator=rng) < quality:
                    tokens.append(true)
                    parents.append(spine)
                    spine = len(tokens) - 1
            trees.append((tokens, parents))
        rows = [len(t) for t, _ in trees]
        now = [lengths[b] + rows[b] for b in range(2)]
        seen = [ref.tree_seen(p, 0) for _, p in trees]
        depth = []
        for b, (t, p) in enumerate(trees):
            for i in range(len(t)):
                depth.append(lengths[b] + int(seen[b][i].sum()) - 1)
        mask = ref.mask_words([s[i].nonzero()[:, 0].tolist() for s in seen for i in range(len(s))], 1).cuda()
        batch = PagedBatch(table, ints(now), ref.offsets(rows).cuda(), max(rows), 64)
        tokens = ints([x for t, _ in trees for x in t])
        logits = dev.forward(batch, tokens, positions=ints(depth), mask=mask)
        path, accepted, correction, new_len = dev.cache.tree_commit(
            batch, tokens, ints([x for _, p in trees for x in p]), logits.argmax(-1).to(torch.int32))
        for b in range(2):
            nodes = path[b, 1:1 + int(accepted[b])].tolist()
            done[b] += [trees[b][0][i] for i in nodes] + [int(correction[b])]
            lengths[b] = int(new_len[b])
            assert lengths[b] == len(prompts[b]) + len(done[b]) - 1
        steps += 1
    dev.cache.check()
    for b in range(2):
        assert done[b][:new] == truth[b][len(prompts[b]):][:new]
    assert quality < 1 or steps <= -(-new // 5) + 1  # every draft accepted: five tokens a step


def test_beam_search(gpu):
    """Beams that share and copy pages against beam search by recomputation."""
    from potpori_b200.paged import PagedBatch, beam_select

    model, W, new, page = Model(2), 4, 14, 8
    prompt = [5, 6, 7, 8, 9, 10]
    beams = [(0.0, list(prompt))]
    for _ in range(new):
        found = []
        for b, (s, t) in enumerate(beams):
            lp = torch.log_softmax(model.full(t)[-1], -1)
            found += [(s + float(lp[v]), b, v) for v in range(V)]
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        assert min(a[0] - b[0] for a, b in zip(found[:W], found[1:W + 1])) > 1e-4  # no ties to F32's error
        beams = [(s, beams[b][1] + [v]) for s, b, v in found[:W]]
    dev = Paged(model, torch.float32, page, pages=64)
    # Every beam starts on the prompt's pages; the pages not in use are kept on the host.
    free = list(range(63, -1, -1))
    first = [free.pop()]
    table = torch.full((1, W, 4), -1, dtype=torch.int32)
    table[0, :, 0] = first[0]
    table, lengths = table.cuda(), ints([[len(prompt)] * W])
    b0 = PagedBatch(table[0, :1].contiguous(), lengths[0, :1].contiguous(), ints([0, len(prompt)]), len(prompt), 32)
    logits = dev.forward(b0, ints(prompt))[-1:]
    # One beam in use; the others wait at -inf.
    scores = torch.tensor([[0.0] + [-math.inf] * (W - 1)], device="cuda")
    logits = logits.expand(W, V).contiguous()[None]
    tokens = [[] for _ in range(W)]
    for step in range(new):
        scores, chosen, picked = beam_select(logits, scores, W)
        spare = [free.pop() for _ in range(W)]
        table, lengths, taken = dev.cache.beam_reorder(table, lengths, chosen, ints([spare]))
        free += [p for p, t in zip(spare, taken[0].tolist()) if not t]
        tokens = [tokens[p] + [t] for p, t in zip(chosen[0].tolist(), picked[0].tolist())]
        # The new tokens' rows: a fresh page where the last is full.
        host = table[0].tolist()
        for j, n in enumerate(lengths[0].tolist()):
            if n % page == 0:
                host[j][n // page] = free.pop()
        table, lengths = ints([host]), lengths + 1
        batch = PagedBatch(table[0], lengths[0], ref.offsets([1] * W).cuda(), 1, 32)
        logits = dev.forward(batch, picked[0].contiguous())[None]
    dev.cache.check()
    assert [prompt + t for t in tokens] == [t for _, t in beams]
    assert all(abs(a - b[0]) < 1e-3 for a, b in zip(scores[0].tolist(), beams))
