"""Appending to pages and eviction on the GPU (msd_paged_append, msd_paged_evict), which move values and so are exact, and a model's
layers run on the paged cache's operators together."""
import math
import random

import pytest
import torch

from test_paged_attention_gpu import rand, rows_of, tables_of
from transformer_amd.attention import attention
from transformer_amd.norm import rms_norm
from transformer_amd.paged import PagePool
from transformer_amd.paged_attention import PagedEviction, PagedSequences, paged_append, paged_attention, paged_evict
from transformer_amd.rotary import rotary, rotary_frequencies
from transformer_amd.swiglu import swiglu

pytestmark = pytest.mark.gpu


def same(a, b):
    """Bit for bit (NaNs of any payload among them)."""
    a, b = a.contiguous(), b.contiguous()
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.view(kind), b.view(kind))


# ---- append ----

def appended(k, k_pages, q_lens, lengths, tables, starts):
    want = k_pages.clone()
    for s, (n, L) in enumerate(zip(q_lens, lengths)):
        for i in range(n):
            p = L - n + i
            want[:, 16 * tables[s][p // 16] + p % 16] = k[starts[s] + i]
    return want


@pytest.mark.parametrize("q_lens,lengths,KV,D", [
    ([1], [1], 1, 64),
    ([1, 1, 1, 1], [16, 17, 32, 300], 4, 64),
    ([3, 0, 40, 1], [18, 50, 40, 1], 2, 128),
    ([100, 77], [115, 300], 3, 96),
    ([15, 16, 17], [15, 31, 49], 1, 8),
    ([2000], [2100], 2, 40),
])
@pytest.mark.parametrize("starts", [None, "apart"])
def test_append(q_lens, lengths, KV, D, starts):
    tables, n = tables_of(lengths, 1)
    at = [sum(q_lens[:s]) for s in range(len(q_lens))]
    if starts:
        at = [x + 2 * s + 1 for s, x in enumerate(at)]
    k, v = (rand((sum(q_lens) + 2 * len(q_lens), KV, D), i) for i in (1, 2))
    k[0], v[-1] = math.nan, math.inf
    kp, vp = rand((KV, 16 * n, D), 3), rand((KV, 16 * n, D), 4)
    want = [appended(x, p, q_lens, lengths, tables, at) for x, p in ((k, kp), (v, vp))]
    sequences = PagedSequences(q_lens, lengths, tables, 2 * KV, KV, q_starts=at)
    version = kp._version
    assert paged_append(k, v, kp, vp, sequences) is None
    assert same(kp, want[0]) and same(vp, want[1]) and kp._version > version


@pytest.mark.parametrize("D", [64, 72])
def test_append_of_other_strides(D):
    """Parts of a projection, to layers of a pool of (position, head) order; rows that have to be copied first."""
    q_lens, lengths, H, KV = [5, 20], [30, 20], 4, 2
    tables, n = tables_of(lengths, 2)
    sequences = PagedSequences(q_lens, lengths, tables, H, KV)
    qkv = rand((25, H + 2 * KV, D), 1)
    k, v = qkv[:, H:H + KV], qkv[:, H + KV:]
    pool = rand((3, 2, 16 * n, KV, D), 2).transpose(2, 3)
    want = pool.clone()
    for i, x in enumerate((k, v)):
        want[1, i] = appended(x, pool[1, i], q_lens, lengths, tables, [0, 5])
    paged_append(k, v, pool[1, 0], pool[1, 1], sequences)
    assert same(pool, want)
    odd = torch.zeros((25, KV, D + 1), dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = v
    paged_append(k, odd[..., 1:], pool[1, 0], pool[1, 1], sequences)
    assert same(pool, want)


def test_append_past_32_bit_offsets():
    n = 600000 // 16
    pool = torch.zeros((3, 16 * n, 1536), dtype=torch.bfloat16, device="cuda")
    k_pages, v_pages = pool[..., 1280:1408], pool[..., 1408:]
    k, v = rand((20, 3, 128), 1), rand((20, 3, 128), 2)
    table = [n - 1, n - 3]
    paged_append(k, v, k_pages, v_pages, PagedSequences([20], [25], [table], 3, 3))
    for x, pages in ((k, k_pages), (v, v_pages)):
        assert same(rows_of(pages, table, 25)[:, 5:], x.transpose(0, 1))
    for s in (slice(0, 16 * (n - 3)), slice(16 * (n - 2), 16 * (n - 1))):
        assert not any(pool[h, s].any() for h in range(3))


def test_append_refusals():
    tables, n = tables_of([20, 20], 1)
    k, kp = rand((2, 2, 64), 1), rand((2, 16 * n, 64), 2)
    s = PagedSequences([1, 1], [20, 20], tables, 4, 2)
    for bad, match in (((k[:1], k, kp, kp), "rows"), ((k, k[:, :1], kp, kp), "v .rows"), ((k.float(), k, kp, kp), "bfloat16"), ((k, k.cpu(), kp, kp), "GPU"),
                       ((k, k, kp[:, :32], kp[:, :32]), "tables reach"), ((k, k, kp[:1].expand(2, -1, -1), kp), "overlap"),
                       ((k, k, kp, kp[:, :1].expand(-1, 16 * n, -1)), "overlap"), ((k, k, rand((2, 16 * n, 72), 1)[..., 4:68], kp), "16-byte"),
                       ((k, k, rand((2, 16 * n, 68), 1)[..., :64], kp), "16-byte"), ((k, k, rand((2, 64, 16 * n), 1).transpose(1, 2), kp), "contiguous")):
        with pytest.raises(ValueError, match=match):
            paged_append(*bad, s)
    with pytest.raises(ValueError, match="same memory"):
        paged_append(k, k, kp, kp, s)
    with pytest.raises(ValueError, match="elsewhere"):
        paged_append(k, k, kp, kp.clone(), PagedSequences([1, 1], [20, 20], [tables[0]] * 2, 4, 2))
    leaf = k.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        paged_append(leaf, k, kp, kp.clone(), s)
    with torch.no_grad():
        paged_append(leaf, k, kp, kp.clone(), s)


# ---- eviction ----

def evicted(k, v, w, lengths, tables, to, keep, recent):
    """(k, v, weights, kept) of (layers, kv heads, ..) by lists."""
    k, v = k.clone(), v.clone()
    Ly, n, KV, width = w.shape
    weights, kept = torch.zeros((Ly, n, KV, keep)), torch.full((Ly, n, KV, keep), -1, dtype=torch.int32)
    lists = w.cpu().tolist()
    for l in range(Ly):
        for s, L in enumerate(lengths):
            for h in range(KV):
                x = (lists[l][s][h] + [0.0] * L)[:L]
                old = L - min(recent, L)
                order = sorted(range(old), key=lambda j: (not math.isnan(x[j]), -x[j] if not math.isnan(x[j]) else 0, j))
                left = sorted(order[:max(0, min(L, keep) - (L - old))]) + list(range(old, L))
                source = [16 * tables[s][j // 16] + j % 16 for j in left]
                at = [16 * to[s][i // 16] + i % 16 for i in range(len(left))]
                for pages in (k, v):
                    pages[l, h, at] = pages[l, h, source]
                kept[l, s, h, :len(left)] = torch.tensor(left, dtype=torch.int32)
                weights[l, s, h, :len(left)] = torch.tensor([x[j] for j in left])
    return k, v, weights.cuda(), kept.cuda()


def weights_of(shape, seed, kind):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(shape, generator=g))
    if kind == "ties":
        w = torch.round(w)
    if kind == "alike":
        w = torch.ones(shape)
    if kind == "any":   # negative, both zeros, infinities, NaNs of both signs, subnormal numbers
        some = torch.tensor([0.0, -0.0, -1.0, math.inf, -math.inf, math.nan, 1e-45, -1e-45, 1.0, 1 + 2.0 ** -23])
        some = torch.cat([some, torch.tensor([-1], dtype=torch.int32).view(torch.float32)])
        w = some[torch.randint(0, len(some), shape, generator=g)]
    return w.cuda()


def _evict(lengths, KV, D, keep, recent, layers=2, kind="ties", width=None, seed=0):
    needed = [min(n, keep) for n in lengths]
    both, n = tables_of(lengths + needed, seed)
    tables, to = both[:len(lengths)], both[len(lengths):]
    k, v = rand((layers, KV, 16 * n, D), seed), rand((layers, KV, 16 * n, D), seed + 1)
    w = weights_of((layers, len(lengths), KV, max(lengths) if width is None else width), seed, kind)
    want = evicted(k, v, w, lengths, tables, to, keep, recent)
    e = PagedEviction(PagedSequences([0] * len(lengths), lengths, tables, KV, KV), keep, recent, to)
    one = k.clone(), v.clone()
    got = (k, v, *paged_evict(k, v, w, e))
    for a, b in zip(got[:2] + got[3:], want[:2] + want[3:]):
        assert torch.equal(a, b)
    assert torch.equal(got[2].nan_to_num(nan=-77.0), want[2].nan_to_num(nan=-77.0))
    for l in range(layers):   # layer by layer
        weights, kept = paged_evict(one[0][l], one[1][l], w[l], e)
        assert same(weights, got[2][l]) and torch.equal(kept, got[3][l])
    assert same(one[0], k) and same(one[1], v)
    assert e.lengths == needed


@pytest.mark.parametrize("kind", ["random", "ties", "alike", "any"])
@pytest.mark.parametrize("lengths,KV,D,keep,recent", [
    ([40], 1, 64, 16, 4),
    ([500, 512, 100, 1, 256, 257], 4, 64, 256, 64),
    ([300, 33], 2, 128, 47, 0),                # none for being new
    ([300, 20], 2, 96, 40, 40),                # all for being new
    ([70, 69], 3, 8, 69, 5),
    ([1000, 0, 3], 1, 72, 1, 1),
    ([1000, 0, 3], 1, 72, 1, 0),
    ([90], 1, 64, 400, 300),                   # more than there are
])
def test_evict(lengths, KV, D, keep, recent, kind):
    _evict(lengths, KV, D, keep, recent, kind=kind, seed=sum(lengths))


@pytest.mark.parametrize("kind", ["random", "ties", "any"])
@pytest.mark.parametrize("longest", [4096, 4097, 9001])
def test_evict_long(longest, kind):
    _evict([longest, longest // 2], 1, 64, longest // 3, 100, layers=1, kind=kind, seed=longest)


@pytest.mark.parametrize("kind", ["ties", "any"])
@pytest.mark.parametrize("D,keep,recent", [(64, 64, 8), (128, 100, 100), (72, 33, 0), (8, 1, 1)])
def test_evict_all_layers(D, keep, recent, kind):
    """Enough sequences, layers and heads for a workgroup each to choose and move."""
    _evict([100, 33, 0, 1, 64, 257, 300], 2, D, keep, recent, layers=40, kind=kind, seed=keep)
    _evict([700, 2048], 2, D, 3 * keep, recent, layers=128, kind=kind, seed=keep, width=500)


@pytest.mark.parametrize("width", [0, 1, 100, 1000])
def test_evict_with_weights_of_any_width(width):
    _evict([300, 120], 2, 64, 64, 8, width=width, seed=3)


def test_evict_to_nothing():
    _evict([40, 3], 2, 64, 0, 0, seed=4)


def test_evict_takes_any_strides_and_shared_sources():
    """Layers between keys and values of a pool, weights that are not contiguous, sources that sequences share; the old pages stay."""
    tables, n = tables_of([64, 40, 30, 30], 5)
    tables, to = [tables[0], tables[0][:2] + tables[1]], tables[2:]
    lengths, keep, recent = [64, 60], 30, 7
    pool = rand((3, 2, 2, 16 * n, 64), 1)
    w = weights_of((3, 2, 2, 128), 2, "random")[..., ::2]
    want = evicted(pool[:, 0], pool[:, 1], w, lengths, tables, to, keep, recent)
    e = PagedEviction(PagedSequences([1, 1], lengths, tables, 4, 2), keep, recent, to)
    weights, kept = paged_evict(pool[:, 0], pool[:, 1], w, e)
    assert same(pool[:, 0], want[0]) and same(pool[:, 1], want[1]) and same(weights, want[2]) and torch.equal(kept, want[3])


def test_evict_past_32_bit_offsets():
    n = 600000 // 16
    pool = torch.zeros((3, 16 * n, 1536), dtype=torch.bfloat16, device="cuda")
    k, v = pool[..., 1280:1408], pool[..., 1408:]
    table, to = [n - 2, n - 4, n - 6], [n - 1, n - 3]
    for p in table:
        k[:, 16 * p:16 * p + 16], v[:, 16 * p:16 * p + 16] = rand((3, 16, 128), p), rand((3, 16, 128), p + 1)
    w = weights_of((1, 3, 45), 1, "random")
    _, kept = paged_evict(k, v, w, PagedEviction(PagedSequences([0], [45], [table], 3, 3), 20, 4, [to]))
    for h in range(3):
        at = kept[0, h].long()
        for pages in (k, v):
            assert same(rows_of(pages, to, 20)[h], rows_of(pages, table, 45)[h, at])


def test_evict_refusals():
    tables, n = tables_of([40, 16], 1)
    k, v = rand((2, 16 * n, 64), 1), rand((2, 16 * n, 64), 2)
    s = PagedSequences([1], [40], tables[:1], 4, 2, longest=48)
    e, w = PagedEviction(s, 16, 4, tables[1:]), torch.zeros(1, 2, 40, device="cuda")
    for bad, match in (((k, v, w.double()), "float32"), ((k, v, w[0]), "float32"), ((k, v, w.cpu()), "float32"), ((k[None], v[None], w), "float32"),
                       ((k[:, :16], v[:, :16], w), "reach"), ((k, k[:1].expand(2, -1, -1), w), "overlap"), ((k[None].expand(2, -1, -1, -1), v[None].expand(2, -1, -1, -1), w), "overlap")):
        with pytest.raises(ValueError, match=match):
            paged_evict(*bad, e)
    s.update([41], tables[:1])
    with pytest.raises(ValueError, match="updated"):
        paged_evict(k, v, w, e)


def test_captured_appends_and_evictions():
    """A step's append and attention in a graph that goes on with the next steps, an eviction in another; replays beside eager calls."""
    n, longest = 40, 200
    order = torch.randperm(n, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [order[:13], order[13:26]]
    pool = rand((2, 2, 16 * n, 64), 1)
    sequences = PagedSequences([1, 20], [9, 30], tables, 4, 2, longest=longest)
    q, k, v = rand((21, 4, 64), 2), rand((21, 2, 64), 3), rand((21, 2, 64), 4)
    start = pool.clone()
    paged_append(k, v, pool[0], pool[1], sequences)
    w = paged_attention(q, pool[0], pool[1], sequences, weights=torch.zeros(2, 2, 0, device="cuda"))[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_append(k, v, pool[0], pool[1], sequences)
        out, counted = paged_attention(q, pool[0], pool[1], sequences, weights=w)
    for lengths in ([9, 30], [10, 50], [200, 199], [1, 20]):
        sequences.update(lengths, tables)
        pool.copy_(start)
        w.copy_(torch.rand_like(w))
        graph.replay()
        torch.cuda.synchronize()
        mine = start.clone()
        eager = PagedSequences([1, 20], lengths, tables, 4, 2, longest=longest)
        paged_append(k, v, mine[0], mine[1], eager)
        want = paged_attention(q, mine[0], mine[1], eager, weights=w)
        assert same(pool, mine) and same(out, want[0]) and same(counted, want[1])
    last = PagedSequences([0, 0], [200, 199], tables, 4, 2)
    e = PagedEviction(last, 60, 10, [order[26:30], order[30:34]])
    want, results = start.clone(), paged_evict(pool[0], pool[1], w, e)
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        got = paged_evict(pool[0], pool[1], w, e)
    for seed in range(3):
        pool.copy_(rand(pool.shape, seed))
        w.copy_(weights_of(w.shape, seed, "ties"))
        g2.replay()
        torch.cuda.synchronize()
        want.copy_(rand(pool.shape, seed))
        results = paged_evict(want[0], want[1], w, e)
        assert same(pool, want) and all(same(a, b) for a, b in zip(got, results))


# ---- together ----

def _model(layers, d, H, KV, dh, ff, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    mat = lambda *s: (torch.randn(s, generator=g) * s[0] ** -0.5).to(torch.bfloat16).cuda()  # noqa: E731
    return dict(emb=(torch.randn((vocab, d), generator=g)).to(torch.bfloat16).cuda(), layers=[
        dict(ln1=torch.ones(d, dtype=torch.bfloat16, device="cuda"), ln2=torch.ones(d, dtype=torch.bfloat16, device="cuda"), qkv=mat(d, (H + 2 * KV) * dh),
             o=mat(H * dh, d), gate_up=mat(d, 2 * ff), down=mat(ff, d)) for _ in range(layers)])


class _Server:
    """A model's layers over a pool: every step appends, attends, counts and, where a cache has become too long, evicts."""

    def __init__(self, m, H, KV, dh, n, pages):
        self.m, self.H, self.KV, self.dh, self.n = m, H, KV, dh, n
        self.freq = rotary_frequencies(dh)
        L = len(m["layers"])
        self.pool = PagePool(dict(n_layers=L, n_kv_heads=KV, d_head=dh, d_model=H * dh, n_heads=H), pages)
        self.free = list(range(pages))
        random.Random(0).shuffle(self.free)
        self.tables, self.lengths, self.position = [[] for _ in range(n)], [0] * n, [0] * n
        self.weights = [torch.zeros((n, KV, 0), device="cuda") for _ in range(L)]

    def step(self, tokens):
        """tokens: a list of each sequence's new ones; the hidden states after the last layer."""
        q_lens = [len(t) for t in tokens]
        at = [self.position[s] + i for s in range(self.n) for i in range(q_lens[s])]
        for s in range(self.n):
            self.lengths[s] += q_lens[s]
            self.position[s] += q_lens[s]
            while 16 * len(self.tables[s]) < self.lengths[s]:
                self.tables[s].append(self.free.pop())
        seqs = PagedSequences(q_lens, self.lengths, self.tables, self.H, self.KV)
        positions = torch.tensor(at, dtype=torch.int32, device="cuda")
        h = self.m["emb"][torch.tensor([t for x in tokens for t in x], device="cuda")]
        res = torch.zeros_like(h)
        for l, p in enumerate(self.m["layers"]):
            x, res = rms_norm(h, p["ln1"], res)
            qkv = (x @ p["qkv"]).view(len(at), self.H + 2 * self.KV, self.dh)
            q, k = rotary(qkv[:, :self.H], qkv[:, self.H:self.H + self.KV], self.freq, positions)
            kp, vp = self.pool.view()[l]
            paged_append(k, qkv[:, self.H + self.KV:], kp, vp, seqs)
            a, self.weights[l] = paged_attention(q, kp, vp, seqs, weights=self.weights[l])
            x, res = rms_norm(a.reshape(len(at), -1) @ p["o"], p["ln2"], res)
            gate, up = (x @ p["gate_up"]).chunk(2, -1)
            h = swiglu(gate, up) @ p["down"]
        return res + h

    def evict(self, keep, recent):
        seqs = PagedSequences([0] * self.n, self.lengths, self.tables, self.H, self.KV)
        to = [[self.free.pop() for _ in range(-(-min(n, keep) // 16))] for n in self.lengths]
        e = PagedEviction(seqs, keep, recent, to)
        view = self.pool.view()
        w, kept = paged_evict(view[:, 0], view[:, 1], torch.stack(self.weights), e)
        self.weights = list(w)
        for t in self.tables:
            self.free += t
        self.tables, self.lengths = to, e.lengths
        return kept


def test_a_model_over_pages():
    """Prompts in chunks, then single tokens, mixed in one step: the states of a forward pass over the whole sequences with the dense
    attention.  Both round the same products to bf16, but not the same probabilities: those are off by 2^-8 of a value once in each
    layer, and so are the bf16 results that follow from them (each of four roundings of a layer may fall on the other side, 2^-7
    of a value); the relative error of the whole state then stays below 4 layers x 5 roundings x 2^-8."""
    H, KV, dh, ff, L = 8, 2, 64, 512, 4
    m = _model(L, H * dh, H, KV, dh, ff, 100, 1)
    r = random.Random(1)
    tokens = [[r.randrange(100) for _ in range(n)] for n in (150, 37, 90)]
    server, done, states = _Server(m, H, KV, dh, 3, 64), [0, 0, 0], [[], [], []]
    for step in ([64, 20, 0], [64, 1, 50], [1, 1, 37], [1, 1, 1], [1, 1, 1], [1, 1, 0], [18, 12, 1]):
        out = server.step([tokens[s][done[s]:done[s] + n] for s, n in enumerate(step)])
        for s, n in enumerate(step):
            states[s].append(out[sum(step[:s]):sum(step[:s]) + n])
            done[s] += n
    assert done == [len(t) for t in tokens]
    for s, t in enumerate(tokens):
        h = m["emb"][torch.tensor(t, device="cuda")]
        res = torch.zeros_like(h)
        for p in m["layers"]:
            x, res = rms_norm(h, p["ln1"], res)
            qkv = (x @ p["qkv"]).view(len(t), H + 2 * KV, dh)
            q, k = rotary(qkv[:, :H], qkv[:, H:H + KV], server.freq)
            a = attention(q, k, qkv[:, H + KV:])
            x, res = rms_norm(a.reshape(len(t), -1) @ p["o"], p["ln2"], res)
            gate, up = (x @ p["gate_up"]).chunk(2, -1)
            h = swiglu(gate, up) @ p["down"]
        want, got = (res + h).double(), torch.cat(states[s]).double()
        assert float((got - want).norm() / want.norm()) < L * 5 * 2.0 ** -8
    for l in range(L):   # every new token's probabilities add to one for each head
        for s, n in enumerate(server.lengths):
            total = server.weights[l][s].double().sum(-1)
            assert torch.allclose(total, torch.full_like(total, n * H // KV), rtol=2.0 ** -11)


def test_eviction_between_steps():
    """After an eviction the cache is what was kept: attention over the new pages is attention over the kept rows, in their order, and
    the counting goes on from their weights; keeping everything changes nothing."""
    H, KV, dh = 4, 2, 64
    m = _model(2, H * dh, H, KV, dh, 256, 100, 2)
    r = random.Random(2)
    server = _Server(m, H, KV, dh, 2, 200)
    server.step([[r.randrange(100) for _ in range(n)] for n in (200, 40)])
    server.step([[3], [4]])
    before = [rows_of(server.pool.view()[0, 0], t, n) for t, n in zip(server.tables, server.lengths)]
    weights = server.weights[0].clone()
    kept = server.evict(64, 16)
    assert server.lengths == [64, 41] and kept.shape == (2, 2, KV, 64)
    for s, n in enumerate(server.lengths):
        for h in range(KV):
            at = kept[0, s, h, :n].long()
            assert at.tolist() == sorted(at.tolist()) and (kept[0, s, h, n:] == -1).all()
            assert same(rows_of(server.pool.view()[0, 0], server.tables[s], n)[h], before[s][h, at])
            assert same(server.weights[0][s, h, :n], weights[s, h, at])
    server.step([[5] * 3, [6]])
    assert server.lengths == [67, 42] and server.position == [204, 42]
    for s, n in enumerate(server.lengths):
        new = 3 - 2 * s
        total = server.weights[0][s].double().sum(-1)
        held = torch.stack([weights[s, h, kept[0, s, h, :n - new].long()].double().sum() for h in range(KV)])
        assert torch.allclose(total, held + new * H // KV, rtol=2.0 ** -11)
