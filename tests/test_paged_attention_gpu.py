"""Attention over pages on the GPU (msd_paged_attn) against the formulas in 64 bits, with what each position receives.

Tolerances, element by element, with u = 2^-8 (half a bf16 step, relative) and e = 2^-12 for what 32 bits leave in a
probability: a score's 128 products of up to a few units add to ~2^-24 * 128 * 16 = 2^-13 at most, times ln 2 in the
exponent, and the exponential and the sums of up to 4096 terms stay below that.
  out: P is rounded to bf16 as an operand, the result once:  (u + e) sum P |v| + u |out|
  weights: P is not rounded; sums of up to 4096 of them, each addition 2^-24, are another e:  2 e sum P + 2^-24 |weights|
"""
import math

import pytest
import torch

from transformer_amd.paged_attention import PagedSequences, paged_attention

pytestmark = pytest.mark.gpu
U, E = 2.0 ** -8, 2.0 ** -12


def rand(shape, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(torch.bfloat16).cuda()


def tables_of(lengths, seed, spare=3):
    """Pages of each sequence in no order, and how many pages there are."""
    used = [-(-n // 16) for n in lengths]
    free = torch.randperm(sum(used) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    return [[free.pop() for _ in range(n)] for n in used], sum(used) + spare


def rows_of(pages, table, n):
    """A sequence's rows (kv heads, n, d)."""
    at = torch.tensor([16 * table[j // 16] + j % 16 for j in range(n)], dtype=torch.long, device=pages.device)
    return pages[:, at]


def reference(q, k_pages, v_pages, q_lens, lengths, tables, starts, scale, weights, width):
    """((out, weights), their tolerances) in 64 bits; rows of no sequence are zeros."""
    H, KV = q.shape[1], k_pages.shape[0]
    g = H // KV
    out, t_out = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    w = torch.zeros((len(q_lens), KV, width), dtype=torch.float64, device=q.device)
    t_w = torch.zeros_like(w)
    for s, (n, L) in enumerate(zip(q_lens, lengths)):
        if weights is not None:
            have = min(L - n, weights.shape[2])
            w[s, :, :have] = weights[s, :, :have].double()
        k, v = rows_of(k_pages, tables[s], L).double(), rows_of(v_pages, tables[s], L).double()
        if not n:
            continue
        i = slice(starts[s], starts[s] + n)
        see = torch.arange(L, device=q.device)[None] <= torch.arange(L - n, L, device=q.device)[:, None]
        for h in range(H):
            p = torch.softmax((q[i, h].double() @ k[h // g].T * scale).masked_fill(~see, -math.inf), -1)
            out[i, h] = p @ v[h // g]
            t_out[i, h] = (U + E) * (p @ v[h // g].abs()) + U * out[i, h].abs()
            w[s, h // g, :L] += p.sum(0)
            t_w[s, h // g, :L] += 2 * E * p.sum(0)
    return (out, w), (t_out, t_w + 2.0 ** -24 * w.abs())


def near(x, ref, tol, name):
    x, over = x.double(), (x.double() - ref).abs() - tol - 1e-30
    assert torch.isfinite(x).all(), name
    if over.numel():
        assert float(over.max()) <= 0, (name, int(over.argmax()), float(x.reshape(-1)[over.argmax()]), float(ref.reshape(-1)[over.argmax()]))


def check(q_lens, lengths, H, KV, D, seed=0, scale=None, weights=True, starts=None, rows=None, width=None, longest=None):
    tables, n = tables_of(lengths, seed)
    if starts is None:
        starts = [sum(q_lens[:s]) for s in range(len(q_lens))]
    rows = sum(q_lens) if rows is None else rows
    q = rand((rows, H, D), seed, 1.5)
    k, v = rand((KV, 16 * n, D), seed + 1), rand((KV, 16 * n, D), seed + 2)
    sequences = PagedSequences(q_lens, lengths, tables, H, KV, q_starts=starts, longest=longest)
    old = None
    if weights:
        old = torch.rand((len(q_lens), KV, max(lengths, default=0) if width is None else width), generator=torch.Generator().manual_seed(seed)).cuda()
    ref, tol = reference(q, k, v, q_lens, lengths, tables, starts, scale or D ** -0.5, old, sequences.longest)
    out = paged_attention(q, k, v, sequences, scale=scale)
    near(out, ref[0], tol[0], "out")
    assert out.is_contiguous() and out.dtype == torch.bfloat16
    if weights:
        counted, w = paged_attention(q, k, v, sequences, scale=scale, weights=old)   # (may split the keys where the other does not)
        near(counted, ref[0], tol[0], "out")
        assert w.dtype == torch.float32
        near(w, ref[1], tol[1], "weights")
        again = paged_attention(q, k, v, sequences, scale=scale, weights=old)
        assert torch.equal(again[0], counted) and torch.equal(again[1], w)
    assert torch.equal(paged_attention(q, k, v, sequences, scale=scale), out)
    return sequences


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_one_token(n, D):
    check([1], [n], 4, 2, D, seed=n)


@pytest.mark.parametrize("q_lens,lengths,H,KV,D", [
    ([1, 1, 1], [5, 300, 64], 1, 1, 64),
    ([1] * 5, [2000, 16, 1, 777, 2048], 16, 4, 64),
    ([1] * 4, [1500, 33, 900, 16], 32, 4, 128),           # eight heads of a group
    ([1, 1], [700, 90], 32, 1, 128),                      # thirty-two: as many rows as the few have
    ([1, 1], [700, 90], 33, 1, 64),                       # thirty-three: a chunk's kernel
    ([1, 3], [700, 90], 80, 2, 32),
    ([4, 2, 1, 3], [400, 2, 1, 30], 8, 2, 128),           # drafts
    ([8, 7], [100, 300], 4, 1, 64),
    ([1, 1, 1], [40, 50, 60], 3, 3, 8),
    ([1, 2], [100, 130], 6, 2, 96),
    ([2, 1], [70, 300], 10, 2, 40),
    ([1, 5], [200, 37], 2, 1, 72),
    ([3, 1], [33, 500], 4, 4, 120),
])
def test_few_rows(q_lens, lengths, H, KV, D):
    check(q_lens, lengths, H, KV, D, seed=sum(lengths))


@pytest.mark.parametrize("q_lens,lengths,H,KV,D", [
    ([64], [64], 1, 1, 64),
    ([33, 64, 65], [33, 64, 65], 4, 2, 64),
    ([100], [1000], 16, 4, 128),
    ([129, 128], [129, 500], 4, 4, 64),
    ([300, 50], [300, 900], 8, 2, 96),
    ([77], [190], 4, 2, 40),
    ([200], [201], 2, 1, 8),
    ([90, 31], [90, 47], 2, 1, 72),
    ([63], [128], 7, 1, 128),
    ([40, 40], [40, 41], 3, 1, 120),
    ([512], [2049], 2, 2, 32),
    ([11], [4096], 12, 3, 128),
    ([400], [3500], 4, 1, 64),                            # few tiles of many keys: split and joined
])
def test_chunks(q_lens, lengths, H, KV, D):
    check(q_lens, lengths, H, KV, D, seed=sum(lengths))


def test_a_mixed_step():
    """Single tokens, drafts, chunks and sequences without new tokens or without any, in rows that are in another order."""
    q_lens, lengths = [1, 0, 200, 5, 0, 33, 1, 64], [700, 300, 450, 5, 0, 900, 1, 64]
    starts = [303, 0, 40, 1, 7, 260, 0, 310]
    s = check(q_lens, lengths, 8, 2, 64, seed=9, starts=starts, rows=400)
    assert s.q_count == 304
    check(q_lens, lengths, 6, 6, 128, seed=10, starts=starts, rows=380, longest=1500)


def test_many_sequences():
    lengths = [1 + (37 * i) % 400 for i in range(300)]
    check([min(n, 1 + i % 2) for i, n in enumerate(lengths)], lengths, 2, 1, 64, seed=11)


@pytest.mark.parametrize("q_lens,lengths,H,KV,D,longest", [
    ([1] * 6, [511, 512, 513, 1, 32, 33], 8, 2, 64, None), ([1] * 4, [512, 480, 256, 257], 8, 2, 64, None), ([1, 1, 1], [1023, 1024, 700], 8, 2, 64, None),
    ([1, 1], [1025, 1024], 8, 2, 64, None), ([1] * 32, [1024 - 29 * i for i in range(32)], 8, 2, 32, None), ([1] * 35, [900 - 25 * i for i in range(35)], 8, 2, 96, None),
    ([1, 2, 4], [512, 100, 511], 8, 2, 128, None), ([4, 1], [1000, 3], 32, 4, 64, None), ([5, 1], [300, 3], 32, 4, 64, None), ([17, 1], [300, 20], 1, 1, 128, None),
    ([16, 9], [16, 512], 2, 2, 128, None), ([0, 3, 0, 1], [40, 300, 0, 511], 6, 2, 80, None), ([32], [32], 1, 1, 8, None), ([1] * 128, [5 * i + 1 for i in range(128)], 4, 2, 72, None),
    ([1] * 129, [3 * i + 1 for i in range(129)], 4, 2, 64, None), ([1, 0, 2], [50, 33, 260], 8, 2, 64, 512), ([1, 0, 2], [50, 33, 260], 8, 2, 64, 1000), ([2] * 40, [7 * i + 2 for i in range(40)], 4, 2, 128, 1024),
])
def test_few_short_sequences(q_lens, lengths, H, KV, D, longest):
    """Around what a sequence by one workgroup takes: lengths, rows of a group, workgroups, sequences without new tokens."""
    check(q_lens, lengths, H, KV, D, seed=9, longest=longest, width=200)
    check(q_lens, lengths, H, KV, D, seed=10, longest=longest, weights=False)


@pytest.mark.parametrize("width", [0, 1, 30, 63, 5000])
def test_weights_of_any_width(width):
    check([1, 40, 2], [64, 300, 40], 4, 2, 64, seed=12, width=width)


def test_scales():
    check([2, 40], [100, 300], 4, 2, 64, seed=13, scale=0.01)
    check([2, 40], [100, 300], 4, 2, 64, seed=14, scale=2.0 ** -60)


@pytest.mark.parametrize("D", [48, 128])
def test_operands_of_other_strides(D):
    """Queries as part of a projection, pages of (position, head) order, with room between heads and at the side of each, layers
    between the keys and the values of one pool, and queries that have to be copied."""
    q_lens, lengths, H, KV = [1, 50, 3], [200, 130, 3], 4, 2
    tables, n = tables_of(lengths, 1)
    sequences = PagedSequences(q_lens, lengths, tables, H, KV)
    q, pool = rand((54, H + 2 * KV, D), 1, 1.5), rand((3, 2, KV, 16 * n, D), 2)
    want = paged_attention(q[:, :H].contiguous(), pool[1, 0].contiguous(), pool[1, 1].contiguous(), sequences)
    ref, tol = reference(q[:, :H], pool[1, 0], pool[1, 1], q_lens, lengths, tables, [0, 1, 51], D ** -0.5, None, 200)
    near(want, ref[0], tol[0], "out")
    assert torch.equal(paged_attention(q[:, :H], pool[1, 0], pool[1, 1], sequences), want)
    turned = pool.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(paged_attention(q[:, :H], turned[1, 0], turned[1, 1], sequences), want)
    wide = torch.full((KV, 16 * n, D + 24), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[..., 8:8 + D] = pool[1, 0]
    assert torch.equal(paged_attention(q[:, :H], wide[..., 8:8 + D], turned[1, 1], sequences), want)
    odd = torch.zeros((54, H, D + 1), dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = q[:, :H]
    assert torch.equal(paged_attention(odd[..., 1:], pool[1, 0], pool[1, 1], sequences), want)
    assert torch.equal(paged_attention(q[:1, :1].expand(54, H, D), pool[1, 0], pool[1, 1], sequences),
                       paged_attention(q[:1, :1].repeat(54, H, 1), pool[1, 0], pool[1, 1], sequences))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_lies_behind_a_length_is_not_read(bad):
    """Not finite everywhere but in the sequences' positions: pages of nobody, slots behind a length in the last page."""
    q_lens, lengths = [1, 3, 70, 1], [33, 19, 90, 300]
    tables, n = tables_of(lengths, 5)
    q, k, v = rand((75, 4, 64), 1), rand((2, 16 * n, 64), 2), rand((2, 16 * n, 64), 3)
    sequences = PagedSequences(q_lens, lengths, tables, 4, 2)
    want = paged_attention(q, k, v, sequences, weights=torch.zeros(4, 2, 0, device="cuda"))
    mine = torch.zeros(16 * n, dtype=torch.bool)
    for t, L in zip(tables, lengths):
        mine[[16 * t[j // 16] + j % 16 for j in range(L)]] = True
    k[:, ~mine.cuda()] = v[:, ~mine.cuda()] = bad
    got = paged_attention(q, k, v, sequences, weights=torch.full((4, 2, 0), math.nan, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.isfinite(got[1]).all()


def test_values_that_are_not_finite():
    """In a row that a query sees they reach it, and not the queries of other sequences."""
    q_lens, lengths = [1, 1, 40], [100, 300, 200]
    tables, n = tables_of(lengths, 6)
    q, k, v = rand((42, 2, 64), 1), rand((2, 16 * n, 64), 2), rand((2, 16 * n, 64), 3)
    sequences = PagedSequences(q_lens, lengths, tables, 2, 2)
    want = paged_attention(q, k, v, sequences)
    v[0, 16 * tables[1][3] + 5] = math.nan
    k[1, 16 * tables[2][0] + 1] = math.nan
    got = paged_attention(q, k, v, sequences)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, 1], want[1, 1]) and torch.equal(got[2:, 0], want[2:, 0])
    assert got[1, 0].isnan().all() and got[2:, 1].isnan().all()


def test_shared_pages():
    """A prompt's pages read by several sequences."""
    tables, n = tables_of([160, 33, 50, 20], 7)
    prefix = tables[0]
    tables = [prefix, prefix + tables[1], prefix + tables[2], prefix[:4] + tables[3]]
    q_lens, lengths = [1, 20, 1, 40], [160, 193, 210, 84]
    q, k, v = rand((62, 8, 64), 1, 1.5), rand((2, 16 * n, 64), 2), rand((2, 16 * n, 64), 3)
    old = torch.rand((4, 2, 210)).cuda()
    got = paged_attention(q, k, v, PagedSequences(q_lens, lengths, tables, 8, 2), weights=old)
    ref, tol = reference(q, k, v, q_lens, lengths, tables, [0, 1, 21, 22], 0.125, old, 210)
    near(got[0], ref[0], tol[0], "out")
    near(got[1], ref[1], tol[1], "weights")


def test_a_pool_past_32_bit_offsets():
    """Pages beyond 2^32 bytes and 2^31 elements, of a head beyond both, with weights and with a chunk."""
    KV, n = 3, 600000 // 16   # 3 x 600000 x 1536: 2.8e9 elements
    pool = torch.empty((KV, 16 * n, 1536), dtype=torch.bfloat16, device="cuda")
    k, v = pool[..., 1280:1408], pool[..., 1408:]
    q_lens, lengths = [1, 60], [130, 200]
    tables = [[n - 1 - 2 * i for i in range(9)], [n - 2 - 2 * i for i in range(13)]]
    for t in tables:
        for p in t:
            k[:, 16 * p:16 * p + 16] = rand((KV, 16, 128), p)
            v[:, 16 * p:16 * p + 16] = rand((KV, 16, 128), p + 1)
    q = rand((61, 2 * KV, 128), 3, 1.5)
    old = torch.zeros(2, KV, 0, device="cuda")
    got = paged_attention(q, k, v, PagedSequences(q_lens, lengths, tables, 2 * KV, KV), weights=old)
    ref, tol = reference(q, k, v, q_lens, lengths, tables, [0, 1], 128 ** -0.5, None, 200)
    near(got[0], ref[0], tol[0], "out")
    near(got[1], ref[1], tol[1], "weights")


def test_long_caches():
    """One sequence of many keys, whose parts are joined; and its chunk."""
    check([1], [40000], 8, 2, 128, seed=20)
    check([1, 1], [20001, 9], 4, 4, 64, seed=21)
    check([70], [9000], 4, 1, 128, seed=22)


@pytest.mark.parametrize("last", [40, 4])
def test_a_captured_step_goes_on(last):
    """A graph over sequences with room: lengths and pages of the next steps, replayed and beside eager calls on the same object;
    two graphs on two streams share it."""
    q_lens, steps = [1, 2, last], [[60, 700, 90], [61, 702, 130], [62, 1000, 400], [1, 2, 40], [1000, 1000, 1000]]
    n = 200
    order = torch.randperm(n, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [order[i * 66:i * 66 + 66] for i in range(3)]
    q, k, v = rand((3 + last, 8, 64), 1, 1.5), rand((2, 16 * n, 64), 2), rand((2, 16 * n, 64), 3)
    old = torch.rand((3, 2, 1000), generator=torch.Generator().manual_seed(3)).cuda()
    sequences = PagedSequences(q_lens, steps[0], tables, 8, 2, longest=1000)
    paged_attention(q, k, v, sequences, weights=old)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged_attention(q, k, v, sequences, weights=old))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for lengths in steps + steps:
        sequences.update(lengths, tables)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        eager = paged_attention(q, k, v, sequences, weights=old)
        ref, tol = reference(q, k, v, q_lens, lengths, tables, [0, 1, 3], 0.125, old, 1000)
        for out in (*outs, eager):
            near(out[0], ref[0], tol[0], "out")
            near(out[1], ref[1], tol[1], "weights")
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_two_streams():
    """Calls on streams other than the sequences' own, which are given up while the calls may still run."""
    want, got = [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        q_lens, lengths = [1, 1, 50], [3000 + i, 100, 700]
        tables, n = tables_of(lengths, i)
        q, k, v = rand((52, 8, 128), 1, 1.5), rand((2, 16 * n, 128), 2), rand((2, 16 * n, 128), 3)
        s = PagedSequences(q_lens, lengths, tables, 8, 2)
        want.append(paged_attention(q, k, v, s))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[i % 2]):
            got.append(paged_attention(q, k, v, s))
        del s
        torch.zeros(4096, dtype=torch.int32, device="cuda").fill_(-1)
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("q_lens,lengths", [([1, 60], [300, 200]), ([1, 3], [300, 200])])
def test_device_words_that_have_been_overwritten(q_lens, lengths):
    """Page numbers outside the pool read as rows of zeros; jobs that leave their limits end."""
    tables, n = tables_of(lengths, 3)
    q, k, v = rand((sum(q_lens), 4, 64), 1), rand((2, 16 * n, 64), 2), rand((2, 16 * n, 64), 3)
    old = torch.rand((2, 2, 300)).cuda()
    s = PagedSequences(q_lens, lengths, tables, 4, 2)
    spare = next(p for p in range(n) if all(p not in t for t in tables))
    k[:, 16 * spare:16 * spare + 16] = v[:, 16 * spare:16 * spare + 16] = 0
    want = paged_attention(q, k, v, PagedSequences(q_lens, lengths, [[spare if i in (2, 9) else p for i, p in enumerate(t)] for t in tables], 4, 2), weights=old)
    at = s.table.numel() - 2 * (s.host[5].item())   # the tables are the last words
    for t in range(2):
        s.table[at + t * s.host[5] + 2], s.table[at + t * s.host[5] + 9] = -5, 2 ** 30
    got = paged_attention(q, k, v, s, weights=old)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    s.table[40:at] = 2 ** 30
    paged_attention(q, k, v, s, weights=old)
    s.table[40:at] = -2 ** 31
    paged_attention(q, k, v, s, weights=old)
    torch.cuda.synchronize()
    assert torch.equal(paged_attention(q, k, v, PagedSequences(q_lens, lengths, tables, 4, 2)), paged_attention(q, k, v, PagedSequences(q_lens, lengths, tables, 4, 2)))


def test_nothing_to_do():
    k = torch.zeros(2, 0, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    s = PagedSequences([], [], [], 4, 2)
    assert paged_attention(q, k, k, s).shape == (0, 4, 64)
    out, w = paged_attention(rand((3, 4, 64), 1), k, k, PagedSequences([0, 0], [0, 0], [[], []], 4, 2, longest=20), weights=torch.ones(2, 2, 5, device="cuda"))
    assert out.shape == (3, 4, 64) and not out.any() and w.shape == (2, 2, 20) and not w.any()
    out, w = paged_attention(q, k, k, s, weights=torch.ones(0, 2, 5, device="cuda"))
    assert w.shape == (0, 2, 0)
