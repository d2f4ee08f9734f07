"""Attention forward and backward on the GPU (msd_attn_forward / msd_attn_backward) against the formulas in 64 bits.

Tolerances, element by element, with u = 2^-8 (half a bf16 step, relative) and e = 2^-12 for what 32 bits leave in a
probability: a score's 128 products of up to a few units add to ~2^-24 * 128 * 16 = 2^-13 at most, times ln 2 in the
exponent, and the exponential and the sums of up to 4096 terms stay below that.
  out: P is rounded to bf16 as an operand, the result once:  (u + e) sum P |v| + u |out|
  dv:  likewise                                              (u + e) sum P |dout| + u |dv|
  dS = P (dP - D): D is formed from the rounded out, so it is off by E = sum |dout| tol(out); dS is rounded as an operand:
       t = P E + (u + 2 e) |dS| + e P sum_d |dout| |v|;      dq: scale sum t |k| + u |dq|,  dk: scale sum t |q| + u |dk|
"""
import math

import pytest
import torch

from transformer_amd.attention import Sequences, attention

pytestmark = pytest.mark.gpu
U, E = 2.0 ** -8, 2.0 ** -12


def _one(q, k, v, do, causal, scale):
    """(results, tolerances) of out, dq, dk, dv for one sequence and head group: q, do (g, Tq, D), k, v (Tk, D)."""
    g, tq, D = q.shape
    tk = k.shape[0]
    q, do = q.reshape(-1, D), do.reshape(-1, D)
    s = q @ k.T * scale
    if causal:
        see = torch.arange(tk, device=q.device)[None] <= torch.arange(tk - tq, tk, device=q.device)[:, None]
        s = s.masked_fill(~see.repeat(g, 1), -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if tk else s
    out = p @ v
    t_out = (U + E) * (p @ v.abs()) + U * out.abs()
    dv = p.T @ do
    t_dv = (U + E) * (p.T @ do.abs()) + U * dv.abs()
    ds = p * (do @ v.T - (do * out).sum(-1, keepdim=True))
    t = p * (do.abs() * t_out).sum(-1, keepdim=True) + (U + 2 * E) * ds.abs() + E * p * (do.abs() @ v.abs().T)
    dq, dk = scale * (ds @ k), scale * (ds.T @ q)
    t_dq, t_dk = scale * (t @ k.abs()) + U * dq.abs(), scale * (t.T @ q.abs()) + U * dk.abs()
    back = [x.reshape(g, tq, D) for x in (out, dq, t_out, t_dq)]
    return (back[0], back[1], dk, dv), (back[2], back[3], t_dk, t_dv)


def _reference(q, k, v, do, causal, scale, ranges):
    """The same over flat tensors (rows, heads, D) and (q0, nq, k0, nk) ranges; rows of none are zeros."""
    got = [torch.zeros(x.shape, dtype=torch.float64, device=q.device) for x in (q, q, k, v)]
    tol = [torch.zeros_like(x) for x in got]
    g = q.shape[1] // k.shape[1]
    for q0, nq, k0, nk in ranges:
        for h in range(k.shape[1]):
            i, j, hs = slice(q0, q0 + nq), slice(k0, k0 + nk), slice(h * g, h * g + g)
            a, b = _one(*(x.double().transpose(0, 1).contiguous() for x in (q[i, hs],)),
                        k[j, h].double(), v[j, h].double(), do[i, hs].double().transpose(0, 1).contiguous(), causal, scale)
            for out, part in ((got, a), (tol, b)):
                out[0][i, hs], out[1][i, hs] = part[0].transpose(0, 1), part[1].transpose(0, 1)
                out[2][j, h], out[3][j, h] = part[2], part[3]
    return got, tol


def _rand(shape, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(torch.bfloat16).cuda()


def _grads(q, k, v, do, **kw):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = attention(*leaves, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, do))


def _check(got, ref, tol):
    for name, x, r, t in zip(("out", "dq", "dk", "dv"), got, ref, tol):
        x, r, t = x.double().reshape(-1), r.reshape(-1), t.reshape(-1)
        assert torch.isfinite(x).all(), name
        over = (x - r).abs() - t - 1e-30
        if over.numel():
            assert float(over.max()) <= 0, (name, int(over.argmax()), float(x[over.argmax()]), float(r[over.argmax()]))


def _dense(B, tq, tk, H, KV, D, causal, seed=0, scale=None):
    q, do = _rand((B, tq, H, D), seed, 1.5), _rand((B, tq, H, D), seed + 1, 0.3)
    k, v = _rand((B, tk, KV, D), seed + 2), _rand((B, tk, KV, D), seed + 3)
    got = _grads(q, k, v, do, causal=causal, scale=scale)
    ranges = [(b * tq, tq, b * tk, tk) for b in range(B)]
    ref, tol = _reference(*(x.flatten(0, 1) for x in (q, k, v, do)), causal, scale or D ** -0.5, ranges)
    _check(got, ref, tol)
    assert torch.equal(got[0], attention(q, k, v, causal=causal, scale=scale))   # the call without gradients


@pytest.mark.parametrize("B,tq,tk,H,KV,D,causal", [
    (1, 1, 1, 1, 1, 64, True),
    (2, 63, 63, 4, 2, 64, True),
    (1, 64, 64, 1, 1, 128, True),
    (2, 65, 65, 6, 2, 64, True),          # three heads of a group
    (1, 200, 200, 7, 1, 128, True),       # seven
    (3, 128, 128, 4, 4, 32, False),
    (1, 129, 257, 4, 4, 96, False),
    (2, 100, 37, 2, 1, 64, False),
    (1, 130, 130, 2, 2, 8, True),
    (1, 77, 190, 4, 2, 40, True),
    (1, 90, 90, 2, 1, 72, True),
    (2, 33, 70, 2, 1, 120, True),
    (2, 300, 300, 8, 2, 80, True),
])
def test_shapes(B, tq, tk, H, KV, D, causal):
    _dense(B, tq, tk, H, KV, D, causal, seed=B + tq)


@pytest.mark.parametrize("B,H,KV,D", [(8, 32, 16, 64), (8, 32, 16, 128)])
def test_workgroups_of_four_waves(B, H, KV, D):
    """Enough rows for 128-row workgroups without splits, with ragged ends."""
    _dense(B, 333, 333, H, KV, D, True, seed=5)


def test_306m_heads():
    _dense(8, 512, 512, 16, 4, 64, True, seed=6)


@pytest.mark.parametrize("tq,tk", [(1, 2000), (1, 64), (1, 65), (3, 4096), (4, 3)])
@pytest.mark.parametrize("D", [64, 128])
def test_few_queries_over_many_keys(tq, tk, D):
    """Split over the keys and joined; more queries than keys."""
    _dense(2, tq, tk, 16, 4, D, True, seed=tk)


@pytest.mark.parametrize("tq,tk", [(70, 5), (200, 64), (64, 1), (300, 170)])
def test_rows_that_see_nothing(tq, tk):
    """More queries than keys under the causal mask: the first tq - tk rows are zeros and give no gradient."""
    q, do, k, v = (_rand((1, n, 4, 64), i) for i, n in enumerate((tq, tq, tk, tk)))
    got = _grads(q, k, v, do)
    assert not got[0][:, :tq - tk].any() and not got[1][:, :tq - tk].any()
    ref, tol = _reference(q[0], k[0], v[0], do[0], True, 64 ** -0.5, [(0, tq, 0, tk)])
    _check(got, ref, tol)


@pytest.mark.parametrize("tq,tk", [(0, 5), (5, 0), (0, 0)])
def test_no_rows(tq, tk):
    q, k, v, do = (_rand((2, n, 4, 64), 1) for n in (tq, tk, tk, tq))
    got = _grads(q, k, v, do, causal=False)
    assert [tuple(x.shape) for x in got] == [(2, tq, 4, 64)] * 2 + [(2, tk, 4, 64)] * 2
    assert all(not x.any() for x in got)


@pytest.mark.parametrize("spread,scale", [(20.0, None), (1.0, 4.0), (1e-3, None), (1.0, 1e-6)])
def test_peaked_and_flat_scores(spread, scale):
    """Scores in the hundreds: one key takes all (the 32-bit error of a score of 400 is 2^-15, inside e); and nearly
    equal ones."""
    q, do = _rand((2, 150, 4, 64), 1, spread), _rand((2, 150, 4, 64), 2)
    k, v = _rand((2, 150, 2, 64), 3, 0.05 if scale == 4.0 else 1.0), _rand((2, 150, 2, 64), 4)
    got = _grads(q, k, v, do, scale=scale)
    ref, tol = _reference(*(x.flatten(0, 1) for x in (q, k, v, do)), True, scale or 0.125,
                          [(b * 150, 150, b * 150, 150) for b in range(2)])
    _check(got, ref, tol)


LENS = [5, 0, 130, 1, 64, 300, 17]


@pytest.mark.parametrize("D,H,KV", [(64, 4, 2), (128, 3, 1)])
@pytest.mark.parametrize("tail", [0, 9])
def test_packed_sequences(D, H, KV, tail):
    """Sequences one behind the other, an empty one among them; what lies behind the last is not read (NaN) and has
    zero outputs and gradients."""
    n = sum(LENS) + tail
    q, k, v, do = (_rand((n, h, D), i) for i, h in enumerate((H, KV, KV, H)))
    starts = [sum(LENS[:i]) for i in range(len(LENS))]
    ranges = [(a, m, a, m) for a, m in zip(starts, LENS)]
    ref, tol = _reference(q, k, v, do, True, D ** -0.5, ranges)
    for x in (q, k, v, do):
        x[n - tail:] = math.nan if tail else 0
    got = _grads(q, k, v, do, sequences=Sequences(LENS))
    _check(got, ref, tol)
    assert all(not x[n - tail:].any() for x in got)


def test_padded_batch():
    """A padded batch as its flat view: the padding holds NaN and is neither read nor given gradients."""
    B, T, lens = 5, 150, [150, 1, 0, 77, 128]
    q, k, v, do = (_rand((B * T, h, 64), i) for i, h in enumerate((4, 2, 2, 4)))
    starts = range(0, B * T, T)
    ref, tol = _reference(q, k, v, do, True, 0.125, [(a, n, a, n) for a, n in zip(starts, lens)])
    for a, n in zip(starts, lens):
        for x in (q, k, v, do):
            x[a + n:a + T] = math.nan
    got = _grads(q, k, v, do, sequences=Sequences(lens, q_starts=starts))
    _check(got, ref, tol)


def test_sequences_of_their_own_keys():
    """Cross-attention of packed queries over packed keys of other lengths, out of order and with gaps."""
    ql, kl, qs, ks = [30, 64, 7], [100, 3, 250], [10, 100, 50], [0, 400, 120]
    q, k, v, do = (_rand((n, h, 64), i) for i, (n, h) in enumerate(((170, 4), (410, 2), (410, 2), (170, 4))))
    for causal in (False, True):
        got = _grads(q, k, v, do, causal=causal, sequences=Sequences(ql, kl, qs, ks))
        ref, tol = _reference(q, k, v, do, causal, 0.125, list(zip(qs, ql, ks, kl)))
        _check(got, ref, tol)


def test_many_short_sequences_and_one_token_each():
    lens = [1 + i % 7 for i in range(300)]
    q, k, v, do = (_rand((sum(lens), h, 64), i) for i, h in enumerate((8, 2, 2, 8)))
    starts = [sum(lens[:i]) for i in range(len(lens))]
    got = _grads(q, k, v, do, sequences=Sequences(lens))
    ref, tol = _reference(q, k, v, do, True, 0.125, [(a, n, a, n) for a, n in zip(starts, lens)])
    _check(got, ref, tol)


def test_strided_operands():
    """Views of a fused projection, a cache's (kv head, row) order, expanded keys, offsets off 16 bytes: the bits of
    contiguous copies."""
    qkv = _rand((2, 90, 8, 64), 1)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    do = _rand((2, 4, 90, 64), 2).transpose(1, 2)
    want = _grads(*(x.contiguous() for x in (q, k, v, do)))
    got = _grads(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    cache = [torch.empty((2, 2, 100, 64), dtype=torch.bfloat16, device="cuda").fill_(math.nan) for _ in range(2)]
    for c, x in zip(cache, (k, v)):
        c[:, :, :90] = x.transpose(1, 2)
    got = _grads(q, *(c.transpose(1, 2)[:, :90] for c in cache), do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    flat = torch.empty(q.numel() + 3, dtype=torch.bfloat16, device="cuda")
    odd = flat[3:].view(q.shape).copy_(q)
    got = _grads(odd, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = k[:1].expand(2, -1, -1, -1)
    got, want = _grads(q, one, v, do), _grads(q, one.contiguous(), v, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got, want = attention(q, k, v)[..., 0].sum(), attention(q.contiguous(), k, v)[..., 0].sum()
    assert torch.equal(got, want)


def test_gradient_of_an_expanded_sum():
    q, k, v = (_rand((1, 40, 2, 64), i).requires_grad_() for i in range(3))
    out = attention(q, k, v)
    got = torch.autograd.grad(out.float().sum(), (q, k, v), retain_graph=True)
    want = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_shared_keys_and_values_add_their_gradients():
    """One tensor as keys and values: its gradient is the sum of both."""
    q, x, do = _rand((1, 50, 2, 64), 1), _rand((1, 50, 2, 64), 2), _rand((1, 50, 2, 64), 3)
    _, _, dk, dv = _grads(q, x, x.clone(), do)
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(attention(q, leaf, leaf), leaf, do)
    assert torch.equal(got, dk + dv)


def test_gradients_against_differences():
    """(L(x + h d) - L(x - h d)) / 2 h along random directions, L = sum(w out) of the 64-bit formula at the kernel's
    bf16 inputs: an h of 1e-4 leaves 1e-8 of curvature, far below the gradients' bf16 error (bounded as above)."""
    q, k, v, do = (_rand((1, 40, h, 64), i) for i, h in enumerate((4, 2, 2, 4)))
    got = _grads(q, k, v, do)
    ref, tol = _reference(q[0], k[0], v[0], do[0], True, 0.125, [(0, 40, 0, 40)])
    x = [t[0].double() for t in (q, k, v)]

    def loss(a, b, c):
        return float((_reference(a, b, c, do[0], True, 0.125, [(0, 40, 0, 40)])[0][0] * do[0].double()).sum())

    for i in range(3):
        d = torch.randn(x[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i)).cuda()
        h = 1e-4
        plus, minus = ([y + s * h * d if j == i else y for j, y in enumerate(x)] for s in (1, -1))
        diff = (loss(*plus) - loss(*minus)) / (2 * h)
        assert abs(float((got[1 + i][0].double() * d).sum()) - diff) <= float((tol[1 + i] * d.abs()).sum()) + 1e-5


def test_deterministic_and_streams_and_threads():
    """Equal bits from call to call, on several streams at once and from several threads."""
    import threading
    xs = [[_rand((2, 200, h, 64), 10 * i + j) for j, h in enumerate((8, 2, 2, 8))] for i in range(2)]
    alone = [_grads(*x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_grads(*xs[i]))
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            for _ in range(6):
                got[i].append(_grads(*xs[i]))
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(2):
        assert len(got[i]) == 12
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, alone[i]))


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed over new inputs, with eager work between the replays."""
    x = [_rand((2, 130, h, 64), i) for i, h in enumerate((8, 2, 2, 8))]
    static = [t.clone() for t in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _grads(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _grads(*static)
    for i in range(4):
        new = [_rand(t.shape, 50 + 10 * i + j) for j, t in enumerate(x)]
        for s, t in zip(static, new):
            s.copy_(t)
        graph.replay()
        want = _grads(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_two_graphs_do_not_share_scratch():
    xs = [[_rand((2, 150, h, 64), 7 * i + j) for j, h in enumerate((8, 2, 2, 8))] for i in range(2)]
    want = [_grads(*x) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_grads(*x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_a_cache_past_32_bit_offsets():
    """Key rows beyond 2^32 bytes (and 2^31 elements) of a long cache, one token's rows among them."""
    rows, KV = 20000, 900   # 20000 * 900 * 128 = 2.3e9 elements, 4.6 GB
    k = torch.zeros((1, rows, KV, 128), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    sub = slice(KV - 2, KV)
    k[:, :, sub], v[:, :, sub] = _rand((1, rows, 2, 128), 1), _rand((1, rows, 2, 128), 2)
    q, do = _rand((1, 2, 4, 128), 3), _rand((1, 2, 4, 128), 4)
    ref, tol = _reference(q[0], k[0, :, sub], v[0, :, sub], do[0], True, 128 ** -0.5, [(0, 2, 0, rows)])
    _check(_grads(q, k[:, :, sub], v[:, :, sub], do), ref, tol)
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]   # (kv head, row) order
    _check(_grads(q, turned[0][:, :, sub], turned[1][:, :, sub], do), ref, tol)


@pytest.mark.parametrize("tk", [129, 257, 512, 700, 1024, 1100])
def test_joins_of_two_to_many_splits(tk):
    """Few rows whose keys are split: 2 to 4, 5 to 8 and more splits are joined by different numbers of lanes."""
    _dense(1, 3, tk, 4, 2, 64, True, seed=tk)
    _dense(2, 130, tk, 2, 1, 72, False, seed=tk + 1)


@pytest.mark.parametrize("T,H,KV,D,causal", [(2500, 1, 1, 128, True), (1800, 3, 1, 64, True), (1500, 2, 1, 96, False)])
def test_key_blocks_in_several_parts(T, H, KV, D, causal):
    """Few heads over long sequences: the rows that see a key block are shared out to parts."""
    _dense(1, T, T, H, KV, D, causal, seed=T)


def test_captured_sequences_and_an_overwritten_table():
    """Packed rows in a graph over a table made before; a table whose entries have come to leave the rows reads as empty
    sequences, whose rows stay as they were."""
    lens = [300, 40, 0, 129]
    n = sum(lens)
    x = [_rand((n + 5, h, 64), i) for i, h in enumerate((4, 2, 2, 4))]
    seqs = Sequences(lens)
    want = _grads(*x, sequences=seqs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _grads(*x, sequences=seqs)
    for _ in range(3):
        graph.replay()
        again = _grads(*x, sequences=seqs)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, out, again))
    assert seqs.table[:, 1].tolist() == [300, 129, 40, 0]
    seqs.table[0, 0], seqs.table[1, 3], seqs.table[2, 1] = -7, 2 ** 30, n + 1   # start, keys, rows
    got = _grads(*x, sequences=Sequences([], device="cuda"))
    assert all(not g.any() for g in got)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.isfinite(a).all() for a in out)
    assert all(not a[n:].any() for a in out)
