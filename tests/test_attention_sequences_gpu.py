"""Attention over sequences that leave rows out, with few rows, whose keys and rows are split: the same bits as packed, and the
formulas' values (tolerances: test_attention_gpu.py); and over a cache of a million rows a head."""
import math

import pytest
import torch

from test_attention_gpu import _check, _grads, _rand, _reference
from transformer_amd.attention import Sequences, _fits, attention

pytestmark = pytest.mark.gpu


def _starts(lens, gap=0):
    return [sum(gap or n for n in lens[:i]) for i in range(len(lens))]


def _padded(x, lens, gap):
    """The packed rows of x where each sequence has `gap` rows; the others hold NaN."""
    out = torch.full((gap * len(lens), *x.shape[1:]), math.nan, dtype=x.dtype, device="cuda")
    for n, a, b in zip(lens, _starts(lens), _starts(lens, gap)):
        out[b:b + n] = x[a:a + n]
    return out


@pytest.mark.parametrize("q_lens,k_lens,gap", [
    ([1] * 6, [700, 1, 64, 2000, 129, 0], 2048),       # 16 parts
    ([3, 1, 4] * 6, [600, 300, 513] * 6, 1000),        # 5 to 8
    ([40, 100] * 20, [300, 129] * 20, 300),            # 2 to 4
    ([300, 17, 170], None, 1024),                      # dK and dV in parts too
    ([1000, 2], [2, 1000], 1500),
    ([33], None, 5000),
])
@pytest.mark.parametrize("H,KV,D", [(8, 2, 64), (3, 1, 128), (2, 2, 72)])
@pytest.mark.parametrize("causal", [True, False])
def test_padded_rows_and_few_of_them(q_lens, k_lens, gap, H, KV, D, causal):
    k_lens = k_lens or q_lens
    q, do = (_rand((sum(q_lens), H, D), i) for i in (1, 2))
    k, v = (_rand((sum(k_lens), KV, D), i) for i in (3, 4))
    want = _grads(q, k, v, do, causal=causal, sequences=Sequences(q_lens, k_lens))
    ref, tol = _reference(q, k, v, do, causal, D ** -0.5, list(zip(_starts(q_lens), q_lens, _starts(k_lens), k_lens)))
    _check(want, ref, tol)
    lens = (q_lens, k_lens, k_lens, q_lens)
    seqs = Sequences(q_lens, k_lens, _starts(q_lens, gap), _starts(k_lens, gap))
    got = _grads(*(_padded(x, n, gap) for x, n in zip((q, k, v, do), lens)), causal=causal, sequences=seqs)
    for x, y, n in zip(got, want, (q_lens, q_lens, k_lens, k_lens)):
        rows = torch.zeros(len(x), dtype=torch.bool)
        for a, m in zip(_starts(n, gap), n):
            rows[a:a + m] = True
        assert torch.equal(x[rows.cuda()], y) and not x[~rows.cuda()].any()


def test_a_new_row_in_each_sequence_of_a_large_padded_batch():
    """32 x 4096 rows: out, its saved bytes and the gradients take what they take; parts over all rows would take gigabytes."""
    B, T, H, KV, D = 32, 4096, 32, 8, 128
    q, k, v = (_rand((1, 1, h, D), i).expand(B * T, -1, h, D)[:, 0] for i, h in enumerate((H, KV, KV)))
    seqs = Sequences([1] * B, [T] * B, range(T - 1, B * T, T), range(0, B * T, T))
    k, v = k.contiguous(), v.contiguous()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = _grads(q, k, v, q, sequences=seqs)
    taken = torch.cuda.max_memory_allocated() - before
    out, kv = B * T * H * D * 2, B * T * KV * D * 2
    assert taken < 2 * out + out // 2 + 2 * kv + B * T * H * 4 * 3 + 100e6, taken
    # equal keys: every output is v; dv of a sequence's rows is dout / T each, summed over a group's heads
    assert torch.equal(got[0][T - 1::T], v[T - 1::T].repeat_interleave(H // KV, 1))
    want = q[:1].double().reshape(KV, H // KV, D).sum(1) / T
    assert ((got[3].double() - want).abs() <= 2.0 ** -7 * q[:1].double().abs().reshape(KV, H // KV, D).sum(1) / T).all()


# Past 256 sequences: launches of 256, and one of all that follow where their lengths are alike
MANY = {
    "one long": [900] + [1 + i % 40 for i in range(500)],
    "long ones": [300 + i % 50 for i in range(300)] + [1 + 7 * i % 23 for i in range(300)],
    "alike": [20 + i % 7 for i in range(400)],
    "257": [400] + [3] * 256,
    "none but one": [0] * 300 + [130] + [0] * 300,
}


@pytest.mark.parametrize("lens", MANY)
@pytest.mark.parametrize("H,KV,D,causal", [(4, 1, 64, True), (2, 2, 72, False)])
def test_many_sequences(lens, H, KV, D, causal):
    lens = MANY[lens]
    q, k, v, do = (_rand((sum(lens) + 3, h, D), i) for i, h in enumerate((H, KV, KV, H)))
    ref, tol = _reference(q, k, v, do, causal, D ** -0.5, [(a, n, a, n) for a, n in zip(_starts(lens), lens)])
    got = _grads(q, k, v, do, causal=causal, sequences=Sequences(lens))
    _check(got, ref, tol)
    turned = Sequences(lens)   # the shortest first, as a C caller may have them
    turned.host = turned.host.flip(0).contiguous()
    turned.table.copy_(turned.host)
    _check(_grads(q, k, v, do, causal=causal, sequences=turned), ref, tol)


def test_many_sequences_of_their_own_keys():
    """One new row of each over caches of different lengths, a long one among them, and rows of a padded batch."""
    k_lens = [5000] + [1 + 13 * i % 90 for i in range(400)]
    q_lens = [1 + i % 3 for i in range(401)]
    q, do = (_rand((sum(q_lens), 4, 64), i) for i in (1, 2))
    k, v = (_rand((sum(k_lens), 2, 64), i) for i in (3, 4))
    got = _grads(q, k, v, do, sequences=Sequences(q_lens, k_lens))
    ref, tol = _reference(q, k, v, do, True, 0.125, list(zip(_starts(q_lens), q_lens, _starts(k_lens), k_lens)))
    _check(got, ref, tol)


def test_many_sequences_captured_and_replayed():
    lens = MANY["one long"]
    x = [_rand((sum(lens), h, 64), i) for i, h in enumerate((4, 2, 2, 4))]
    seqs = Sequences(lens)
    want = _grads(*x, sequences=seqs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _grads(*x, sequences=seqs)
    for i in range(3):
        graph.replay()
        again = _grads(*x, sequences=seqs)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, out, again)), i


def test_host_numbers_that_change_after_the_first_call():
    """Each call reads the numbers that its workspaces were made for."""
    lens = [1, 1, 1, 700]
    x = [_rand((sum(lens), h, 64), i) for i, h in enumerate((4, 2, 2, 4))]
    seqs = Sequences(lens)
    want = _grads(*x, sequences=seqs)
    seqs.host[1:] = torch.tensor([3, 700, 3, 700], dtype=torch.int32)
    assert all(torch.equal(a, b) for a, b in zip(_grads(*x, sequences=seqs), want))


def test_a_cache_of_a_million_rows_a_head_is_read_where_it_lies():
    """(kv head, row) order, 8 heads of 128: the heads together span 2^30 elements and more, each by itself does not."""
    rows, KV, H, D = 2 ** 20 + 16, 8, 16, 128
    caches = [torch.empty((1, KV, rows, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for i, c in enumerate(caches):
        c[:, :, :3000] = _rand((1, KV, 3000, D), i)
    k, v = (c.transpose(1, 2)[:, :3000] for c in caches)
    assert _fits(k.shape, k.stride(), 1) and not _fits(k.shape, k.stride(), KV)
    q, do = _rand((1, 2, H, D), 2), _rand((1, 2, H, D), 3)
    want = _grads(q, k.contiguous(), v.contiguous(), do)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    assert torch.equal(attention(q, k, v), want[0])
    taken = torch.cuda.max_memory_allocated() - before
    assert taken < k.numel() * 2, taken   # (no copy)
    assert all(torch.equal(a, b) for a, b in zip(_grads(q, k, v, do), want))
    whole = [c.transpose(1, 2) for c in caches]
    for c in caches:
        c[:, :, 3000:] = 0
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = attention(q, *whole)
    taken = torch.cuda.max_memory_allocated() - before
    assert taken < 100e6 and torch.isfinite(out).all()
