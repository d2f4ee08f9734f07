"""Attention in layouts outside the ordinary: pages whose positions share memory, sequences without new tokens that start anywhere.
Tolerances as in test_paged_attention_gpu.py."""
import pytest
import torch

from test_paged_attention_gpu import near, rand, reference, tables_of
from transformer_amd.paged_attention import PagedSequences, paged_attention

pytestmark = pytest.mark.gpu


def spread(KV, positions, D, stride, seed):
    """Pages (KV, positions, D) whose positions are `stride` elements apart."""
    head = positions * stride + D + 8 - D % 8
    return rand((KV * head,), seed).as_strided((KV, positions, D), (head, stride, 1))


@pytest.mark.parametrize("q_lens,lengths", [([1], [200]), ([1, 2], [3000, 37]), ([100], [170]), ([333, 40], [2000, 41]), ([1, 60, 5], [300, 61, 5])])
@pytest.mark.parametrize("D,k_stride,v_stride", [(64, 0, 0), (64, 0, 64), (128, 8, 120), (128, 256, 0), (64, 56, 32), (40, 8, 32), (96, 48, 8), (24, 8, 16)])
def test_positions_that_overlap(q_lens, lengths, D, k_stride, v_stride):
    """Keys and values whose rows are nearer than they are long, down to one row for all positions, against tokens and chunks."""
    H, KV = 4, 2
    tables, n = tables_of(lengths, 1)
    q = rand((sum(q_lens), H, D), 2, 1.5)
    k, v = spread(KV, 16 * n, D, k_stride, 3), spread(KV, 16 * n, D, v_stride, 4)
    sequences = PagedSequences(q_lens, lengths, tables, H, KV)
    starts = [sum(q_lens[:s]) for s in range(len(q_lens))]
    old = torch.rand((len(q_lens), KV, max(lengths)), generator=torch.Generator().manual_seed(5)).cuda()
    ref, tol = reference(q, k, v, q_lens, lengths, tables, starts, D ** -0.5, old, max(lengths))
    near(paged_attention(q, k, v, sequences), ref[0], tol[0], "out")
    out, weights = paged_attention(q, k, v, sequences, weights=old)
    near(out, ref[0], tol[0], "out")
    near(weights, ref[1], tol[1], "weights")


def test_one_row_for_all_positions():
    """The same row everywhere is the output, for a token and for a chunk alike."""
    q, row = rand((201, 4, 64), 1), rand((2, 1, 64), 2)
    pages = row.expand(-1, 320, -1)
    out = paged_attention(q, pages, pages, PagedSequences([1, 200], [90, 219], [range(6), range(6, 20)], 4, 2))
    want = row[:, 0].repeat_interleave(2, 0).expand(201, -1, -1)
    # (sums of up to 219 probabilities, each rounded to bf16 as an operand, and the output)
    assert ((out.double() - want.double()).abs() <= (2.0 ** -7 + 2.0 ** -12) * want.double().abs()).all()


@pytest.mark.parametrize("q_lens,lengths", [([1, 0], [30, 40]), ([0, 2, 0], [500, 300, 16]), ([1, 0], [3000, 2000]), ([50, 0], [300, 40]), ([0, 0], [30, 700]),
                                            ([0, 0, 1, 70], [5, 900, 60, 700])])
@pytest.mark.parametrize("longest", [None, 3100])
def test_weights_of_a_sequence_that_starts_behind_the_rows(q_lens, lengths, longest):
    """A sequence without new tokens keeps its weights, wherever its start lies: in one launch, in pieces, beside chunks."""
    rows, H, KV = sum(q_lens), 4, 2
    tables, n = tables_of(lengths, 1)
    starts = [sum(q_lens[:s]) if q else rows + 7 + 2 ** 30 * (s % 2) for s, q in enumerate(q_lens)]
    q, k, v = rand((rows, H, 64), 2, 1.5), rand((KV, 16 * n, 64), 3), rand((KV, 16 * n, 64), 4)
    old = 1 + torch.rand((len(q_lens), KV, max(lengths)), generator=torch.Generator().manual_seed(5)).cuda()
    sequences = PagedSequences(q_lens, lengths, tables, H, KV, q_starts=starts, longest=longest)
    torch.full((4096, 1024), float("nan"), device="cuda")   # (freed: what a call leaves unwritten is not a number)
    ref, tol = reference(q, k, v, q_lens, lengths, tables, starts, 0.125, old, sequences.longest)
    out, weights = paged_attention(q, k, v, sequences, weights=old)
    near(out, ref[0], tol[0], "out")
    near(weights, ref[1], tol[1], "weights")
