"""A step's device words that something else has written since: calls on them end, whatever single numbers they hold.  (What
is no longer the step's plan has no result to be compared; calls on sequences of their own are right afterwards.)"""
import pytest
import torch

from test_paged_attention_gpu import rand, tables_of
from test_paged_plan import AT_APPENDS, AT_FEW, AT_FEWS, AT_MANY, AT_MANYS, AT_SEQS, AT_TILES, N_APPENDS, N_FEW, N_FEWS, N_MANY, N_MANYS, N_TILES, SEQS
from transformer_amd.paged_attention import PagedEviction, PagedSequences, paged_append, paged_attention, paged_evict

pytestmark = pytest.mark.gpu
LISTS = {"few": (AT_FEW, N_FEW, 8), "few, weights": (AT_FEW + 1, N_FEW + 1, 8), "few sequences": (AT_FEWS, N_FEWS, 8), "few sequences, weights": (AT_FEWS + 1, N_FEWS, 8),
         "many": (AT_MANY, N_MANY, 8), "row tiles": (AT_TILES, N_TILES, 8), "many sequences": (AT_MANYS, N_MANYS, 8),
         "appends": (AT_APPENDS, N_APPENDS, 4), "sequences": (AT_SEQS, SEQS, 4)}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("q_lens,lengths", [([1, 60], [3000, 2000]), ([1, 3], [300, 200]), ([200, 70], [2900, 90])])
def test_calls_on_overwritten_numbers_end(name, q_lens, lengths):
    b = len(lengths)
    tables, n = tables_of(lengths + [32] * b, 3)
    rows = sum(q_lens)
    q, k, v = rand((rows, 4, 64), 1), rand((rows, 2, 64), 2), rand((rows, 2, 64), 3)
    kp, vp = rand((2, 16 * n, 64), 4), rand((2, 16 * n, 64), 5)
    old = torch.rand((b, 2, max(lengths))).cuda()
    s = PagedSequences(q_lens, lengths, tables[:b], 4, 2)
    e = PagedEviction(s, 32, 8, tables[b:])
    at, count, each = (s.host[LISTS[name][0]].item(), s.host[LISTS[name][1]].item(), LISTS[name][2])
    words = s.table[at:at + each * count].view(count, each)
    for i in range(each):
        for x in (0, 1, 2 ** 31 - 1, -2 ** 31, -1, 2 ** 31 - 100):
            held = words[:, i].clone()
            words[:, i] = x
            paged_append(k, v, kp, vp, s)
            paged_attention(q, kp, vp, s)
            paged_attention(q, kp, vp, s, weights=old)
            paged_evict(kp, vp, old, e)
            words[:, i] = held
    torch.cuda.synchronize()
    assert torch.equal(s.table.cpu(), s.host)
    assert torch.equal(paged_attention(q, kp, vp, s), paged_attention(q, kp, vp, PagedSequences(q_lens, lengths, tables[:b], 4, 2)))
