"""Pages and rows that share memory: what is refused, and what is as if the rows had been read before any page is written."""
import pytest
import torch

from test_paged_attention_gpu import rand, rows_of, tables_of
from test_paged_cache_gpu import appended, same
from transformer_amd.paged_attention import PagedEviction, PagedSequences, paged_append, paged_evict

pytestmark = pytest.mark.gpu


def _views(n):
    """(keys, values, whether they share memory) of two heads of 64, 16 n positions each."""
    P = 16 * n
    x = rand((4, 2 * P + 16, 128), 1)
    y = rand((2, P, 2, 64), 2)
    z = rand((P, 4, 64), 3).transpose(0, 1)
    return [
        (x[:2, :P, :64], x[:2, :P, :64], True),
        (x[:2, :P, :64], x[1:3, :P, :64], True),             # a head
        (x[:2, :P, :64], x[:2, 16:P + 16, :64], True),       # all pages but one
        (x[:2, :P, :64], x[:2, P - 16:2 * P - 16, :64], True),   # a page
        (x[:2, :P, :64], x[:2, :P, 56:120], True),           # a piece of each row
        (x[:2, :P, :64], x[:2, :P, 64:], False),
        (x[:2, :P, :64], x[2:, :P, :64], False),
        (x[::2, :P, :64], x[1::2, :P, :64], False),
        (x[:2, :P, :64], x[:2, P:2 * P, :64], False),
        (y[:, :, 0], y[:, :, 1], False),
        (y[:, :, 1], y[:, :, 0], False),
        (z[:2], z[2:], False),
        (z[::2], z[1::2], False),
        (z[:2], y[:, :, 0], False),                          # other strides in other memory
        (z[::3], z[1:3], False),                             # heads 0 and 3, heads 1 and 2
        (z[::3], z[2:], True),
    ]


@pytest.mark.parametrize("which", range(16))
def test_keys_and_values_in_one_memory(which):
    lengths = [40, 20]
    tables, n = tables_of(lengths + [16, 16], 1)
    k_pages, v_pages, shared = _views(n)[which]
    k, v, w = rand((12, 2, 64), 4), rand((12, 2, 64), 5), torch.rand(2, 2, 40).cuda()
    s = PagedSequences([5, 7], lengths, tables[:2], 4, 2)
    e = PagedEviction(s, 16, 4, tables[2:])
    if shared:
        held = k_pages.clone(), v_pages.clone()
        with pytest.raises(ValueError, match="same memory"):
            paged_append(k, v, k_pages, v_pages, s)
        with pytest.raises(ValueError, match="same memory"):
            paged_evict(k_pages, v_pages, w, e)
        assert same(k_pages, held[0]) and same(v_pages, held[1])
        return
    want = [appended(x, pages, [5, 7], lengths, tables, [0, 5]) for x, pages in ((k, k_pages), (v, v_pages))]
    paged_append(k, v, k_pages, v_pages, s)
    assert same(k_pages, want[0]) and same(v_pages, want[1])
    _, kept = paged_evict(k_pages, v_pages, w, e)
    for pages, before in ((k_pages, want[0]), (v_pages, want[1])):
        for b in range(2):
            for h in range(2):
                assert same(rows_of(pages, tables[2 + b], 16)[h], rows_of(before, tables[b], lengths[b])[h, kept[b, h].long()])


def test_layers_of_keys_and_values_in_one_memory():
    """All layers of a pool, keys and values in turn: apart; a layer's values as the next one's keys: not."""
    lengths = [40, 20]
    tables, n = tables_of(lengths + [16, 16], 1)
    pool = rand((4, 2, 2, 16 * n, 64), 1)
    s = PagedSequences([1, 1], lengths, tables[:2], 4, 2)
    e = PagedEviction(s, 16, 4, tables[2:])
    flat = pool.view(8, 2, 16 * n, 64)
    with pytest.raises(ValueError, match="same memory"):
        paged_evict(flat[:4], flat[1:5], torch.rand(4, 2, 2, 40).cuda(), e)
    with pytest.raises(ValueError, match="same memory"):
        paged_evict(flat[::2], flat[2:6:1], torch.rand(4, 2, 2, 40).cuda(), e)   # (other strides; two of four are the same)
    paged_evict(pool[:, 0], pool[:, 1], torch.rand(4, 2, 2, 40).cuda(), e)


@pytest.mark.parametrize("D", [64, 128])
def test_new_rows_that_lie_in_the_pages(D):
    """A page's rows as another sequence's, and rows that each move on by one position or one page."""
    n = 40
    for count, first, length in ((16, 0, 32), (13, 3, 20), (200, 0, 217), (600, 0, 616), (600, 5, 606)):
        k_pages, v_pages = rand((2, 16 * n, D), 1), rand((2, 16 * n, D), 2)
        k, v = (x[:, first:first + count].transpose(0, 1) for x in (k_pages, v_pages))
        s = PagedSequences([count], [length], [range(-(-length // 16))], 4, 2)
        want = [appended(x.clone(), pages, [count], [length], [range(n)], [0]) for x, pages in ((k, k_pages), (v, v_pages))]
        paged_append(k, v, k_pages, v_pages, s)
        assert same(k_pages, want[0]) and same(v_pages, want[1]), (count, first, length)
        k_pages, v_pages = rand((2, 16 * n, D), 1), rand((2, 16 * n, D), 2)
        k, v = (x[:, first:first + count].transpose(0, 1) for x in (v_pages, k_pages))   # each from the other's
        want = [appended(x.clone(), pages, [count], [length], [range(n)], [0]) for x, pages in ((k, k_pages), (v, v_pages))]
        paged_append(k, v, k_pages, v_pages, s)
        assert same(k_pages, want[0]) and same(v_pages, want[1]), (count, first, length)
