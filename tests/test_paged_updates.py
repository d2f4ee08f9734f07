"""An update that cannot be made leaves a step's sequences as they were, on the CPU."""
import pytest
import torch

from transformer_amd.paged_attention import PagedEviction, PagedSequences


def test_an_update_whose_copy_fails():
    """The device's words could not be written: the host's, the lengths, the pages in use and the evictions made are those from before."""
    s = PagedSequences([1, 3], [5, 40], [[3], [0, 1, 2]], 4, 2, longest=100, device="cpu")
    e = PagedEviction(s, 16, 4, [[9], [8]])
    s.table, table, host, used = torch.zeros(3, dtype=torch.int32), s.host.clone(), s.host.clone(), s.used().tolist()
    with pytest.raises(RuntimeError):
        s.update([17, 50], [[3, 4], [0, 1, 2, 5]])
    assert torch.equal(s.host, host) and s.lengths == [5, 40] and s.used().tolist() == used and s.version == e.version == 0
    s.table = table
    s.update([17, 50], [[3, 4], [0, 1, 2, 5]])
    want = PagedSequences([1, 3], [17, 50], [[3, 4], [0, 1, 2, 5]], 4, 2, longest=100, device="cpu")
    assert torch.equal(s.host, want.host) and torch.equal(s.table, want.host) and s.lengths == [17, 50] and s.version == 1
