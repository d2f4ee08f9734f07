"""Calls of the layer operators that their first tests leave out: saved tensors with other strides."""

import pytest
import torch

from transformer_amd.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_rotary_positions_whose_saved_copy_has_other_strides(kind):
    """Strided positions that go to host memory and back between forward and backward come back contiguous."""
    freq, (B, T) = rotary_frequencies(64), (3, 50)
    every = torch.randint(0, 5000, (B, 3 * T), generator=torch.Generator().manual_seed(1)).to(kind).cuda()
    x, dx = _rand((B, T, 4, 64), 2), _rand((B, T, 4, 64), 3)
    for positions in (every[:, ::3], every[:, :T], every[:1, ::3].expand(B, T), every[1, ::3], every.t()[:T, :B].t()):
        grads = []
        for moved in (False, True):
            leaf = x.clone().requires_grad_()
            if moved:
                with torch.autograd.graph.save_on_cpu():
                    y = rotary(leaf, None, freq, positions)
            else:
                y = rotary(leaf, None, freq, positions.contiguous())
            grads += torch.autograd.grad(y, leaf, dx)
        assert torch.equal(*grads)
