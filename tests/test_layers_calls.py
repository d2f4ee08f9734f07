"""Calls of the layer operators that are refused before anything reaches a device, on the CPU: the torch calls themselves
(transformer_amd/_ops.so) over host tensors, as the Python modules hand them over."""
import ctypes

import pytest
import torch

from transformer_amd import _lib


def _rope(tokens=4, heads=2, d=8, rot=8):
    r = _lib.MsdRope()
    r.batch, r.tokens, r.n_heads, r.d_head, r.d_rot, r.type, r.sign, r.amplitude = 1, tokens, heads, d, rot, 1, 1, 1.0
    r.q_stride[:] = (0, heads * d, d)
    return _lib.ops().RopePlan(ctypes.addressof(r), ctypes.addressof(r))


def _turns(n=4):
    return torch.linspace(0, 0.1, n, dtype=torch.float64)


@pytest.mark.parametrize("turns", [_turns().float(), _turns().half(), _turns(3), _turns(5), _turns(8)[::2], _turns().reshape(2, 2),
                                   torch.zeros(4, dtype=torch.float64, device="meta")])
def test_replaced_frequencies(turns):
    """A vector that is not what the plan was made for would be read past its end."""
    with pytest.raises(ValueError, match="float64"):
        _lib.ops().rotary(torch.zeros(4, 2, 8), None, turns, None, _rope())


def test_frequencies_that_want_a_gradient():
    """They would get none, without a word."""
    with pytest.raises(ValueError, match="no gradient"):
        _lib.ops().rotary(torch.zeros(4, 2, 8), None, _turns().requires_grad_(), None, _rope())
