"""Calls of the layer operators that are refused before anything reaches a device, on the CPU: the torch calls themselves
(transformer_amd/_ops.so) over host tensors, as the Python modules hand them over."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from transformer_amd import _lib
from transformer_amd.rotary import rotary, rotary_frequencies
from transformer_amd.swiglu import swiglu


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


def _calls():
    """(call, its operands) of every operator: host tensors and plans of their shapes."""
    ops, x = _lib.ops(), [torch.linspace(-1, 1, 64).reshape(4, 16) * (i + 1) for i in range(3)]
    a = _lib.MsdAttn()
    h = [t.to(torch.bfloat16).reshape(4, 2, 8) for t in x]
    attn = ops.AttnPlan(ctypes.addressof(a), 0, 0, False, False, None, None, 0)
    rms, glu, rope = ops.RmsPlan(4, 16, 1, 1, 1e-5, 16, 16, 0, 16), ops.GluPlan(4, 16, 1, 16, 16, 0), _rope()
    return [
        (lambda q, k, v: ops.attention(q, k, v, attn), h),
        (lambda q: ops.rotary(q, None, _turns(), None, rope)[0], [x[0].reshape(4, 2, 8)]),
        (lambda s, w: ops.rms_norm(s, w, None, rms)[0], [x[0], x[1][0]]),
        (lambda s, w, r: ops.rms_norm(s, w, r, rms)[0], [x[0], x[1][0], x[2]]),
        (lambda g, u: ops.swiglu(g, u, glu), x[:2]),
    ]


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode(which, recorded):
    """An operand with a tangent, whichever it is: a result without one would stand for a tangent of zero."""
    f, x = _calls()[which]
    for i in range(len(x)):
        with fwd.dual_level(), torch.set_grad_enabled(recorded):
            y = [t.clone().requires_grad_(recorded) for t in x]
            y[i] = fwd.make_dual(y[i], torch.ones_like(y[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*y)


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("recorded", [False, True])
def test_traces(which, recorded):
    """A trace would keep the outputs' allocation and none of the kernels."""
    f, x = _calls()[which]
    x = tuple(t.clone().requires_grad_(recorded) for t in x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, x, check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(f)(*x)


@pytest.mark.parametrize("shape", [(2 ** 27, 1, 8), (2 ** 32 + 5, 1, 8), (2 ** 32 + 1, 3, 2, 8), (3, 2 ** 32 + 1, 2, 8), (4, 4097, 8),
                                   (2 ** 20, 2 ** 12, 2 ** 8), (2, 2, 4104)])
def test_more_tokens_or_heads_than_the_library_counts(shape):
    """2^32 + 5 tokens would be 5 in 32 bits: the others' outputs would stay whatever the memory held."""
    q = torch.zeros(1, dtype=torch.bfloat16).expand(shape)
    with pytest.raises(ValueError, match=r"2 \*\* 27 tokens"):
        rotary(q, None, rotary_frequencies(8, device="cpu"))


@pytest.mark.parametrize("start", [2 ** 62 + 1, 2 ** 64 + 3, -2 ** 63])
def test_starts_past_64_bits(start):
    with pytest.raises(ValueError, match="start"):
        rotary(torch.zeros(4, 2, 8), None, rotary_frequencies(8, device="cpu"), start=start)


@pytest.mark.parametrize("d", [2 ** 24, 2 ** 32 + 128])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_rows_longer_than_the_library_counts(d, checkpoint):
    x = torch.zeros(1, dtype=torch.bfloat16).expand(2, d)
    with pytest.raises(ValueError, match=r"2 \*\* 24"):
        swiglu(x, x, checkpoint=checkpoint)


@pytest.mark.parametrize("back", [torch.zeros(4, 6).half(), torch.zeros(24), torch.zeros(6, 4), torch.zeros(4, 5),
                                  torch.zeros(4, 6, device="meta")])
def test_saved_tensors_that_come_back_as_others(back):
    """The check that every backward begins with (test_layers_calls_gpu.py): anything but other strides."""
    saved = torch.zeros(4, 6)
    _lib.ops().restored(torch.zeros(6, 4).t(), saved)
    with pytest.raises(RuntimeError, match="saved tensor"):
        _lib.ops().restored(back, saved)
