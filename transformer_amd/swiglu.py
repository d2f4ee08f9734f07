"""SwiGLU between the feed-forward's projections, forward and gradient: the reference's silu(x W_gate) * (x W_up)
(model.py:159).

  y = swiglu(gate, up, checkpoint=None)

What runs (``msd_swiglu_forward`` / ``msd_swiglu_backward``, ``csrc/layers.hip``): one pass each way, f32 arithmetic.
``checkpoint="int8"`` keeps gate and up in 8 bits (one f32 scale per 128 values of a row) for the backward instead of
holding on to them: half the memory of bf16 for the widest activations of a layer; the gradients are then those at the
values that the checkpoint stands for, off by up to 1/254 of a block's largest.
"""
import math

import torch

from . import _lib


class _Plan:
    """How calls on tensors of one layout go."""

    def __init__(self, gate, up, checkpoint):
        _check(gate, up, checkpoint)
        self.rows, self.d, self.type, self.index = math.prod(gate.shape[:-1]), gate.shape[-1], _lib.TYPES[gate.dtype], gate.get_device()
        strides = [_lib.row_stride(x.shape, x.stride()) for x in (gate, up)]
        self.copies = None in strides
        self.gate_stride, self.up_stride = (self.d, self.d) if self.copies else strides
        self.held = 2 * _lib.keep_bytes(self.rows, self.d, checkpoint)


_plans = {}


def _plan(gate, up, checkpoint):
    key = gate.shape, gate.stride(), gate.dtype, gate.device, up.shape, up.stride(), up.dtype, up.device, checkpoint
    found = _plans.get(key)
    if found is None:
        found = _Plan(gate, up, checkpoint)
        if len(_plans) >= 256:
            _plans.clear()
        _plans[key] = found
    return found


def _forward(gate, up, plan, keep):
    if plan.copies:
        gate, up = gate.contiguous(), up.contiguous()
    y = _lib.empty(gate)
    held = gate.new_empty(plan.held, dtype=torch.uint8) if keep and plan.held else None
    _lib.launch(_lib.lib().msd_swiglu_forward, "msd_swiglu_forward", plan.index, gate.data_ptr(), plan.gate_stride,
                up.data_ptr(), plan.up_stride, plan.rows, plan.d, plan.type, y.data_ptr(),
                None if held is None else held.data_ptr())
    return y, gate, up, held


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, plan):
        y, gate, up, held = _forward(gate, up, plan, True)
        ctx.plan = plan
        if held is None:
            ctx.save_for_backward(gate, up)
        else:
            ctx.save_for_backward(held)
        return y

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy):
        plan, saved = ctx.plan, ctx.saved_tensors
        dy, stride = _lib.rows_of(dy)
        dgate, dup = _lib.empty(dy), _lib.empty(dy)
        gate, up, held = (saved[0].data_ptr(), saved[1].data_ptr(), None) if len(saved) == 2 else (None, None, saved[0].data_ptr())
        _lib.launch(_lib.lib().msd_swiglu_backward, "msd_swiglu_backward", plan.index, gate, plan.gate_stride, up,
                    plan.up_stride, held, dy.data_ptr(), stride, plan.rows, plan.d, plan.type, dgate.data_ptr(),
                    dup.data_ptr())
        return dgate, dup, None


def _check(gate, up, checkpoint):
    if gate.dim() < 1 or gate.shape != up.shape or gate.dtype != up.dtype or gate.shape[-1] == 0:
        raise ValueError(f"gate and up of one shape (..., d) and type expected, got {tuple(gate.shape)} {gate.dtype} and "
                         f"{tuple(up.shape)} {up.dtype}")
    if gate.dtype not in _lib.TYPES:
        raise ValueError("gate and up must be bfloat16 or float32")
    if checkpoint not in (None, "int8"):
        raise ValueError(f'checkpoint must be None or "int8" (got {checkpoint!r})')
    if not gate.is_cuda or up.device != gate.device:
        raise ValueError("gate and up must be on one GPU")


def swiglu(gate, up, checkpoint=None):
    """gate / (1 + exp(-gate)) * up: (..., d) bf16 or f32 on one GPU, any strides (halves of one projection, say); returns
    a contiguous tensor of their shape and type.  checkpoint: None, or "int8" (see the module)."""
    plan = _plan(gate, up, checkpoint)
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        return _Swiglu.apply(gate, up, plan)
    return _forward(gate, up, plan, False)[0]
