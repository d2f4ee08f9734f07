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
    """How calls on tensors of one layout go; ``native``: the library's arguments, where one stride describes the rows of
    each."""

    def __init__(self, gate, up, checkpoint):
        _check(gate, up, checkpoint)
        self.native = None
        strides = [_lib.ops().row_stride(x) for x in (gate, up)]
        if None not in strides:
            rows, d = math.prod(gate.shape[:-1]), gate.shape[-1]
            self.native = _lib.ops().GluPlan(rows, d, _lib.TYPES[gate.dtype], *strides, 2 * _lib.keep_bytes(rows, d, checkpoint))


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


def _check(gate, up, checkpoint):
    if gate.dim() < 1 or gate.shape != up.shape or gate.dtype != up.dtype or gate.shape[-1] == 0:
        raise ValueError(f"gate and up of one shape (..., d) and type expected, got {tuple(gate.shape)} {gate.dtype} and "
                         f"{tuple(up.shape)} {up.dtype}")
    if gate.shape[-1] >= 2 ** 24:
        raise ValueError(f"rows of up to 2 ** 24 - 1 values expected (got {gate.shape[-1]})")
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
    if plan.native is None:
        gate, up = gate.contiguous(), up.contiguous()
        plan = _plan(gate, up, checkpoint)
    return _lib.ops().swiglu(gate, up, plan.native)
