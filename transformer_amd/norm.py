"""RMSNorm with the residual's addition, forward and gradients: the reference's rms_norm (model.py:94-98) and the
residual sums around it (:157-160).

  y = rms_norm(x, scale)                        # model.py:94
  y, h = rms_norm(x, scale, residual)           # h = x + residual, y = rms_norm(h)

What runs (``msd_rms_forward`` / ``msd_rms_backward``, ``csrc/layers.hip``): one pass over each row, f32 sums; the scale's
gradient from f32 sums in a fixed order.  ``checkpoint="int8"`` keeps the normalised rows in 8 bits (one f32 scale per 128
values) for the backward instead of holding on to x or h: half the memory of bf16; the gradients are then those at the
values that the checkpoint stands for, off by up to 1/254 of a block's largest.
"""
import math

import torch

from . import _lib


class _Plan:
    """How calls on tensors of one layout go; ``native``: the library's arguments, where one stride describes the rows of
    each."""

    def __init__(self, x, scale, residual, eps, checkpoint):
        _check(x, scale, residual, eps, checkpoint)
        self.native = None
        strides = [0 if t is None else _lib.ops().row_stride(t) for t in (x, residual)]
        if None in strides:
            return
        rows, d = math.prod(x.shape[:-1]), x.shape[-1]
        parts = _lib.check(_lib.lib().msd_rms_workspace_bytes(rows, d), "msd_rms_workspace_bytes") // 4
        self.native = _lib.ops().RmsPlan(rows, d, _lib.TYPES[x.dtype], _lib.TYPES[scale.dtype], eps, *strides,
                                         _lib.keep_bytes(rows, d, checkpoint), parts)


_plans = {}


def _plan(x, scale, residual, eps, checkpoint):
    key = (x.shape, x.stride(), x.dtype, x.device, scale.shape, scale.dtype, scale.device, eps, checkpoint,
           None if residual is None else (residual.shape, residual.stride(), residual.dtype, residual.device))
    found = _plans.get(key)
    if found is None:
        found = _Plan(x, scale, residual, eps, checkpoint)
        if len(_plans) >= 256:
            _plans.clear()
        _plans[key] = found
    return found


def _check(x, scale, residual, eps, checkpoint):
    if x.dim() < 1 or scale.dim() != 1 or x.shape[-1] != scale.shape[0]:
        raise ValueError(f"x (..., d) and scale (d,) expected, got {tuple(x.shape)} and {tuple(scale.shape)}")
    if not 1 <= x.shape[-1] <= 16384:
        raise ValueError(f"rows of 1 to 16384 values expected (got {x.shape[-1]})")
    if x.dtype not in _lib.TYPES or scale.dtype not in _lib.TYPES:
        raise ValueError("x and scale must be bfloat16 or float32")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be x's shape and type, got {tuple(residual.shape)} {residual.dtype} beside "
                         f"{tuple(x.shape)} {x.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must be at least 0 (got {eps})")
    if checkpoint not in (None, "int8"):
        raise ValueError(f'checkpoint must be None or "int8" (got {checkpoint!r})')
    if not x.is_cuda or scale.device != x.device or (residual is not None and residual.device != x.device):
        raise ValueError("x, scale and residual must be on one GPU")


def rms_norm(x, scale, residual=None, eps=1e-5, checkpoint=None):
    """s / sqrt(mean(s^2) + eps) * scale over the last axis, s = x, or x + residual (rounded to x's type), which is then
    returned too: y, or (y, s).

    x (..., d) bf16 or f32 on one GPU, any strides, d up to 16384; residual of x's shape and type; scale (d,) bf16 or f32.
    checkpoint: None, or "int8" (see the module)."""
    plan = _plan(x, scale, residual, float(eps), checkpoint)
    if plan.native is None:
        x, residual = x.contiguous(), None if residual is None else residual.contiguous()
        plan = _plan(x, scale, residual, float(eps), checkpoint)
    out = _lib.ops().rms_norm(x, scale, residual, plan.native)
    return out[0] if residual is None else tuple(out)
