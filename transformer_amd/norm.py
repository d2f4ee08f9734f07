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
    """How calls on tensors of one layout go."""

    def __init__(self, x, scale, residual, eps, checkpoint):
        _check(x, scale, residual, eps, checkpoint)
        self.rows, self.d, self.type, self.index = math.prod(x.shape[:-1]), x.shape[-1], _lib.TYPES[x.dtype], x.get_device()
        self.scale_type, self.eps = _lib.TYPES[scale.dtype], eps
        strides = [0 if t is None else _lib.row_stride(t.shape, t.stride()) for t in (x, residual)]
        self.copies = None in strides
        self.x_stride, self.residual_stride = (self.d, self.d) if self.copies else strides
        self.sums = residual is not None
        self.held = _lib.keep_bytes(self.rows, self.d, checkpoint)
        self.kept_stride = self.x_stride if residual is None else self.d   # of what the backward reads: x, or the sum
        self.parts = _lib.check(_lib.lib().msd_rms_workspace_bytes(self.rows, self.d), "msd_rms_workspace_bytes") // 4


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


def _forward(x, scale, residual, plan, keep):
    if plan.copies:
        x, residual = x.contiguous(), None if residual is None else residual.contiguous()
    scale = scale.contiguous()
    y = _lib.empty(x)
    total = None if residual is None else _lib.empty(x)
    rstd = x.new_empty(plan.rows, dtype=torch.float32) if keep else None
    held = x.new_empty(plan.held, dtype=torch.uint8) if keep and plan.held else None
    _lib.launch(_lib.lib().msd_rms_forward, "msd_rms_forward", plan.index, x.data_ptr(), plan.x_stride,
                None if residual is None else residual.data_ptr(), plan.residual_stride, scale.data_ptr(), plan.scale_type,
                plan.rows, plan.d, plan.type, plan.eps, y.data_ptr(), None if total is None else total.data_ptr(),
                None if rstd is None else rstd.data_ptr(), None if held is None else held.data_ptr())
    return y, total, x, scale, rstd, held


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, residual, plan):
        ctx.scale_grad = scale.requires_grad
        y, total, x, scale, rstd, held = _forward(x, scale, residual, plan, True)
        ctx.save_for_backward(x if held is None and total is None else total if held is None else held, scale, rstd)
        ctx.plan, ctx.held = plan, held is not None
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy, dtotal=None):
        if dy is None:   # only the sum was used: the norm adds nothing
            return dtotal, None, dtotal, None   # (there is a residual then)
        plan = ctx.plan
        kept, scale, rstd = ctx.saved_tensors
        dy, dy_stride = _lib.rows_of(dy)
        ds, ds_stride = (None, 0) if dtotal is None else _lib.rows_of(dtotal)
        dx = _lib.empty(dy)
        dscale, ws = (torch.empty_like(scale), rstd.new_empty(plan.parts)) if ctx.scale_grad else (None, None)
        at = kept.data_ptr()
        _lib.launch(_lib.lib().msd_rms_backward, "msd_rms_backward", plan.index, None if ctx.held else at, plan.kept_stride,
                    rstd.data_ptr(), at if ctx.held else None, scale.data_ptr(), plan.scale_type, dy.data_ptr(), dy_stride,
                    None if ds is None else ds.data_ptr(), ds_stride, plan.rows, plan.d, plan.type, dx.data_ptr(),
                    None if dscale is None else dscale.data_ptr(), None if ws is None else ws.data_ptr())
        return dx, dscale, dx if plan.sums else None, None


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
    if torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or (residual is not None and residual.requires_grad)):
        return _RmsNorm.apply(x, scale, residual, plan)
    y, total, *_ = _forward(x, scale, residual, plan, False)
    return y if total is None else (y, total)
