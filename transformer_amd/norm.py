"""RMSNorm with the residual's addition, forward and gradients: the reference's rms_norm (model.py:94-98) and the
residual sums around it (:157-160).

  y = rms_norm(x, scale)                        # model.py:94
  y, h = rms_norm(x, scale, residual)           # h = x + residual, y = rms_norm(h)

What runs (``msd_rms_forward`` / ``msd_rms_backward``, ``csrc/layers.hip``): one pass over each row, f32 sums; the scale's
gradient from f32 sums in a fixed order.  ``checkpoint="int8"`` keeps the normalised rows in 8 bits (one f32 scale per 128
values) for the backward instead of holding on to x or h: half the memory of bf16; the gradients are then those at the
values that the checkpoint stands for, off by up to 1/254 of a block's largest.
"""
import torch

from . import _lib


def _forward(x, scale, residual, eps, checkpoint, keep):
    rows, stride = _lib.rows_of(x)
    n, d = rows.shape
    res, res_stride = _lib.rows_of(residual) if residual is not None else (None, 0)
    scale = scale.contiguous()
    y = _lib.empty(x)
    total = _lib.empty(x) if res is not None else None
    rstd = rows.new_empty(n, dtype=torch.float32) if keep else None
    held = rows.new_empty(_lib.keep_bytes(n, d, checkpoint), dtype=torch.uint8) if keep and checkpoint else None
    _lib.launch(_lib.lib().msd_rms_forward, "msd_rms_forward", y.get_device(), rows.data_ptr(), stride,
                None if res is None else res.data_ptr(), res_stride, scale.data_ptr(), _lib.TYPES[scale.dtype], n, d,
                _lib.TYPES[y.dtype], eps, y.data_ptr(), None if total is None else total.data_ptr(),
                None if rstd is None else rstd.data_ptr(), None if held is None else held.data_ptr())
    return y, total, scale, rstd, held, rows, stride


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, residual, eps, checkpoint):
        y, total, scale, rstd, held, rows, stride = _forward(x, scale, residual, eps, checkpoint, True)
        ctx.save_for_backward(held if held is not None else total if total is not None else rows, scale, rstd)
        n, d = rows.shape
        parts = _lib.check(_lib.lib().msd_rms_workspace_bytes(n, d), "msd_rms_workspace_bytes") // 4
        ctx.how = n, d, stride if total is None else d, held is not None, residual is not None, parts
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy, dtotal=None):
        n, d, stride, held, residual, parts = ctx.how
        if dy is None:   # only the sum was used: the norm adds nothing
            return dtotal, None, dtotal if residual else None, None, None
        kept, scale, rstd = ctx.saved_tensors
        rows, dy_stride = _lib.rows_of(dy)
        ds, ds_stride = _lib.rows_of(dtotal) if dtotal is not None else (None, 0)
        dx = _lib.empty(dy)
        dscale = ws = None
        if ctx.needs_input_grad[1]:
            dscale, ws = torch.empty_like(scale), rstd.new_empty(parts)
        at = kept.data_ptr()
        _lib.launch(_lib.lib().msd_rms_backward, "msd_rms_backward", dy.get_device(), None if held else at, stride,
                    rstd.data_ptr(), at if held else None, scale.data_ptr(), _lib.TYPES[scale.dtype], rows.data_ptr(),
                    dy_stride, None if ds is None else ds.data_ptr(), ds_stride, n, d, _lib.TYPES[dy.dtype], dx.data_ptr(),
                    None if dscale is None else dscale.data_ptr(), None if ws is None else ws.data_ptr())
        return dx, dscale, dx if residual else None, None, None


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
    _check(x, scale, residual, eps, checkpoint)
    if torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or (residual is not None and residual.requires_grad)):
        return _RmsNorm.apply(x, scale, residual, float(eps), checkpoint)
    y, total, *_ = _forward(x, scale, residual, float(eps), checkpoint, False)
    return y if total is None else (y, total)
