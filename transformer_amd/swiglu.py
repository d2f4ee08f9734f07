"""SwiGLU between the feed-forward's projections, forward and gradient: the reference's silu(x W_gate) * (x W_up)
(model.py:159).

  y = swiglu(gate, up, checkpoint=None)

What runs (``msd_swiglu_forward`` / ``msd_swiglu_backward``, ``csrc/layers.hip``): one pass each way, f32 arithmetic.
``checkpoint="int8"`` keeps gate and up in 8 bits (one f32 scale per 128 values of a row) for the backward instead of
holding on to them: half the memory of bf16 for the widest activations of a layer; the gradients are then those at the
values that the checkpoint stands for, off by up to 1/254 of a block's largest.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib


def _forward(gate, up, checkpoint, keep):
    g, g_stride = _lib.rows_of(gate)
    u, u_stride = _lib.rows_of(up)
    n, d = g.shape
    y = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
    held = g.new_empty(2 * _lib.keep_bytes(n, d, checkpoint), dtype=torch.uint8) if keep and checkpoint else None
    _lib.launch(_lib.lib().msd_swiglu_forward, "msd_swiglu_forward", gate.device, g.data_ptr(), g_stride, u.data_ptr(),
                u_stride, n, d, _lib.TYPES[gate.dtype], y.data_ptr(), None if held is None else held.data_ptr())
    return y, g, u, held


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, checkpoint):
        y, g, u, held = _forward(gate, up, checkpoint, True)
        ctx.save_for_backward(*((held,) if held is not None else (g, u)))
        ctx.how = gate.shape, gate.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        shape, dtype = ctx.how
        held, g, u, strides = None, None, None, (0, 0)
        if len(ctx.saved_tensors) == 1:
            held, = ctx.saved_tensors
        else:
            g, u = ctx.saved_tensors
            strides = tuple(x.stride(0) if x.shape[0] > 1 else 0 for x in (g, u))
        dy, dy_stride = _lib.rows_of(dy)
        n, d = dy.shape
        dgate, dup = (torch.empty(shape, dtype=dtype, device=dy.device) for _ in range(2))
        _lib.launch(_lib.lib().msd_swiglu_backward, "msd_swiglu_backward", dy.device, None if held is not None else g.data_ptr(),
                    strides[0], None if held is not None else u.data_ptr(), strides[1],
                    None if held is None else held.data_ptr(), dy.data_ptr(), dy_stride, n, d, _lib.TYPES[dtype],
                    dgate.data_ptr(), dup.data_ptr())
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
    _check(gate, up, checkpoint)
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        return _Swiglu.apply(gate, up, checkpoint)
    return _forward(gate, up, checkpoint, False)[0]
