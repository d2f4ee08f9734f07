"""SwiGLU between the feed-forward's projections, forward and gradient: the reference's silu(x W_gate) * (x W_up)
(model.py:159).

  y = swiglu(gate, up, checkpoint=None)

What runs (``msd_swiglu_forward`` / ``msd_swiglu_backward``, ``csrc/layers.hip``): one pass each way, f32 arithmetic.
``checkpoint="int8"`` keeps gate and up in 8 bits (one f32 scale per 128 values of a row) for the backward instead of
holding on to them: half the memory of bf16 for the widest activations of a layer; the gradients are then those at the
values that the checkpoint stands for, off by up to 1/254 of a block's largest.
"""
import torch

from . import _lib


def _forward(gate, up, checkpoint, keep):
    g, g_stride = _lib.rows_of(gate)
    u, u_stride = _lib.rows_of(up)
    n, d = g.shape
    y = _lib.empty(gate)
    held = g.new_empty(2 * _lib.keep_bytes(n, d, checkpoint), dtype=torch.uint8) if keep and checkpoint else None
    _lib.launch(_lib.lib().msd_swiglu_forward, "msd_swiglu_forward", y.get_device(), g.data_ptr(), g_stride, u.data_ptr(),
                u_stride, n, d, _lib.TYPES[y.dtype], y.data_ptr(), None if held is None else held.data_ptr())
    return y, g, u, held, (g_stride, u_stride)


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, checkpoint):
        y, g, u, held, ctx.strides = _forward(gate, up, checkpoint, True)
        if held is None:
            ctx.save_for_backward(g, u)
        else:
            ctx.save_for_backward(held)
        return y

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        rows, stride = _lib.rows_of(dy)
        n, d = rows.shape
        dgate, dup = _lib.empty(dy), _lib.empty(dy)
        kept = len(saved) == 1
        g, u, held = (None, None, saved[0].data_ptr()) if kept else (saved[0].data_ptr(), saved[1].data_ptr(), None)
        _lib.launch(_lib.lib().msd_swiglu_backward, "msd_swiglu_backward", dy.get_device(), g, ctx.strides[0], u,
                    ctx.strides[1], held, rows.data_ptr(), stride, n, d, _lib.TYPES[dy.dtype], dgate.data_ptr(),
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
    _check(gate, up, checkpoint)
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        return _Swiglu.apply(gate, up, checkpoint)
    return _forward(gate, up, checkpoint, False)[0]
