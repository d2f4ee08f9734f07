"""Rotary positions for q and k, forward and gradient: the reference's apply_rope (model.py:110-117) with both pair
layouts, part of the head, and frequencies scaled for long contexts.

  frequencies = rotary_frequencies(d_rot, base=10000.0, scaling=None, ...)     # once per model
  q, k = rotary(q, k, frequencies, positions)

What runs (``msd_rope_apply``, ``csrc/layers.hip``): one launch for q and k; a position's angles are formed in float64 and
reduced to a turn before they are rounded, so far positions keep f32's precision, and any position is valid (there is no
table to run past).  The gradient is the same kernel turning back.
"""
import ctypes
import functools
import math

import torch

from . import _lib


class RotaryFrequencies:
    """Turns per position of each pair (device float64, d_rot / 2) and the amplitude of the rotated values."""

    def __init__(self, turns, amplitude=1.0):
        if turns.dim() != 1 or turns.numel() == 0 or turns.dtype != torch.float64 or not turns.is_contiguous():
            raise ValueError("turns must be a contiguous float64 vector")
        self.turns, self.amplitude, self.d_rot = turns, float(amplitude), 2 * turns.numel()


def rotary_frequencies(d_rot, base=10000.0, scaling=None, factor=1.0, original_context=None, slow=1.0, fast=32.0,
                       amplitude=None, device="cuda"):
    """The frequencies base ** (-2 i / d_rot) (radians per position; model.py:101-107), scaled for contexts ``factor``
    times the trained one:

      None          as they are
      "linear"      all divided by factor (positions interpolated)
      "ntk"         base raised to base * factor ** (d_rot / (d_rot - 2)): the lowest is divided by factor, the highest kept
      "by_parts"    by the turns n a pair makes over ``original_context`` positions: kept for n >= fast, divided by factor for
                    n <= slow, mixed linearly in n between; the amplitude defaults to 0.1 ln(factor) + 1
    """
    d_rot = int(d_rot)
    if d_rot < 2 or d_rot % 2:
        raise ValueError(f"d_rot must be even and at least 2 (got {d_rot})")
    if not (base > 1 and math.isfinite(base) and factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"base must be above 1 and factor at least 1 (got {base} and {factor})")
    if scaling == "ntk":
        if d_rot < 4:
            raise ValueError("ntk scaling needs d_rot of at least 4")
        base = base * factor ** (d_rot / (d_rot - 2))
    turns = base ** (-torch.arange(0, d_rot, 2, dtype=torch.float64) / d_rot) / (2 * math.pi)
    if scaling == "linear":
        turns = turns / factor
    elif scaling == "by_parts":
        if original_context is None or original_context < 1 or not fast > slow:
            raise ValueError("by_parts scaling needs original_context, and fast above slow")
        keep = ((original_context * turns - slow) / (fast - slow)).clamp(0, 1)
        turns = turns * (keep + (1 - keep) / factor)
        amplitude = 0.1 * math.log(factor) + 1 if amplitude is None else amplitude
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return RotaryFrequencies(turns.to(device), 1.0 if amplitude is None else amplitude)


LAYOUTS = {"half": 0, "interleaved": 1}


def _strides(x):
    s = tuple(0 if n <= 1 else k for n, k in zip(x.shape[:-1], x.stride()))
    return s if len(s) == 3 else (0, *s)


@functools.lru_cache(maxsize=256)
def _call(shape, kv, q_stride, k_stride, dtype, d_rot, amplitude, interleaved, sign, pos_bytes, pos_stride, start):
    r = _lib.MsdRope()
    *_, r.tokens, r.n_heads, r.d_head = shape
    r.batch = shape[0] if len(shape) == 4 else 1
    r.n_kv_heads, r.d_rot, r.interleaved, r.type, r.sign = kv, d_rot, interleaved, _lib.TYPES[dtype], sign
    r.position_bytes, r.amplitude, r.start = pos_bytes, amplitude, start
    r.q_stride[:], r.k_stride[:], r.position_stride[:] = q_stride, k_stride, pos_stride
    return r


def _heads(x):
    return x if x.shape[-1] == 1 or x.stride(-1) == 1 else x.contiguous()


def _apply(q, k, turns, amplitude, positions, start, layout, sign):
    q, k = _heads(q), None if k is None else _heads(k)
    pos_bytes, pos_stride = 0, (0, 0)
    if positions is not None:
        pos_bytes = positions.element_size()
        pos_stride = positions.stride() if positions.dim() == 2 else (0, *positions.stride())
    r = _call(q.shape, 0 if k is None else k.shape[-2], _strides(q), (0, 0, 0) if k is None else _strides(k), q.dtype,
              2 * turns.numel(), amplitude, LAYOUTS[layout], sign, pos_bytes, pos_stride, start)
    q_out = _lib.empty(q)
    k_out = None if k is None else _lib.empty(k)
    _lib.launch(_lib.lib().msd_rope_apply, "msd_rope_apply", q.get_device(), ctypes.byref(r), q.data_ptr(),
                None if k is None else k.data_ptr(), None if positions is None else positions.data_ptr(), turns.data_ptr(),
                q_out.data_ptr(), None if k is None else k_out.data_ptr())
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, turns, amplitude, positions, start, layout):
        ctx.save_for_backward(turns, positions)
        ctx.how = amplitude, start, layout
        q, k = _apply(q, k, turns, amplitude, positions, start, layout, 1)
        return q if k is None else (q, k)

    @staticmethod
    @_lib.first_order
    def backward(ctx, dq, dk=None):
        turns, positions = ctx.saved_tensors
        amplitude, start, layout = ctx.how
        dq, dk = _apply(dq, dk, turns, amplitude, positions, start, layout, -1)
        return dq, dk, None, None, None, None, None


def _check(q, k, frequencies, positions, layout):
    if q.dim() not in (3, 4):
        raise ValueError(f"q (batch, tokens, heads, d_head) or (tokens, heads, d_head) expected, got {tuple(q.shape)}")
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype):
        raise ValueError(f"k must be q's tokens, d_head and type, got {tuple(k.shape)} {k.dtype} beside {tuple(q.shape)} {q.dtype}")
    if q.dtype not in _lib.TYPES:
        raise ValueError("q and k must be bfloat16 or float32")
    if layout not in LAYOUTS:
        raise ValueError(f'layout must be "half" or "interleaved" (got {layout!r})')
    if frequencies.d_rot > q.shape[-1]:
        raise ValueError(f"d_rot {frequencies.d_rot} exceeds d_head {q.shape[-1]}")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be int32 or int64")
        if tuple(positions.shape) not in (tuple(q.shape[:-2]), tuple(q.shape[-3:-2])):
            raise ValueError(f"positions {tuple(positions.shape)} do not match q {tuple(q.shape)}")
    if not q.is_cuda or any(x is not None and x.device != q.device for x in (k, frequencies.turns, positions)):
        raise ValueError("q, k, the frequencies and the positions must be on one GPU")


def rotary(q, k, frequencies, positions=None, start=0, layout="half"):
    """q and k with the first ``frequencies.d_rot`` values of every head turned by their token's position.

    q (batch, tokens, n_heads, d_head) or (tokens, n_heads, d_head), k alike with its own heads, or None; bf16 or f32 on
    one GPU, any strides.  positions: (batch, tokens) or (tokens,) int32 or int64, any values; without them token t is at
    position start + t.  layout: pairs (i, i + d_rot / 2) ("half", the reference's) or (2 i, 2 i + 1) ("interleaved").
    Returns contiguous (q, k), with autograd; q alone without a k."""
    _check(q, k, frequencies, positions, layout)
    args = (q, k, frequencies.turns, frequencies.amplitude, positions, int(start), layout)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(*args)
    q, k = _apply(*args, 1)
    return q if k is None else (q, k)
