"""Rotary positions for q and k, forward and gradient: the reference's apply_rope (model.py:110-117) with both pair
layouts, part of the head, and frequencies scaled for long contexts.

  frequencies = rotary_frequencies(d_rot, base=10000.0, scaling=None, ...)     # once per model
  q, k = rotary(q, k, frequencies, positions)

What runs (``msd_rope_apply``, ``csrc/layers.hip``): one launch for q and k; a position's angles are formed in float64 and
reduced to a turn before they are rounded, so far positions keep f32's precision, and any position is valid (there is no
table to run past).  The gradient is the same kernel turning back.
"""
import ctypes
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
    """(batch, token, head) strides of x with contiguous heads; 0 along an axis of one (or none)."""
    s = tuple(0 if n <= 1 else k for n, k in zip(x.shape[:-1], x.stride()))
    return s if len(s) == 3 else (0, *s)


def _contiguous(shape):
    s, d, h = shape[-3] * shape[-2] * shape[-1], shape[-1], shape[-2] * shape[-1]
    return (s, h, d)


def _turns_heads(x):
    return x.shape[-1] == 1 or x.stride(-1) == 1


class _Plan:
    """How calls on tensors of one layout go: the library's arguments forward and, for contiguous gradients, backward."""

    def __init__(self, q, k, frequencies, positions, start, layout):
        _check(q, k, frequencies, positions, layout)
        self.q_shape, self.kv, self.dtype, self.index = q.shape, 0 if k is None else k.shape[-2], q.dtype, q.get_device()
        self.d_rot, self.amplitude, self.start, self.layout = frequencies.d_rot, frequencies.amplitude, start, layout
        self.position_bytes, self.position_stride = 0, (0, 0)
        if positions is not None:
            self.position_bytes = positions.element_size()
            self.position_stride = positions.stride() if positions.dim() == 2 else (0, *positions.stride())
        self.copies = not _turns_heads(q) or (k is not None and not _turns_heads(k))
        whole = _contiguous(q.shape), None if k is None else _contiguous(k.shape)
        self.forward = self.call(1, *(whole if self.copies else (_strides(q), None if k is None else _strides(k))))
        self.backward = self.call(-1, *whole)

    def call(self, sign, q_stride, k_stride):
        r = _lib.MsdRope()
        *_, r.tokens, r.n_heads, r.d_head = self.q_shape
        r.batch = self.q_shape[0] if len(self.q_shape) == 4 else 1
        r.n_kv_heads, r.d_rot, r.interleaved, r.type, r.sign = self.kv, self.d_rot, LAYOUTS[self.layout], _lib.TYPES[self.dtype], sign
        r.position_bytes, r.amplitude, r.start = self.position_bytes, self.amplitude, self.start
        r.q_stride[:], r.k_stride[:], r.position_stride[:] = q_stride, k_stride or (0, 0, 0), self.position_stride
        return ctypes.byref(r)


_plans = {}


def _plan(q, k, frequencies, positions, start, layout):
    key = (q.shape, q.stride(), q.dtype, q.device, None if k is None else (k.shape, k.stride(), k.dtype, k.device),
           None if positions is None else (positions.shape, positions.stride(), positions.dtype, positions.device),
           frequencies.d_rot, frequencies.amplitude, frequencies.turns.device, start, layout)
    found = _plans.get(key)
    if found is None:
        found = _Plan(q, k, frequencies, positions, start, layout)
        if len(_plans) >= 256:
            _plans.clear()
        _plans[key] = found
    return found


def _apply(index, call, q, k, turns, positions):
    q_out = _lib.empty(q)
    k_out = None if k is None else _lib.empty(k)
    _lib.launch(_lib.lib().msd_rope_apply, "msd_rope_apply", index, call, q.data_ptr(), None if k is None else k.data_ptr(),
                None if positions is None else positions.data_ptr(), turns.data_ptr(), q_out.data_ptr(),
                None if k is None else k_out.data_ptr())
    return q_out, k_out


def _forward(q, k, turns, positions, plan):
    if plan.copies:
        q, k = q.contiguous(), None if k is None else k.contiguous()
    return _apply(plan.index, plan.forward, q, k, turns, positions)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, turns, positions, plan):
        ctx.save_for_backward(turns, positions)
        ctx.plan = plan
        q, k = _forward(q, k, turns, positions, plan)
        return q if k is None else (q, k)

    @staticmethod
    @_lib.first_order
    def backward(ctx, dq, dk=None):
        turns, positions = ctx.saved_tensors
        plan = ctx.plan
        call = plan.backward
        if not dq.is_contiguous() or (dk is not None and not dk.is_contiguous()):
            if not _turns_heads(dq) or (dk is not None and not _turns_heads(dk)):
                dq, dk = dq.contiguous(), None if dk is None else dk.contiguous()
            call = plan.call(-1, _strides(dq), None if dk is None else _strides(dk))
        dq, dk = _apply(plan.index, call, dq, dk, turns, positions)
        return dq, dk, None, None, None


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
    plan = _plan(q, k, frequencies, positions, int(start), layout)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, frequencies.turns, positions, plan)
    q, k = _forward(q, k, frequencies.turns, positions, plan)
    return q if k is None else (q, k)
