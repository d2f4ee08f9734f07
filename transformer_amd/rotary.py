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
    """Turns per position of each pair (device float64, d_rot / 2) and the amplitude of the rotated values.  They take no
    gradient: ``rotary`` refuses turns that want one while gradients are recorded."""

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


def _set(struct, name, values):
    getattr(struct, name)[:] = values   # (by name: torch.compile, which runs these lines itself, cannot assign to struct.name[:])


class _Plan:
    """How calls on tensors of one layout go; ``native``: the library's arguments, where the heads are contiguous."""

    def __init__(self, q, k, frequencies, positions, start, layout):
        _check(q, k, frequencies, positions, start, layout)
        self.native = None
        if not all(x is None or x.shape[-1] == 1 or x.stride(-1) == 1 for x in (q, k)):
            return
        r = [_lib.MsdRope(), _lib.MsdRope()]   # forward, and for gradients, whose strides are set when they are known
        for r_, sign in zip(r, (1, -1)):
            *_, r_.tokens, r_.n_heads, r_.d_head = q.shape
            r_.batch = q.shape[0] if q.dim() == 4 else 1
            r_.n_kv_heads, r_.d_rot = 0 if k is None else k.shape[-2], frequencies.d_rot
            r_.interleaved, r_.type, r_.sign, r_.amplitude, r_.start = LAYOUTS[layout], _lib.TYPES[q.dtype], sign, frequencies.amplitude, start
            if positions is not None:
                r_.position_bytes = positions.element_size()
                _set(r_, "position_stride", positions.stride() if positions.dim() == 2 else (0, *positions.stride()))
        _set(r[0], "q_stride", _strides(q))
        _set(r[0], "k_stride", (0, 0, 0) if k is None else _strides(k))
        self.native = _lib.ops().RopePlan(*map(ctypes.addressof, r))


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


def _check(q, k, frequencies, positions, start, layout):
    if q.dim() not in (3, 4):
        raise ValueError(f"q (batch, tokens, heads, d_head) or (tokens, heads, d_head) expected, got {tuple(q.shape)}")
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype):
        raise ValueError(f"k must be q's tokens, d_head and type, got {tuple(k.shape)} {k.dtype} beside {tuple(q.shape)} {q.dtype}")
    rows, heads, d = math.prod(q.shape[:-2]), q.shape[-2] + (0 if k is None else k.shape[-2]), q.shape[-1]
    if rows >= 2 ** 27 or heads > 4096 or d > 4096 or rows * heads * d >= 2 ** 40:   # (the library takes 32-bit counts)
        raise ValueError(f"fewer than 2 ** 27 tokens, up to 4096 heads of q and k together, heads of up to 4096 values and fewer than "
                         f"2 ** 40 values in all expected, got {rows} tokens and {heads} heads of {d}")
    if not -2 ** 62 <= start <= 2 ** 62:
        raise ValueError(f"start must lie in [-2 ** 62, 2 ** 62] (got {start})")
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
    if plan.native is None:
        q, k = q.contiguous(), None if k is None else k.contiguous()
        plan = _plan(q, k, frequencies, positions, int(start), layout)
    out = _lib.ops().rotary(q, k, frequencies.turns, positions, plan.native)
    return out[0] if k is None else tuple(out)
