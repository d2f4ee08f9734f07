"""Attention for training and scoring: grouped heads, forward and a backward that recomputes the probabilities.

The reference's causal_attention (model.py:122-147) between its projections: q (T, n_heads, d_head), k and v
(T, n_kv, d_head), over torch tensors on the GPU in bf16, with autograd:

  attention(q, k, v, causal=True, scale=None, sequences=None)

What runs (``msd_attn_forward`` / ``msd_attn_backward``, ``csrc/attn.hip``): one pass over the keys with the running
maximum and sum of the softmax, so no score matrix is stored; the forward keeps each row's logsumexp, from which the
backward forms the probabilities again, and a byte beside each value of the output for what its rounding took off.
Scores, softmax statistics and every sum are f32; the probabilities and the scores' gradients are rounded to bf16 as
operands of the matrix cores, the results once to bf16.  Deterministic.
"""
import ctypes
import math

import torch

from . import _lib


class Sequences:
    """Which rows of flat q (Nq, n_heads, d_head) and k, v (Nk, n_kv, d_head) tensors belong to which sequence.

    Sequence s has ``q_lens[s]`` query rows from ``q_starts[s]`` and ``k_lens[s]`` key rows from ``k_starts[s]``; the
    starts default to the sequences packed one behind the other, the keys to the queries' (self-attention).  A padded
    batch is its flat view with ``q_starts=range(0, B * T, T)`` and each sequence's own length.  Rows of no sequence are
    neither read nor attended to; their outputs and gradients are zeros.  Built once per batch from host integers
    (checked here) and used by every layer; the device copy is made on the current stream.  A captured graph goes on
    reading that copy: like the graph's other inputs the object has to be kept, and made before the capture."""

    def __init__(self, q_lens, k_lens=None, q_starts=None, k_starts=None, device="cuda"):
        q_lens = [int(n) for n in q_lens]
        if k_lens is None and k_starts is None and q_starts is not None:
            k_starts = q_starts
        k_lens = q_lens if k_lens is None else [int(n) for n in k_lens]
        q_starts, self.q_end, self.q_count = _ranges(q_lens, q_starts, "q")
        k_starts, self.k_end, self.k_count = _ranges(k_lens, k_starts, "k")
        if len(q_lens) != len(k_lens):
            raise ValueError(f"{len(q_lens)} query and {len(k_lens)} key sequences")
        self.n = len(q_lens)
        self.q_longest, self.k_longest = max(q_lens, default=0), max(k_lens, default=0)
        rows = sorted(zip(q_starts, q_lens, k_starts, k_lens), key=lambda r: -r[1] * r[3])   # the most work first
        self.host = torch.tensor(rows, dtype=torch.int32).reshape(-1, 4)
        self.table = self.host.to(device)
        self.stream = _lib.current_stream(self.table)
        self._plans = {}


def _ranges(lens, starts, what):
    """(starts, one past the last row, rows in all) of checked, disjoint ranges."""
    if any(n < 0 for n in lens):
        raise ValueError(f"negative {what} length")
    if starts is None:
        starts, at = [], 0
        for n in lens:
            starts.append(at)
            at += n
    starts = [int(x) for x in starts]
    if len(starts) != len(lens):
        raise ValueError(f"{len(starts)} {what} starts for {len(lens)} lengths")
    end = 0
    for at, n in sorted((a, n) for a, n in zip(starts, lens) if n):
        if at < end:
            raise ValueError(f"{what} ranges overlap or start below 0")
        end = at + n
    if end >= 2 ** 31 or any(not 0 <= a < 2 ** 31 for a in starts):
        raise ValueError(f"{what} ranges outside [0, 2**31)")
    return starts, end, sum(lens)


def _fits(shape, stride, group):
    """Whether heads of these strides are contiguous, on 16-byte boundaries and within the kernels' reach: 128 rows and the heads
    that share a K/V head."""
    row, head = (s if n > 1 else 0 for n, s in zip(shape[-3:-1], stride[-3:-1]))
    return ((stride[-1] == 1 or shape[-1] == 1) and all(n <= 1 or s % 8 == 0 for n, s in zip(shape, stride[:-1]))
            and 128 * row + group * head < 2 ** 30)


def _strides(shape, stride):
    """(sequence, row, head) strides; 0 along an axis of one (or none)."""
    s = tuple(0 if n <= 1 else k for n, k in zip(shape[:-1], stride))
    return s if len(s) == 3 else (0, *s)


class _Plan:
    """How calls on operands of one layout go.  ``fits``: which operands can be read where they lie; ``native``: the library's
    arguments and workspaces, where all can."""

    def __init__(self, q, k, v, causal, scale, sequences):
        _check(q, k, v, scale, sequences)
        group = q.shape[-2] // k.shape[-2]
        self.fits = tuple(_fits(x.shape, x.stride(), heads) for x, heads in ((q, group), (k, 1), (v, 1)))
        self.native = self._native(q, k, v, causal, scale, sequences) if all(self.fits) else None

    @staticmethod
    def _native(q, k, v, causal, scale, sequences):
        a = _lib.MsdAttn()
        if sequences is None:
            a.n_seqs, a.q_len, a.k_len = q.shape[0] if q.dim() == 4 else 1, q.shape[-3], k.shape[-3]
        else:
            a.n_seqs, a.q_len, a.k_len = sequences.n, sequences.q_longest, sequences.k_longest
            host = sequences.host.clone()   # (the plan's own: its workspaces are as large as these numbers ask)
            a.seqs, a.seqs_host = sequences.table.data_ptr() or 16, host.data_ptr() or 16   # (16: nothing to read)
        a.q_rows, a.k_rows = math.prod(q.shape[:-2]), math.prod(k.shape[:-2])
        a.n_heads, a.n_kv_heads, a.d_head, a.causal, a.scale = q.shape[-2], k.shape[-2], q.shape[-1], causal, scale
        for name, x in (("q_stride", q), ("k_stride", k), ("v_stride", v)):
            getattr(a, name)[:] = _strides(x.shape, x.stride())
        sizes = [_lib.check(_lib.lib().msd_attn_workspace_bytes(ctypes.byref(a), i), "msd_attn_workspace_bytes") for i in (0, 1)]
        if sequences is None:
            return _lib.ops().AttnPlan(ctypes.addressof(a), *sizes, False, False, None, None, 0)
        return _lib.ops().AttnPlan(ctypes.addressof(a), *sizes, sequences.q_count != q.shape[0], sequences.k_count != k.shape[0],
                                   sequences.table, host, sequences.stream or 0)


_plans = {}   # of calls without sequences; a Sequences keeps its own (the layers of a step make the same call)


def _plan(q, k, v, causal, scale, sequences):
    key = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype, q.device, k.device,
           v.device, causal, scale)
    plans = _plans if sequences is None else sequences._plans
    found = plans.get(key)
    if found is None:
        found = _Plan(q, k, v, causal, scale, sequences)
        if len(plans) >= 256:
            plans.clear()
        plans[key] = found
    return found


def _check(q, k, v, scale, sequences):
    if q.dim() not in (3, 4) or k.dim() != q.dim() or v.shape != k.shape:
        raise ValueError(f"q (batch, rows, heads, d_head) or (rows, heads, d_head) and k, v alike expected, got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        raise ValueError("q, k and v must be bfloat16")
    if not (q.is_cuda and k.is_cuda and v.is_cuda) or not q.device == k.device == v.device:
        raise ValueError("q, k and v must be on one GPU")
    D, H, KV = q.shape[-1], q.shape[-2], k.shape[-2]
    if k.shape[-1] != D or D % 8 or not 0 < D <= 128:
        raise ValueError(f"d_head must be a multiple of 8 up to 128, the same for q, k and v (got {D} and {k.shape[-1]})")
    if KV == 0 or H == 0 or H % KV or H > 4096:
        raise ValueError(f"n_heads ({H}) must be a multiple of n_kv_heads ({KV}), up to 4096")
    if not 2.0 ** -60 <= scale <= 2.0 ** 60:
        raise ValueError(f"scale must lie in [2 ** -60, 2 ** 60] (got {scale})")
    if q.dim() == 4 and q.shape[0] != k.shape[0]:
        raise ValueError(f"q holds {q.shape[0]} sequences, k and v {k.shape[0]}")
    if sequences is not None:
        if q.dim() != 3:
            raise ValueError("sequences go with flat q (rows, heads, d_head)")
        if sequences.q_end > q.shape[0] or sequences.k_end > k.shape[0]:
            raise ValueError(f"sequences reach row {sequences.q_end} of {q.shape[0]} query rows and row "
                             f"{sequences.k_end} of {k.shape[0]} key rows")
        if sequences.table.device != q.device:
            raise ValueError(f"sequences were made for {sequences.table.device}, q is on {q.device}")


def attention(q, k, v, causal=True, scale=None, sequences=None):
    """softmax(scale q k^T) v for every head, q head h with k/v head h // (n_heads // n_kv_heads).

    q (batch, Tq, n_heads, d_head), k and v (batch, Tk, n_kv_heads, d_head), or without the batch axis one sequence, or
    with ``sequences`` (a ``Sequences``) several in flat tensors; bf16 on one GPU, any strides, d_head a multiple of 8 up
    to 128.  ``causal``: query i sees keys 0 .. Tk - Tq + i (the last query the last key, as one token sees its cache).
    A query that sees nothing has output 0.  ``scale`` defaults to d_head ** -0.5.  Returns q's shape, contiguous.

    What lies behind a sequence's own rows is not read.  Within a sequence, a key or value row that is not finite
    reaches every query that sees it, and may reach those that do not; a row of the incoming gradient likewise the
    gradients of keys and values (a masked probability is a zero that is multiplied)."""
    scale = q.shape[-1] ** -0.5 if scale is None and q.dim() and q.shape[-1] else float(scale or 0)
    plan = _plan(q, k, v, bool(causal), scale, sequences)
    if plan.native is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        q, k, v = (x if f and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)
                   for x, f in zip((q, k, v), plan.fits))
        plan = _plan(q, k, v, bool(causal), scale, sequences)
    return _lib.ops().attention(q, k, v, plan.native)
