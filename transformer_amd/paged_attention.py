"""Serving over a paged cache as torch calls: a step's keys and values into their pages, attention of each sequence's newest
tokens over its pages, and eviction of the positions that have received the least attention.

The reference's causal_attention (model.py:122-147) of new tokens over cached keys and values, the cache its paged one
(described in knowledge/program.md:214-216, 245-250): pages of 16 positions in a pool, ``PagePool.view()[layer, 0]`` (keys)
and ``[layer, 1]`` (values), each (n_kv_heads, positions, d_head) bf16, or any tensors of that shape.

  sequences = PagedSequences(q_lens, lengths, tables, n_heads, n_kv_heads)      # once a step, for all layers
  paged_append(k, v, k_pages, v_pages, sequences)
  out = paged_attention(q, k_pages, v_pages, sequences)
  out, weights = paged_attention(q, k_pages, v_pages, sequences, weights=weights)

  eviction = PagedEviction(sequences, keep, recent, tables)                     # other pages
  weights, kept = paged_evict(k_pages, v_pages, weights, eviction)              # a layer's pages, or all layers'

What runs (``msd_paged_append`` / ``msd_paged_attn`` / ``msd_paged_evict``, ``csrc/paged.hip``): attention in one pass over the
keys with the running maximum and sum of the softmax, on the matrix cores; f32 scores, statistics and sums; the
probabilities are rounded to bf16 as operands of the product with the values (not in the weights), the output once to bf16.
Deterministic.  No gradients.
"""
import ctypes

import numpy as np
import torch

from . import _lib
from .attention import _fits, _ranges
from .paged import PAGE

LONGEST = 2 ** 31 - 2 ** 16 - 1   # positions of a sequence


def _words(q_lens, lengths, q_starts, tables, n_heads, n_kv_heads, longest):
    """The library's plan of a step as an int32 tensor on the host."""
    seqs = np.ascontiguousarray(np.stack([np.asarray(x, dtype=np.int32) for x in (q_starts, q_lens, lengths)], 1)) if q_lens else np.zeros((0, 3), np.int32)
    n, width = tables.shape
    args = n, seqs.ctypes.data, tables.ctypes.data, width, n_heads, n_kv_heads, longest
    words = torch.empty(_lib.check(_lib.lib().msd_paged_plan(*args, None, 0), "msd_paged_plan"), dtype=torch.int32)
    _lib.check(_lib.lib().msd_paged_plan(*args, words.data_ptr(), words.numel()), "msd_paged_plan")
    return words


def _integers(x, what):
    out = [int(n) for n in x]
    if any(a != b for a, b in zip(out, x)):
        raise ValueError(f"{what} must be whole numbers")
    return out


def _tables(tables, needed, what):
    """The tables of pages as one int32 array, each at least as long as `needed` says; what lies behind that is not looked at."""
    if isinstance(tables, torch.Tensor):
        tables = tables.cpu().numpy()
    if isinstance(tables, np.ndarray) and (tables.ndim != 2 or tables.dtype.kind not in "iu"):
        raise ValueError(f"{what} must be a list of page numbers for each sequence, or a table of integers")
    if len(tables) != len(needed):
        raise ValueError(f"{len(tables)} {what} for {len(needed)} sequences")
    out = np.zeros((len(needed), max(needed, default=0)), np.int32)
    for row, pages, n in zip(out, tables, needed):
        if len(pages) < n:
            raise ValueError(f"{what}: {len(pages)} pages where {n} are needed")
        pages = np.asarray(pages[:n])
        if n and pages.dtype.kind not in "iu":
            raise ValueError(f"{what} must be whole numbers")
        if n and not (0 <= pages.min() and pages.max() < 2 ** 27 - 1):
            raise ValueError(f"{what}: page numbers outside [0, 2**27 - 1)")
        row[:n] = pages
    return out


class PagedSequences:
    """Which rows of flat q (rows, n_heads, d_head) and k, v (rows, n_kv_heads, d_head) tensors are which sequence's newest tokens, and
    where its cached positions lie.

    Sequence s has ``q_lens[s]`` new tokens (0, 1 or more) in the rows from ``q_starts[s]`` (packed one behind the other unless
    given), the last of its ``lengths[s]`` positions, so a length counts the new tokens; position p lies in page
    ``tables[s][p // 16]``, slot ``p % 16``.  Sequences may share pages that they only read.  Host integers, checked here; the
    device copy is made on the current stream.

    ``longest``: room for lengths up to it, and ``update``: the object, and a captured graph that reads it, then goes on with the
    lengths and pages of the next step (the launches are those of the longest lengths, what has no work ends at once).  A
    captured graph's object has to be kept, and made before the capture."""

    def __init__(self, q_lens, lengths, tables, n_heads, n_kv_heads, q_starts=None, longest=None, device="cuda"):
        self.q_lens = _integers(q_lens, "lengths")
        self.q_starts, self.q_end, self.q_count = _ranges(self.q_lens, None if q_starts is None else _integers(q_starts, "starts"), "q")
        self.n, self.n_heads, self.n_kv_heads = len(self.q_lens), int(n_heads), int(n_kv_heads)
        if self.n_kv_heads < 1 or self.n_heads < 1 or self.n_heads % self.n_kv_heads or self.n_heads > 4096:
            raise ValueError(f"n_heads ({n_heads}) must be a multiple of n_kv_heads ({n_kv_heads}), up to 4096")
        if longest is not None and not 1 <= longest <= LONGEST:
            raise ValueError(f"longest must lie in [1, {LONGEST}] (got {longest})")
        self._reserved = 0 if longest is None else int(longest)
        self.host = self._plan(lengths, tables)
        self.table = self.host.to(device)
        self.stream = _lib.current_stream(self.table)
        self._plans, self.version = {}, 0

    def _plan(self, lengths, tables):
        lengths = _integers(lengths, "lengths")
        if len(lengths) != self.n:
            raise ValueError(f"{self.n} lengths of new tokens, {len(lengths)} lengths")
        if any(n < q for n, q in zip(lengths, self.q_lens)):
            raise ValueError("a length counts the new tokens and cannot be less")
        if max(lengths, default=0) > (self._reserved or LONGEST):
            raise ValueError(f"length {max(lengths)} outside [0, {self._reserved or LONGEST}]")
        pages = _tables(tables, [-(-n // PAGE) for n in lengths], "tables")
        if self._reserved:
            pages = np.pad(pages, ((0, 0), (0, -(-self._reserved // PAGE) - pages.shape[1])))
        words = _words(self.q_lens, lengths, self.q_starts, np.ascontiguousarray(pages), self.n_heads, self.n_kv_heads, self._reserved)
        self.lengths, self.longest, self._pages = lengths, self._reserved or max(lengths, default=0), pages
        return words

    def update(self, lengths, tables):
        """The same sequences' next step: new lengths and pages, as many new tokens in the same rows.  Ordered on the current stream, on
        which the calls have to be."""
        if not self._reserved:
            raise ValueError("update needs room: give the sequences a longest length")
        self.host.copy_(self._plan(lengths, tables))
        self.table.copy_(self.host)
        self.version += 1

    def used(self):
        """The pages in use, in order, without repetitions."""
        return np.unique(np.concatenate([np.zeros(0, np.int32)] + [p[:-(-n // PAGE)] for p, n in zip(self._pages, self.lengths)]))


class PagedEviction:
    """What ``paged_evict`` does to the sequences of a step: each keeps ``min(length, keep)`` positions, the newest ``recent`` among
    them, in the first positions of its pages in ``tables``; these are none that the sequences use, and different from one
    another.  ``lengths``: the lengths afterwards.  Made once, used by every layer."""

    def __init__(self, sequences, keep, recent, tables):
        self.sequences, self.version = sequences, sequences.version
        self.keep, self.recent = int(keep), int(recent)
        if not 0 <= self.recent <= self.keep <= LONGEST:
            raise ValueError(f"0 <= recent <= keep expected (got {recent} and {keep})")
        self.lengths = [min(n, self.keep) for n in sequences.lengths]
        needed = [-(-n // PAGE) for n in self.lengths]
        pages = _tables(tables, needed, "tables")
        flat = np.concatenate([np.zeros(0, np.int32)] + [p[:n] for p, n in zip(pages, needed)])
        if len(np.unique(flat)) != len(flat):
            raise ValueError("tables: a page is named twice")
        if len(np.intersect1d(flat, sequences.used())):
            raise ValueError("tables: a page that the sequences use")
        self.pages = int(flat.max(initial=-1)) + 1
        host = np.full((sequences.n, -(-self.keep // PAGE)), -1, np.int32)   # (-1: not written)
        for row, p, n in zip(host, pages, needed):
            row[:n] = p[:n]
        self.table = torch.from_numpy(host).to(sequences.table.device)
        self.stream = _lib.current_stream(self.table)


def _positions(x):
    return x.shape[-2]


def _check_pages(k_pages, v_pages, sequences, dims, written):
    for x in (k_pages, v_pages):
        if x.dtype != torch.bfloat16:
            raise ValueError("pages must be bfloat16")
    if k_pages.dim() not in dims or k_pages.shape != v_pages.shape or _positions(k_pages) % PAGE:
        raise ValueError(f"pages of one shape (n_kv_heads, positions, d_head), positions a multiple of {PAGE}, expected, got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    D = k_pages.shape[-1]
    if D % 8 or not 0 < D <= 128:
        raise ValueError(f"d_head must be a multiple of 8 up to 128 (got {D})")
    if k_pages.shape[-3] != sequences.n_kv_heads:
        raise ValueError(f"pages of {k_pages.shape[-3]} heads, sequences of {sequences.n_kv_heads}")
    if not k_pages.is_cuda or not k_pages.device == v_pages.device == sequences.table.device:
        raise ValueError(f"pages and sequences must be on one GPU (got {k_pages.device}, {v_pages.device} and {sequences.table.device})")
    for x in (k_pages, v_pages):
        if x.stride(-1) != 1 or any(n > 1 and s % 8 for n, s in zip(x.shape, x.stride()[:-1])) or x.data_ptr() % 16:
            raise ValueError("pages must have contiguous heads on 16-byte boundaries")
        if x.stride(-2) >= 2 ** 25 or any(n > 1 and s >= 2 ** 40 for n, s in zip(x.shape, x.stride()[:-2])):
            raise ValueError("pages: strides out of reach")
        if written:   # no two places of the pages are one
            end = D
            for s, n in sorted((s, n) for s, n in zip(x.stride()[:-1], x.shape[:-1]) if n > 1):
                if s < end:
                    raise ValueError("pages that are written must not overlap")
                end = s * n
    if _positions(k_pages) >= 2 ** 31 or int(sequences.host[9]) > _positions(k_pages) // PAGE:
        raise ValueError(f"tables reach page {int(sequences.host[9]) - 1}, the pages are {_positions(k_pages) // PAGE}")


def _check_new(x, heads, k_pages, sequences, name):
    if x.dim() != 3 or x.shape[1] != heads or x.shape[2] != k_pages.shape[-1]:
        raise ValueError(f"{name} (rows, {heads}, {k_pages.shape[-1]}) expected, got {tuple(x.shape)}")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16")
    if x.device != k_pages.device:
        raise ValueError(f"{name} and the pages must be on one GPU")
    if sequences.q_end > x.shape[0]:
        raise ValueError(f"sequences reach row {sequences.q_end} of {x.shape[0]} rows of {name}")
    if x.shape[0] * sequences.n_heads >= 2 ** 31:
        raise ValueError(f"{name}: rows times heads out of reach")


def _stride(x, axis):
    return x.stride(axis) if x.shape[axis] > 1 else 0


class _Plan:
    """How calls on operands of one layout go.  ``fits``: which new rows can be read where they lie; ``native``: the library's
    arguments, where all can."""

    def __init__(self, new, k_pages, v_pages, sequences, scale=1.0):
        a = _lib.MsdPaged()
        self.fits = tuple(_fits(x.shape, x.stride(), x.shape[1] // (sequences.n_kv_heads if len(new) == 1 else 1)) for x in new)
        a.d_head, a.scale, a.positions = k_pages.shape[-1], scale, _positions(k_pages)
        a.q_rows = new[0].shape[0] if new else sequences.q_end
        if len(new) == 1:
            a.q_stride[:] = _stride(new[0], 0), _stride(new[0], 1)
        a.k_stride[:] = _stride(k_pages, -3), _stride(k_pages, -2)
        a.v_stride[:] = _stride(v_pages, -3), _stride(v_pages, -2)
        a.plan, a.plan_host = sequences.table.data_ptr(), sequences.host.data_ptr()
        new_strides = [(_stride(x, 0), _stride(x, 1)) for x in new] if len(new) == 2 else [(0, 0)] * 2
        self.native = _lib.ops().PagedPlan(ctypes.addressof(a), sequences.table, sequences.host, sequences.stream or 0, *new_strides[0],
                                           *new_strides[1]) if all(self.fits) else None


def _layout(x):
    return x.shape, x.stride(), x.dtype, x.device


def _plan(kind, check, new, k_pages, v_pages, sequences, scale=1.0):
    key = (kind, scale, _layout(k_pages), _layout(v_pages), k_pages.data_ptr() % 16, v_pages.data_ptr() % 16, sequences.version, *map(_layout, new))
    found = sequences._plans.get(key)
    if found is None:
        check()
        found = _Plan(new, k_pages, v_pages, sequences, scale)
        if len(sequences._plans) >= 64:
            sequences._plans.clear()
        sequences._plans[key] = found
    return found


def _operands(new, plan):
    return [x if f and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format) for x, f in zip(new, plan.fits)]


def paged_append(k, v, k_pages, v_pages, sequences):
    """Writes the new tokens' keys and values (rows, n_kv_heads, d_head; bf16, any strides) to their positions of the pages
    (n_kv_heads, positions, d_head; on 16-byte boundaries, strides that are multiples of 8).  Pages that take new rows must be
    in use by one sequence only."""
    def check():
        _check_pages(k_pages, v_pages, sequences, (3,), True)
        for x, name in ((k, "k"), (v, "v")):
            _check_new(x, sequences.n_kv_heads, k_pages, sequences, name)
        if k.shape[0] != v.shape[0]:
            raise ValueError(f"k of {k.shape[0]} rows, v of {v.shape[0]}")
        if int(sequences.host[10]):
            raise ValueError("a page that takes new rows is in use elsewhere too")

    plan = _plan("append", check, (k, v), k_pages, v_pages, sequences)
    if plan.native is None or (k.data_ptr() | v.data_ptr()) % 16:
        k, v = _operands((k, v), plan)
        plan = _plan("append", check, (k, v), k_pages, v_pages, sequences)
    _lib.ops().paged_append(k, v, k_pages, v_pages, plan.native)


def paged_attention(q, k_pages, v_pages, sequences, scale=None, weights=None):
    """softmax(scale q k^T) v of the new tokens over their sequences' positions up to their own: q (rows, n_heads, d_head), any
    strides, query head h with k/v head h // (n_heads // n_kv_heads); bf16 on one GPU, d_head a multiple of 8 up to 128.
    ``scale`` defaults to d_head ** -0.5.  Returns q's shape, contiguous; rows of no sequence are zeros.

    ``weights``: f32 (n, n_kv_heads, width), what each position of a sequence has received so far (positions from width on:
    nothing); then (out, weights) is returned, the weights (n, n_kv_heads, sequences.longest) with what the positions receive in
    this call, the sum of their probabilities over the new tokens and the heads of the group.  New positions start at 0, positions
    behind a length have 0.  The call's memory for a few new tokens of a sequence is 4 bytes for each of their scores.

    What lies behind a sequence's length is not read.  Within it, a key or value row that is not finite reaches every query
    that sees it, and may reach those that do not."""
    scale = q.shape[-1] ** -0.5 if scale is None and q.dim() and q.shape[-1] else float(scale or 0)

    def check():
        _check_pages(k_pages, v_pages, sequences, (3,), False)
        _check_new(q, sequences.n_heads, k_pages, sequences, "q")
        if not 2.0 ** -60 <= scale <= 2.0 ** 60:
            raise ValueError(f"scale must lie in [2 ** -60, 2 ** 60] (got {scale})")

    plan = _plan("attention", check, (q,), k_pages, v_pages, sequences, scale)
    if weights is not None and (weights.dim() != 3 or weights.shape[:2] != (sequences.n, sequences.n_kv_heads) or weights.dtype != torch.float32
                                or weights.device != q.device or weights.shape[2] >= 2 ** 31):
        raise ValueError(f"weights must be float32 ({sequences.n}, {sequences.n_kv_heads}, width) on q's GPU, got {weights.dtype} "
                         f"{tuple(weights.shape)} on {weights.device}")
    if plan.native is None or q.data_ptr() % 16:
        q, = _operands((q,), plan)
        plan = _plan("attention", check, (q,), k_pages, v_pages, sequences, scale)
    out = _lib.ops().paged_attention(q, k_pages, v_pages, weights, plan.native)
    return out[0] if weights is None else tuple(out)


def paged_evict(k_pages, v_pages, weights, eviction):
    """Moves what the eviction keeps to its new pages, for every sequence and K/V head (and layer) by itself: the newest positions, and
    of the others those with the largest weights (of equal ones the lower position; a NaN counts as larger than any number), in
    their order.  Pages (n_kv_heads, positions, d_head), or (layers, ..) of all layers in one call; weights f32 (n, n_kv_heads,
    width) or (layers, ..), positions from width on count as 0.  The old pages are left as they are.

    Returns (weights, kept): the kept positions' weights (.., n_kv_heads, keep) and those positions themselves (int32); 0 and -1
    behind the last."""
    sequences = eviction.sequences
    if sequences.version != eviction.version:
        raise ValueError("the sequences have been updated since the eviction was made")

    def check():
        _check_pages(k_pages, v_pages, sequences, (3, 4), True)
        if eviction.pages > _positions(k_pages) // PAGE:
            raise ValueError(f"tables reach page {eviction.pages - 1}, the pages are {_positions(k_pages) // PAGE}")
        if k_pages.dim() == 4 and k_pages.shape[0] * k_pages.shape[1] >= 65536:
            raise ValueError(f"layers times heads must stay below 65536 (got {k_pages.shape[0]} and {k_pages.shape[1]})")

    plan = _plan(("evict", eviction.pages), check, (), k_pages, v_pages, sequences)
    shape = (*k_pages.shape[:-3], sequences.n, sequences.n_kv_heads)
    if weights.dim() != len(shape) + 1 or tuple(weights.shape[:-1]) != shape or weights.dtype != torch.float32 or weights.device != k_pages.device \
            or weights.shape[-1] >= 2 ** 31:
        raise ValueError(f"weights must be float32 {(*shape, 'width')} on the pages' GPU, got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
    return tuple(_lib.ops().paged_evict(k_pages, v_pages, weights, eviction.table, eviction.keep, eviction.recent, eviction.stream or 0, plan.native))
