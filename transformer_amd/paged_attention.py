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
keys with the running maximum and sum of the softmax, on the matrix cores; f32 scores, statistics and sums; as
operands of the product with the values the probabilities are two bf16 (32 rows of a K/V head's group and fewer; 2^-17) or
rounded to one; in the weights they are f32; the output is rounded to bf16 once.  Deterministic.  No gradients.
"""
import numpy as np
import torch

from . import _lib
from .attention import _ranges
from .paged import PAGE

LONGEST = 2 ** 31 - 2 ** 16 - 1   # positions of a sequence
PAGES = 2 ** 27 - 1               # of a pool


def _words(q_lens, lengths, q_starts, tables, n_heads, n_kv_heads, longest):
    """The library's plan of a step as an int32 tensor on the host."""
    seqs = np.array([q_starts, q_lens, lengths], np.int32).reshape(3, -1).T.copy()
    n, width = tables.shape
    args = n, seqs.ctypes.data, tables.ctypes.data, width, n_heads, n_kv_heads, longest
    words = torch.empty(_lib.check(_lib.lib().msd_paged_plan(*args, None, 0), "msd_paged_plan"), dtype=torch.int32)
    _lib.check(_lib.lib().msd_paged_plan(*args, words.data_ptr(), words.numel()), "msd_paged_plan")
    return words


def _integers(x, what):
    x = x.tolist() if isinstance(x, (torch.Tensor, np.ndarray)) else x
    out = [int(n) for n in x]
    if any(a != b for a, b in zip(out, x)):
        raise ValueError(f"{what} must be whole numbers")
    return out


def _tables(tables, needed, what):
    """The tables of pages as one int32 array, each at least as long as `needed` says; what lies behind that is 0."""
    if isinstance(tables, torch.Tensor):
        tables = tables.cpu().numpy()
    whole = isinstance(tables, np.ndarray)
    if whole and (tables.ndim != 2 or tables.dtype.kind not in "iu"):
        raise ValueError(f"{what} must be a list of page numbers for each sequence, or a table of integers")
    if len(tables) != len(needed):
        raise ValueError(f"{len(tables)} {what} for {len(needed)} sequences")
    width = max(needed, default=0)
    short = next(((len(pages), n) for pages, n in zip(tables, needed) if len(pages) < n), None)
    if short:
        raise ValueError("%s: %d pages where %d are needed" % (what, *short))
    if whole:
        out = np.where(np.arange(width) < np.asarray(needed, np.int64).reshape(-1, 1), tables[:, :width], 0)
    else:
        out = np.zeros((len(needed), width), np.int64)
        for row, pages, n in zip(out, tables, needed):
            pages = np.asarray(pages[:n])
            if n and pages.dtype.kind not in "iu":
                raise ValueError(f"{what} must be whole numbers")
            row[:n] = pages
    if out.size and not (0 <= out.min() and out.max() < PAGES):
        raise ValueError(f"{what}: page numbers outside [0, {PAGES})")
    return np.ascontiguousarray(out, np.int32)


class PagedSequences:
    """Which rows of flat q (rows, n_heads, d_head) and k, v (rows, n_kv_heads, d_head) tensors are which sequence's newest tokens, and
    where its cached positions lie.

    Sequence s has ``q_lens[s]`` new tokens (0, 1 or more) in the rows from ``q_starts[s]`` (packed one behind the other unless
    given), the last of its ``lengths[s]`` positions, so a length counts the new tokens; position p lies in page
    ``tables[s][p // 16]``, slot ``p % 16``.  Sequences may share pages that they only read.  Host integers, checked here; the
    device copy is made on the current stream.

    ``longest``: room for lengths up to it, and ``update``: the object, and a captured graph that reads it, then goes on with the
    lengths and pages of the next step (the launches are those of the longest lengths, what has no work ends at once).  A
    captured graph's object has to be kept, and made before the capture.  A replay checks nothing: pages that take new rows must
    still be in use by one sequence only, pages outside the pool read as zeros and are not written, and a captured eviction
    is of the lengths and pages that it was made for."""

    def __init__(self, q_lens, lengths, tables, n_heads, n_kv_heads, q_starts=None, longest=None, device="cuda"):
        self.q_lens = _integers(q_lens, "lengths")
        self.q_starts, self.q_end, self.q_count = _ranges(self.q_lens, None if q_starts is None else _integers(q_starts, "starts"), "q")
        self.n, self.n_heads, self.n_kv_heads = len(self.q_lens), int(n_heads), int(n_kv_heads)
        if self.n_kv_heads < 1 or self.n_heads < 1 or self.n_heads % self.n_kv_heads or self.n_heads > 4096:
            raise ValueError(f"n_heads ({n_heads}) must be a multiple of n_kv_heads ({n_kv_heads}), up to 4096")
        if longest is not None and not 1 <= longest <= LONGEST:
            raise ValueError(f"longest must lie in [1, {LONGEST}] (got {longest})")
        self._reserved = 0 if longest is None else int(longest)
        self.host, self.lengths, self.longest, self._pages = self._plan(lengths, tables)
        self.table = self.host.to(device)
        self.stream = _lib.current_stream(self.table)
        self.native, self.version = _lib.ops().PagedSteps(self.table, self.host, self.stream or 0), 0

    def _plan(self, lengths, tables):
        """(the library's words, lengths, longest, pages) of a step."""
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
        return words, lengths, self._reserved or max(lengths, default=0), pages

    def update(self, lengths, tables):
        """The same sequences' next step: new lengths and pages, as many new tokens in the same rows.  Ordered on the current stream, on
        which the calls have to be."""
        if not self._reserved:
            raise ValueError("update needs room: give the sequences a longest length")
        words, *state = self._plan(lengths, tables)
        self.table.copy_(words)   # (first: where this fails, as in a capture, nothing has changed)
        self.host.copy_(words)
        self.lengths, self.longest, self._pages = state
        self.version += 1

    def used(self):
        """The pages in use, in order, without repetitions."""
        return np.unique(self._pages[np.arange(self._pages.shape[1]) * PAGE < np.asarray(self.lengths, np.int64).reshape(-1, 1)])


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
        there = np.arange(pages.shape[1]) < np.asarray(needed, np.int64).reshape(-1, 1)
        flat = pages[there]
        if len(np.unique(flat)) != len(flat):
            raise ValueError("tables: a page is named twice")
        if len(np.intersect1d(flat, sequences.used())):
            raise ValueError("tables: a page that the sequences use")
        self.pages = int(flat.max(initial=-1)) + 1
        host = np.full((sequences.n, -(-self.keep // PAGE)), -1, np.int32)   # (-1: not written)
        host[:, :pages.shape[1]][there] = flat
        self.table = torch.from_numpy(host).to(sequences.table.device)
        self.stream = _lib.current_stream(self.table)


def paged_append(k, v, k_pages, v_pages, sequences):
    """Writes the new tokens' keys and values (rows, n_kv_heads, d_head; bf16, any strides) to their positions of the pages
    (n_kv_heads, positions, d_head; on 16-byte boundaries, strides that are multiples of 8; no two places of the keys and the values in
    one memory).  Pages that take new rows must be in use by one sequence only.  k and v may lie in the pages themselves: they are
    read before any page is written."""
    _lib.ops().paged_append(k, v, k_pages, v_pages, sequences.native)


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
    out = _lib.ops().paged_attention(q, k_pages, v_pages, sequences.native, scale, weights)
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
    return tuple(_lib.ops().paged_evict(k_pages, v_pages, weights, sequences.native, eviction.table, eviction.stream or 0, eviction.pages,
                                        eviction.keep, eviction.recent))
