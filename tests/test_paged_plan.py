"""How a step over pages is shared out (msd_paged_plan), and what the paged cache's calls refuse, on the CPU: nothing reaches a
device."""
import ctypes
import random

import numpy as np
import pytest
import torch

from transformer_amd import _lib
from transformer_amd.paged_attention import PagedEviction, PagedSequences, paged_append, paged_attention, paged_evict

# words of a plan: the public ones, then the launches' sizes and where the lists lie; those of few rows for calls without and with weights
(MAGIC, WORDS, SEQS, HEADS, KV_HEADS, WIDTH, LONGEST, Q_END, Q_COUNT, PAGES, SHARED, RESERVED,
 N_MANY, N_FEWS, N_TILES, N_MANYS, N_APPENDS, MANY_PARTS, FEW_ROWS, SCORES,
 AT_SEQS, AT_MANY, AT_TILES, AT_MANYS, AT_APPENDS, AT_TABLES, N_FEW) = range(27)
FEW_PARTS, AT_FEW, AT_FEWS, END = N_FEW + 2, N_FEW + 4, N_FEW + 6, N_FEW + 8


def tables_of(lengths, seed=0):
    order = list(range(sum(-(-n // 16) for n in lengths) + 2))
    random.Random(seed).shuffle(order)
    return [[order.pop() for _ in range(-(-n // 16))] for n in lengths]


def entries(w, at, n, each=8):
    return [w[at + each * i:at + each * i + each] for i in range(n)]


def covered(jobs, parts, slot, tiles):
    """Jobs of one list of tiles: slots slot .. slot + parts, its tiles once, in order, none empty unless there are none."""
    jobs = sorted(jobs, key=lambda j: j[7])
    assert [j[7] for j in jobs] == list(range(slot, slot + parts))
    assert jobs[0][5] == 0 and jobs[-1][6] == tiles and all(a[6] == b[5] for a, b in zip(jobs, jobs[1:]))
    assert all(j[5] < j[6] for j in jobs)


def check(q_lens, lengths, H, KV, longest=None, starts=None):
    tables = tables_of(lengths)
    s = PagedSequences(q_lens, lengths, tables, H, KV, longest=longest, q_starts=starts, device="cpu")
    w, g, n = s.host.tolist(), H // KV, len(q_lens)
    assert len(w) == w[WORDS] and torch.equal(s.host, s.table) and w[SEQS:WIDTH] == [n, H, KV]
    assert w[LONGEST] == (longest or max(lengths, default=0)) == s.longest and w[Q_COUNT] == sum(q_lens) and w[Q_END] == s.q_end
    width, starts = w[WIDTH], s.q_starts
    assert width % 4 == 0 and w[AT_TABLES] % 4 == 0
    for b, t in enumerate(entries(w, w[AT_TABLES], n, width)):
        assert t == tables[b] + [0] * (width - len(tables[b]))
    assert [x[:3] for x in entries(w, w[AT_SEQS], n, 4)] == [[a, q, L] for a, q, L in zip(starts, q_lens, lengths)]
    assert w[PAGES] == max([p + 1 for t in tables for p in t], default=0) and not w[SHARED]
    # few rows
    for c in (0, 1):
        jobs = [j for j in entries(w, w[AT_FEW + c], w[N_FEW + c]) if j[3] >= 0]
        fews = entries(w, w[AT_FEWS + c], w[N_FEWS])
        slots, scores = 0, 0
        assert [f[3] for f in fews] == [b for b in range(n) if q_lens[b] * g <= 32]
        for q0, q, L, b, slot, parts, at, _ in fews:
            assert [q0, q, L] == [starts[b], q_lens[b], lengths[b]] and slot == slots and at == scores
            slots, scores = slots + parts, scores + q * g * -(-(longest or L) // 32)
            mine = [j for j in jobs if j[3] == b]
            assert all(j[:4] == [q0, q, L, b] and j[4] == 2 * at + (parts == 1) for j in mine) and (q > 0) == (parts > 0)
            assert q * g <= w[FEW_ROWS]
            if parts:
                covered(mine, parts, slot, -(-L // 32))
                assert parts == 1 or w[FEW_PARTS + c]
        assert slots == len(jobs) <= w[N_FEW + c] and scores == w[SCORES]
    # many
    jobs = [j for j in entries(w, w[AT_MANY], w[N_MANY]) if j[3] >= 0]
    tiles = entries(w, w[AT_TILES], w[N_TILES])
    many = [b for b in range(n) if q_lens[b] * g > 32]
    assert [m[:4] for m in entries(w, w[AT_MANYS], w[N_MANYS])] == [[starts[b], q_lens[b], lengths[b], b] for b in many]
    assert sorted((t[3], t[4]) for t in tiles) == [(b, r) for b in many for r in range(0, q_lens[b] * g, 128)]
    slots = 0
    for q0, q, L, b, row0, slot, parts, _ in tiles:
        assert [q0, q, L] == [starts[b], q_lens[b], lengths[b]] and slot == slots and parts > 0
        slots += parts
        seen = L - q + 1 + (min(row0 + 128, q * g) - 1) // g
        covered([j for j in jobs if j[3] == b and j[4] == (-row0 - 1 if parts == 1 else row0)], parts, slot, -(-seen // 64))
        assert parts == 1 or w[MANY_PARTS]
    assert slots == len(jobs) <= w[N_MANY]
    # appended rows: each once, in its place
    where = {}
    for row, count, at, _ in entries(w, w[AT_APPENDS], w[N_APPENDS], 4):
        assert 0 <= count <= 16 and at % 16 + count <= 16
        for i in range(count):
            assert row + i not in where
            where[row + i] = at + i
    want = {starts[b] + i: 16 * tables[b][(lengths[b] - q + i) // 16] + (lengths[b] - q + i) % 16 for b, q in enumerate(q_lens) for i in range(q)}
    assert where == want
    return w


@pytest.mark.parametrize("seed", range(60))
def test_any_step(seed):
    r = random.Random(seed)
    KV = r.choice([1, 2, 3, 8])
    H = KV * r.choice([1, 2, 3, 4, 8, 33])
    n = r.choice([1, 2, 7, 40])
    q_lens = [r.choice([0, 1, 1, 1, 4, r.randint(1, 600)]) for _ in range(n)]
    lengths = [q + r.choice([0, 1, 15, 16, r.randint(0, 5000)]) for q in q_lens]
    starts = None
    if r.random() < 0.4:   # in another order, with room between
        starts, at = [0] * n, r.randint(0, 5)
        for b in r.sample(range(n), n):
            starts[b], at = at, at + q_lens[b] + r.randint(0, 3)
    plain = check(q_lens, lengths, H, KV, starts=starts)
    longest = max(max(lengths) + r.randint(0, 700), 1)
    roomy = check(q_lens, lengths, H, KV, longest=longest, starts=starts)
    assert all(roomy[i] >= plain[i] for i in (N_FEW, N_FEW + 1, N_MANY))


@pytest.mark.parametrize("seed", range(30))
def test_room_for_other_lengths(seed):
    """Plans of the same new tokens and room have one size and the same launches, at any lengths."""
    r = random.Random(seed)
    KV = r.choice([1, 2, 4, 8])
    H, n, longest = KV * r.choice([1, 4, 7]), r.choice([1, 5, 33]), r.choice([40, 700, 20000])
    q_lens = [min(longest, r.choice([0, 1, 1, 5, r.randint(1, 400)])) for _ in range(n)]
    same = (*range(WORDS, Q_COUNT + 1), *range(RESERVED, END))
    plans = []
    for kind in range(4):
        lengths = [(q, longest, r.randint(q, longest), r.choice([q, longest]))[kind] for q in q_lens]
        plans.append(check(q_lens, lengths, H, KV, longest=longest))
    assert all([p[i] for i in same] == [plans[0][i] for i in same] for p in plans)


def test_update():
    s = PagedSequences([1, 3], [5, 40], [[3], [0, 1, 2]], 4, 2, longest=100, device="cpu")
    host, table = s.host.data_ptr(), s.table.data_ptr()
    s.update([17, 100], [[3, 4], [0, 1, 2, 5, 6, 7, 8]])
    want = PagedSequences([1, 3], [17, 100], [[3, 4], [0, 1, 2, 5, 6, 7, 8]], 4, 2, longest=100, device="cpu")
    assert torch.equal(s.host, want.host) and torch.equal(s.table, want.host) and (s.host.data_ptr(), s.table.data_ptr()) == (host, table)
    assert s.lengths == [17, 100] and s.version == 1 and s.used().tolist() == list(range(9))
    for lengths, tables in (([17, 101], [[3, 4], range(10)]), ([17], [[3, 4]]), ([0, 3], [[], [1]]), ([17, 33], [[3, 4], [1, 2]]), ([5, 40], [[3], [0, 1, -2]])):
        with pytest.raises(ValueError):
            s.update(lengths, tables)
        assert torch.equal(s.host, want.host) and torch.equal(s.table, want.host) and s.lengths == [17, 100] and s.version == 1
    with pytest.raises(ValueError, match="longest"):
        PagedSequences([1], [5], [[3]], 4, 2, device="cpu").update([6], [[3]])


@pytest.mark.parametrize("args,kw,match", [
    (([-1], [3], [[0]], 4, 2), {}, "negative"),
    (([1], [3, 4], [[0]], 4, 2), {}, "lengths"),
    (([4], [3], [[0]], 4, 2), {}, "counts the new tokens"),
    (([1], [17], [[0]], 4, 2), {}, "pages where"),
    (([1], [17], [[0, -1]], 4, 2), {}, "outside"),
    (([1], [17], [[0, 2 ** 27]], 4, 2), {}, "outside"),
    (([1], [17], [[0, 1.5]], 4, 2), {}, "whole"),
    (([1], [17], [[0, 1], [2]], 4, 2), {}, "1 sequences"),
    (([1], [17], np.zeros((1, 2)), 4, 2), {}, "integers"),
    (([1], [17], np.zeros(2, np.int32), 4, 2), {}, "integers"),
    (([1.5], [17], [[0, 1]], 4, 2), {}, "whole"),
    (([1], [17], [[0, 1]], 4, 3), {}, "multiple"),
    (([1], [17], [[0, 1]], 4, 0), {}, "multiple"),
    (([1], [17], [[0, 1]], 8192, 1), {}, "multiple"),
    (([1], [17], [[0, 1]], 4, 2), dict(longest=16), "outside"),
    (([1], [17], [[0, 1]], 4, 2), dict(longest=0), "longest"),
    (([1, 1], [17, 1], [[0, 1], [2]], 4, 2), dict(q_starts=[0]), "starts"),
    (([2, 1], [17, 1], [[0, 1], [2]], 4, 2), dict(q_starts=[0, 1]), "overlap"),
    (([1], [2 ** 31 - 1], [range(3)], 4, 2), {}, "outside"),
])
def test_sequences(args, kw, match):
    with pytest.raises(ValueError, match=match):
        PagedSequences(*args, **kw, device="cpu")


def test_tables_of_any_kind():
    lists = PagedSequences([1, 1], [20, 3], [[4, 5], [7]], 4, 2, device="cpu")
    for t in (np.array([[4, 5, 0], [7, -1, -1]]), torch.tensor([[4, 5], [7, 2 ** 30]], dtype=torch.int32), [torch.tensor([4, 5]), np.array([7], np.int16)], [range(4, 6), (7,)]):
        assert torch.equal(PagedSequences([1, 1], [20, 3], t, 4, 2, device="cpu").host, lists.host)


@pytest.mark.parametrize("q_lens,lengths,tables,shared", [
    ([1, 1], [20, 20], [[0, 1], [0, 2]], 0),     # a full page of a prompt
    ([1, 1], [20, 20], [[0, 1], [0, 1]], 1),
    ([0, 1], [20, 20], [[0, 1], [0, 1]], 1),     # the other reads it
    ([0, 0], [20, 20], [[0, 1], [0, 1]], 0),
    ([5, 1], [20, 20], [[0, 1], [0, 2]], 1),     # five rows reach back into the first page
    ([1], [33], [[0, 0, 1]], 0),
    ([1], [33], [[1, 0, 1]], 1),
    ([1, 1], [16, 20], [[0, 1], [1, 2]], 0),     # a page behind a length is not in use
])
def test_pages_that_take_rows_and_are_shared(q_lens, lengths, tables, shared):
    assert PagedSequences(q_lens, lengths, tables, 4, 2, device="cpu").host[SHARED] == shared


@pytest.mark.parametrize("keep,recent,tables,match", [
    (16, 17, [[5], [6]], "recent"),
    (16, -1, [[5], [6]], "recent"),
    (32, 0, [[5], [6]], "pages where"),
    (32, 0, [[5, 7], [6, 5]], "twice"),
    (32, 0, [[5, 7], [6, 1]], "sequences use"),
    (32, 0, [[5, 7]], "2 sequences"),
    (32, 0, [[5, 7], [6, -1]], "outside"),
])
def test_evictions(keep, recent, tables, match):
    s = PagedSequences([1, 0], [40, 30], [[0, 1, 2], [1, 3]], 4, 2, device="cpu")
    with pytest.raises(ValueError, match=match):
        PagedEviction(s, keep, recent, tables)


def test_an_eviction():
    s = PagedSequences([1, 0], [40, 10], [[0, 1, 2], [1]], 4, 2, device="cpu")
    e = PagedEviction(s, 24, 8, [[9, 8], [5, 0]])
    assert e.lengths == [24, 10] and e.table.tolist() == [[9, 8], [5, -1]] and e.pages == 10


def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


K = _x(2, 64, 64)


@pytest.mark.parametrize("k,v,match", [
    (_x(64, 64), _x(64, 64), "one shape"),
    (K, _x(2, 48, 64), "one shape"),
    (_x(2, 40, 64), _x(2, 40, 64), "multiple of 16"),
    (_x(2, 64, 64, dtype=torch.float16), K, "bfloat16"),
    (_x(2, 64, 60), _x(2, 64, 60), "d_head"),
    (_x(2, 64, 136), _x(2, 64, 136), "d_head"),
    (_x(3, 64, 64), _x(3, 64, 64), "heads"),
    (K, K, "GPU"),
])
def test_pages(k, v, match):
    s = PagedSequences([1], [3], [[0]], 4, 2, device="cpu")
    with pytest.raises(ValueError, match=match):
        paged_attention(_x(1, 4, 64), k, v, s)
    with pytest.raises(ValueError, match=match):
        paged_append(_x(1, 2, 64), _x(1, 2, 64), k, v, s)
    with pytest.raises(ValueError, match=match):
        paged_evict(k, v, torch.zeros(1, 2, 3), PagedEviction(s, 2, 1, [[1]]))


# ---- the C entries ----

def _call(**kw):
    s = PagedSequences(kw.pop("q_lens", [3]), kw.pop("lengths", [40]), kw.pop("tables", [[0, 1, 2]]), 4, 2, device="cpu")
    a = _lib.MsdPaged()
    a.d_head, a.scale, a.q_rows, a.positions, a.plan, a.plan_host = 64, 0.125, 3, 64, 16, s.host.data_ptr()
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = (256, 64), (4096, 64), (4096, 64)
    for name, x in kw.items():
        if "stride" in name:
            getattr(a, name)[:] = x
        else:
            setattr(a, name, x)
    return s, a


BAD = [dict(d_head=0), dict(d_head=136), dict(d_head=60), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q_rows=2),
       dict(q_rows=-1), dict(q_rows=2 ** 30), dict(positions=32), dict(positions=50), dict(positions=2 ** 31), dict(q_stride=(257, 64)), dict(q_stride=(256, -8)),
       dict(q_stride=(2 ** 25, 64)), dict(k_stride=(4096, 60)), dict(k_stride=(-8, 64)), dict(v_stride=(4100, 64)), dict(v_stride=(4096, 2 ** 27)),
       dict(k_stride=(2 ** 41, 64))]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_c_calls_outside_the_limits(bad):
    keep, a = _call(**bad)
    L, p = _lib.lib(), ctypes.byref(a)
    stride = (ctypes.c_int64 * 2)(128, 64)
    assert L.msd_paged_attn_workspace_bytes(p, 0) == _lib.MSD_E_CONFIG
    assert L.msd_paged_attn(p, 256, 256, 256, 256, None, 0, None, 256, None) == _lib.MSD_E_CONFIG
    assert L.msd_paged_append(p, 256, stride, 256, stride, 256, 256, None) == _lib.MSD_E_CONFIG
    assert L.msd_paged_evict(p, 1, 0, 0, 256, 256, 256, 40, 16, 4, 256, 1, 256, 256, None) == _lib.MSD_E_CONFIG


def test_c_calls_with_bad_pointers():
    keep, a = _call(q_lens=[30], lengths=[40], q_rows=30)
    L, p, A = _lib.lib(), ctypes.byref(a), _lib.MSD_E_ARG
    stride, odd = (ctypes.c_int64 * 2)(128, 64), (ctypes.c_int64 * 2)(130, 64)
    for i in range(4):
        ptrs = [256] * 4
        for bad in (None, 264):
            ptrs[i] = bad
            assert L.msd_paged_attn(p, *ptrs, None, 0, None, 256, None) == A
            assert L.msd_paged_append(p, ptrs[0], stride, ptrs[1], stride, ptrs[2], ptrs[3], None) == A
    assert L.msd_paged_attn(p, 256, 256, 256, 256, None, 5, 256, 256, None) == A     # weights are missing
    assert L.msd_paged_attn(p, 256, 256, 256, 256, 258, 5, 256, 256, None) == A
    assert L.msd_paged_attn(p, 256, 256, 256, 256, 256, 5, 258, 256, None) == A
    assert L.msd_paged_attn(p, 256, 256, 256, 256, 256, 5, 256, None, None) == A     # the workspace is
    assert L.msd_paged_attn(p, 256, 256, 256, 256, 256, -1, 256, 256, None) == _lib.MSD_E_CONFIG
    assert L.msd_paged_append(p, 256, None, 256, stride, 256, 256, None) == A
    assert L.msd_paged_append(p, 256, odd, 256, stride, 256, 256, None) == _lib.MSD_E_CONFIG
    evict = lambda k=256, v=256, w=256, to=256, out=256, kept=256, keep=16, recent=4, width=1, layers=1, layer=0: L.msd_paged_evict(  # noqa: E731
        p, layers, layer, layer, k, v, w, 40, keep, recent, to, width, out, kept, None)
    for name in ("k", "v", "w", "to", "out", "kept"):
        assert evict(**{name: None}) == A and evict(**{name: 257}) == A
    for bad in (dict(recent=17), dict(recent=-1), dict(keep=17), dict(keep=-1, recent=-1), dict(width=-1), dict(layers=-1), dict(layers=32768), dict(layer=4), dict(layer=-8)):
        assert evict(**bad) == _lib.MSD_E_CONFIG, bad
    for field in ("plan", "plan_host"):
        keep, a = _call(**{field: None})
        assert L.msd_paged_attn_workspace_bytes(ctypes.byref(a), 0) == A
    keep, a = _call()
    keep.host[0] = 0   # not a plan
    assert L.msd_paged_attn_workspace_bytes(ctypes.byref(a), 0) == A and L.msd_paged_attn_workspace_bytes(None, 0) == A


def test_c_plans_outside_the_limits():
    L = _lib.lib()
    plan = lambda seqs, pages, width, H=4, KV=2, longest=0, n=1, words=None, room=0, pages_at=None: L.msd_paged_plan(  # noqa: E731
        n, (ctypes.c_int32 * len(seqs))(*seqs), pages_at or (ctypes.c_int32 * max(len(pages), 1))(*pages), width, H, KV, longest, words, room)
    C, A = _lib.MSD_E_CONFIG, _lib.MSD_E_ARG
    n = plan((0, 1, 20), (0, 1), 2)
    assert n > 40 and plan((0, 1, 20), (0, 1), 2, words=(ctypes.c_int32 * n)(), room=n) == n
    assert plan((0, 1, 20), (0, 1), 2, words=(ctypes.c_int32 * n)(), room=n - 1) == A
    assert plan((0, 1, 20), (0, -1), 2, words=(ctypes.c_int32 * n)(), room=n) == C
    for seqs, kw in (((-1, 1, 20), {}), ((0, -1, 20), {}), ((0, 21, 20), {}), ((0, 1, 33), {}), ((0, 1, 20), dict(longest=19)), ((0, 1, 20), dict(longest=40)),
                     ((0, 1, 20), dict(KV=3)), ((0, 1, 20), dict(H=0)), ((0, 1, 20), dict(H=8192)), ((0, 1, 20), dict(longest=-1)), ((0, 1, 20), dict(n=-1)),
                     ((0, 1, 20), dict(n=70000)), ((2 ** 31 - 1, 1, 20), {})):
        assert plan(seqs, (0, 1), 2, **kw) == C, (seqs, kw)
    assert plan((0, 2 ** 29, 2 ** 29), (0, 1), 2 ** 26) == C   # the rows of a group
    # a launch's threads: pages that take new rows; few and many rows together (2^24 pieces and a little more, either alone fewer)
    assert plan((0, 2 ** 28 - 16, 2 ** 28 - 16), (), 2 ** 24, H=1, KV=1, pages_at=256) > 0
    assert plan((0, 2 ** 28, 2 ** 28), (), 2 ** 24, H=1, KV=1, pages_at=256) == C
    few, many = [(i, 1, 16) for i in range(1800)], [(2000 + 40 * i, 40, 48) for i in range(600)]
    for seqs, ok in ((few, True), (many, True), (few + many, False)):
        assert (plan(sum(seqs, ()), (), 3, H=4096, KV=4096, n=len(seqs), pages_at=256) > 0) == ok
    assert L.msd_paged_plan(1, None, (ctypes.c_int32 * 2)(), 2, 4, 2, 0, None, 0) == A
    assert L.msd_paged_plan(1, (ctypes.c_int32 * 3)(0, 1, 20), None, 2, 4, 2, 0, None, 0) == A
    assert L.msd_paged_plan(0, None, None, 0, 4, 2, 0, None, 0) == 40
