"""Calls of the paged cache's operators outside the ordinary: traces and derivatives, inference mode, compiled functions, other
streams, other threads, and steps with room for more than they have."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_paged_attention_gpu import near, rand, reference, rows_of, tables_of
from transformer_amd.paged_attention import PagedEviction, PagedSequences, paged_append, paged_attention, paged_evict

pytestmark = pytest.mark.gpu


def _step(seed=0, q_lens=(1, 40), lengths=(100, 90), H=4, KV=2, D=64, **kw):
    b = len(lengths)
    tables, n = tables_of(list(lengths) + [32] * b, seed)
    pool = rand((2, KV, 16 * n, D), seed + 3)
    s = PagedSequences(q_lens, lengths, tables[:b], H, KV, **kw)
    rows = sum(q_lens)
    return s, PagedEviction(s, 32, 8, tables[b:]), pool[0], pool[1], rand((rows, H, D), seed, 1.5), rand((rows, KV, D), seed + 1), rand((rows, KV, D), seed + 2)


def _calls(s, e, kp, vp, q, k, v):
    w = torch.rand((2, 2, 100), generator=torch.Generator().manual_seed(9)).cuda()
    return [(lambda q: paged_attention(q, kp, vp, s), q), (lambda q: paged_attention(q, kp, vp, s, weights=w)[1], q),
            (lambda w: paged_evict(kp, vp, w, e)[0], w), (lambda k: (paged_append(k, v, kp, vp, s), kp)[1], k)]


@pytest.mark.parametrize("which", range(4))
def test_traces_and_derivatives_are_refused(which):
    f, x = _calls(*_step())[which]
    want = f(x).clone()
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        f(fwd.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, (x,), check_trace=False)
    leaf = x.detach().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        f(leaf)
    with torch.no_grad():
        assert torch.equal(f(leaf), want)
    with torch.inference_mode():
        assert torch.equal(f(x), want)
    assert torch.equal(f(x), want)


def test_inference_tensors():
    """Pages made in inference mode: written in it, refused outside before anything runs."""
    s, e, kp, vp, q, k, v = _step(1)
    with torch.inference_mode():
        kp, vp = kp.clone(), vp.clone()
        paged_append(k, v, kp, vp, s)
        want = paged_attention(q, kp, vp, s)
    held = kp.clone()
    with pytest.raises(RuntimeError, match="nference"):
        paged_append(k + 1, v, kp, vp, s)
    assert torch.equal(kp, held) and torch.equal(paged_attention(q, kp, vp, s), want)


@pytest.mark.parametrize("which", range(4))
def test_inside_a_compiled_function(which):
    f, x = _calls(*_step(2))[which]
    torch._dynamo.reset()
    want = f(x * 2).clone()
    assert torch.equal(torch.compile(lambda x: f(x * 2), backend="eager")(x), want)


def test_threads():
    """Two threads on streams of their own, on one step's sequences."""
    s, e, kp, vp, q, k, v = _step(3, (1, 1, 60), (3000, 50, 700), 8, 2, 128)
    want, got = paged_attention(q, kp, vp, s), [[], []]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(paged_attention(q, kp, vp, s))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(x, want) for x in got[0] + got[1])


@pytest.mark.parametrize("longest", [128, 700, 5000])
def test_room_for_more(longest):
    """Launches for longer sequences than there are give what exact ones give, weights behind the lengths being zeros."""
    q_lens, lengths = [1, 3, 60, 0], [128, 5, 61, 17]
    tables, n = tables_of(lengths, 1)
    q, kp, vp = rand((64, 6, 96), 1, 1.5), rand((2, 16 * n, 96), 2), rand((2, 16 * n, 96), 3)
    old = torch.rand((4, 2, 128), generator=torch.Generator().manual_seed(4)).cuda()
    got = paged_attention(q, kp, vp, PagedSequences(q_lens, lengths, tables, 6, 2, longest=longest), weights=old)
    ref, tol = reference(q, kp, vp, q_lens, lengths, tables, [0, 1, 4, 64], 96 ** -0.5, old, longest)
    near(got[0], ref[0], tol[0], "out")
    near(got[1], ref[1], tol[1], "weights")


def test_an_output_layout_of_a_step_in_a_larger_batch():
    """Rows of other requests between a step's own stay zeros in the output, and are neither read nor written by append."""
    s, e, kp, vp, q, k, v = _step(4)
    starts = [50, 3]
    wide = PagedSequences(s.q_lens, s.lengths, s._pages, 4, 2, q_starts=starts)
    place = lambda x: torch.full((60, *x.shape[1:]), float("nan"), dtype=x.dtype, device=x.device)  # noqa: E731
    big = [place(x) for x in (q, k, v)]
    for b, x in zip(big, (q, k, v)):
        b[50:51], b[3:43] = x[:1], x[1:]
    mine = kp.clone(), vp.clone()
    paged_append(k, v, kp, vp, s)
    paged_append(big[1], big[2], *mine, wide)
    assert torch.equal(kp, mine[0]) and torch.equal(vp, mine[1])
    out, want = paged_attention(big[0], kp, vp, wide), paged_attention(q, kp, vp, s)
    assert torch.equal(out[50:51], want[:1]) and torch.equal(out[3:43], want[1:])
    out[50:51] = out[3:43] = 0
    assert not out.any()


def test_an_eviction_of_pages_that_are_appended_to_afterwards():
    """A step on the new pages after an eviction, whose new rows lie behind the kept ones in the last kept page."""
    s, e, kp, vp, q, k, v = _step(5)
    w = torch.rand((2, 2, 100), generator=torch.Generator().manual_seed(1)).cuda()
    left, kept = paged_evict(kp, vp, w, e)
    assert e.lengths == [32, 32]
    tables = e.table.tolist()
    spare = [p for p in range(kp.shape[1] // 16) if p not in {x for t in tables for x in t} | set(s.used().tolist())]
    t2 = [t + [spare[i]] for i, t in enumerate(tables)]
    step = PagedSequences([1, 2], [33, 34], t2, 4, 2)
    before = [rows_of(kp, t, 32) for t in tables]
    paged_append(k[:3], v[:3], kp, vp, step)
    out, counted = paged_attention(q[:3], kp, vp, step, weights=left)
    ref, tol = reference(q[:3], kp, vp, [1, 2], [33, 34], t2, [0, 1], 0.125, left, 34)
    near(out, ref[0], tol[0], "out")
    near(counted, ref[1], tol[1], "weights")
    assert all(torch.equal(rows_of(kp, t, 32), b) for t, b in zip(tables, before))
