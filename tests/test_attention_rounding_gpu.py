"""The byte that attention keeps beside each output for what its rounding to bf16 took off, and what the backward makes of it.

Probabilities that are powers of two are exact in bf16 and so are their products with v in f32; a sum of n of them is off by up to
n 2^-24 of the magnitudes, the join of the parts by 4 more such roundings.  But for that, out with its byte lies within
2^-15 |out| (the byte's step, 2^8 of the 2^23 of an f32 significand) of the exact value, and out alone within 2^-8 (half a bf16
step).
"""
import ctypes

import pytest
import torch

from transformer_amd import _lib
from transformer_amd.attention import attention

pytestmark = pytest.mark.gpu


def _rand(shape, seed, spread=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * spread).to(torch.bfloat16).cuda()


def _struct(q, k, causal):
    a = _lib.MsdAttn()
    (a.n_seqs, a.q_len, a.n_heads, a.d_head), a.k_len, a.n_kv_heads = q.shape, k.shape[1], k.shape[2]
    a.causal, a.scale, a.q_rows, a.k_rows = causal, a.d_head ** -0.5, q.shape[0] * q.shape[1], k.shape[0] * k.shape[1]
    for n, x in (("q_stride", q), ("dout_stride", q), ("k_stride", k), ("v_stride", k)):
        getattr(a, n)[:] = x.stride()[:3]
    return a


def _call(name, a, *tensors):
    L = _lib.lib()
    n = _lib.check(L.msd_attn_workspace_bytes(ctypes.byref(a), name == "backward"), name)
    ws = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
    p = [None if x is None else x.data_ptr() for x in tensors]
    _lib.check(getattr(L, "msd_attn_" + name)(ctypes.byref(a), *p, ws.data_ptr(), _lib.current_stream(ws)), name)


def _forward(q, k, v, causal=False):
    """(out, its bytes, lse) of the C entry point."""
    out, low = torch.empty_like(q), torch.empty(q.shape, dtype=torch.int8, device="cuda")
    lse = torch.empty(q.shape[:3], device="cuda")
    _call("forward", _struct(q, k, causal), q, k, v, out, low, lse)
    return out, low, lse


def _whole(out, low):
    return ((out.view(torch.int16).int() << 16) + (low.int() << 8)).view(torch.float32).double()


@pytest.mark.parametrize("D", [8, 64, 72, 128])
@pytest.mark.parametrize("tq,tk,live", [
    (40, 1, 1), (40, 2, 2), (40, 4, 4), (40, 64, 2), (300, 128, 4),      # one pass
    (3, 256, 2), (3, 512, 4), (3, 1024, 2), (3, 1024, 16), (3, 2048, 4),   # 2, 4, 8 and 16 parts joined
])
def test_outputs_with_their_bytes(D, tq, tk, live):
    """Equal scores (q = 0): every output is a mean, of two or four values often half-way between two bf16."""
    q, k, v = torch.zeros((2, tq, 4, D), dtype=torch.bfloat16, device="cuda"), _rand((2, tk, 2, D), 1), _rand((2, tk, 2, D), 2)
    v[:, torch.randperm(tk, generator=torch.Generator().manual_seed(3))[live:]] = 0
    out, low, _ = _forward(q, k, v)
    mean, size = (x.double().mean(1).repeat_interleave(2, 1)[:, None].expand(q.shape) for x in (v, v.abs()))
    sums = (live + 4) * 2.0 ** -24 * size
    assert ((out.double() - mean).abs() <= 2.0 ** -8 * mean.abs() + sums).all()
    over = (_whole(out, low) - mean).abs() - 2.0 ** -15 * mean.abs() - sums
    assert float(over.max()) <= 0, (float(over.max()), int((over > 0).sum()), over.numel())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tk", [2, 256, 1024])
def test_gradients_of_means_half_way_between_two_values(D, tk):
    """Half of the keys hold 1, half the next bf16, so that every output lies half-way and is rounded down.  With dout = 1, dS = P (dP -
    rowsum) where P = 1 / tk, dP = D or D (1 + 2^-7) and rowsum = D (1 + 2^-8): -+ D 2^-8 / tk, but 0 and D 2^-7 / tk with the
    rounded outputs' rowsum.  All of these are exact in bf16 and f32; the byte may be off by 2^-15, the rowsum by D 2^-15 and dS by
    a 2^-7th of itself; 2^-12 for P's 32 bits, and dq is rounded once (2^-8)."""
    q = torch.zeros((1, 5, 2, D), dtype=torch.bfloat16, device="cuda")
    k, v = _rand((1, tk, 1, D), 1), torch.ones((1, tk, 1, D), dtype=torch.bfloat16, device="cuda")
    v[:, tk // 2:] += 2.0 ** -7
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    out = attention(q, k, v, causal=False)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    ds = torch.full((tk, 1), D * 2.0 ** -8 / tk, dtype=torch.float64, device="cuda")
    ds[:tk // 2] *= -1
    k64, scale = k[0, :, 0].detach().double(), D ** -0.5
    ref, tol = scale * (ds * k64).sum(0), scale * (2.0 ** -7 + 2.0 ** -12) * (ds.abs() * k64.abs()).sum(0)
    assert ((dq.double() - ref).abs() <= tol + 2.0 ** -8 * ref.abs()).all()
    assert not dk.any()   # (q is zero)
    assert ((dv.double() - 10 / tk).abs() <= 2.0 ** -8 * 10 / tk).all()


def test_the_backward_without_the_bytes():
    """out itself will do: D is then off by half a bf16 step of every output, 2^-8 sum |dout out|, on top of what rounding P, dS
    and the results leaves (2^-8 each, and 2^-12 for 32 bits in a probability)."""
    U, E, D = 2.0 ** -8, 2.0 ** -12, 64
    q, k, v, do = (_rand((1, 150, h, D), i) for i, h in enumerate((2, 1, 1, 2)))
    out, low, lse = _forward(q, k, v, causal=True)
    grads = [[torch.empty_like(x) for x in (q, k, v)] for _ in range(2)]
    for g, b in zip(grads, (low, None)):
        _call("backward", _struct(q, k, True), q, k, v, out, b, lse, do, *g)
    assert not torch.equal(grads[0][0], grads[1][0])
    Q, K, V, O = (x[0].double() for x in (q, k, v, do))
    dq, dk, dv, tq, tk, tv = [], 0, 0, [], 0, 0
    for h in range(2):
        s = (Q[:, h] @ K[:, 0].T * D ** -0.5).masked_fill(torch.ones(150, 150, device="cuda").triu(1).bool(), -torch.inf)
        p = torch.softmax(s, -1)
        o, d = p @ V[:, 0], O[:, h]
        ds = p * (d @ V[:, 0].T - (d * o).sum(-1, keepdim=True))
        t_o = (U + E) * (p @ V[:, 0].abs()) + U * o.abs()
        t = p * (d.abs() * t_o).sum(-1, keepdim=True) + (U + 2 * E) * ds.abs() + E * p * (d.abs() @ V[:, 0].abs().T)
        dq.append(D ** -0.5 * ds @ K[:, 0]), tq.append(D ** -0.5 * t @ K[:, 0].abs())
        dk, tk = dk + D ** -0.5 * ds.T @ Q[:, h], tk + D ** -0.5 * t.T @ Q[:, h].abs()
        dv, tv = dv + p.T @ d, tv + (U + E) * (p.T @ d.abs())
    for g in grads:
        for x, ref, tol in zip(g, (torch.stack(dq, 1), dk[:, None], dv[:, None]), (torch.stack(tq, 1), tk[:, None], tv[:, None])):
            assert ((x[0].double() - ref).abs() <= tol + U * ref.abs()).all()
