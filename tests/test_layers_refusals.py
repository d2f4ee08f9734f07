"""What the layer operators refuse, on the CPU, and the rotary frequencies' formulas."""
import ctypes
import math

import pytest
import torch

from transformer_amd import _lib
from transformer_amd.norm import rms_norm
from transformer_amd.rotary import RotaryFrequencies, rotary, rotary_frequencies
from transformer_amd.swiglu import swiglu


def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("args,kw,match", [
    ((_x(4, 8), _x(7)), {}, "expected"),
    ((_x(4, 0), _x(0)), {}, "16384"),
    ((_x(4, 16385), _x(16385)), {}, "16384"),
    ((_x(4, 8, dtype=torch.float16), _x(8)), {}, "bfloat16 or float32"),
    ((_x(4, 8), _x(8, dtype=torch.float64)), {}, "bfloat16 or float32"),
    ((_x(4, 8), _x(8), _x(3, 8)), {}, "residual"),
    ((_x(4, 8), _x(8), _x(4, 8, dtype=torch.float32)), {}, "residual"),
    ((_x(4, 8), _x(8)), dict(eps=-1.0), "eps"),
    ((_x(4, 8), _x(8)), dict(eps=math.nan), "eps"),
    ((_x(4, 8), _x(8)), dict(checkpoint="int4"), "checkpoint"),
    ((_x(4, 8), _x(8)), {}, "GPU"),
])
def test_rms_norm(args, kw, match):
    with pytest.raises(ValueError, match=match):
        rms_norm(*args, **kw)


@pytest.mark.parametrize("args,kw,match", [
    ((_x(4, 8), _x(4, 9)), {}, "expected"),
    ((_x(4, 0), _x(4, 0)), {}, "expected"),
    ((_x(4, 8), _x(4, 8, dtype=torch.float32)), {}, "expected"),
    ((_x(4, 8, dtype=torch.int32), _x(4, 8, dtype=torch.int32)), {}, "bfloat16 or float32"),
    ((_x(4, 8), _x(4, 8)), dict(checkpoint=8), "checkpoint"),
    ((_x(4, 8), _x(4, 8)), {}, "GPU"),
])
def test_swiglu(args, kw, match):
    with pytest.raises(ValueError, match=match):
        swiglu(*args, **kw)


F = rotary_frequencies(8, device="cpu")


@pytest.mark.parametrize("args,kw,match", [
    ((_x(4, 8), None, F), {}, "expected"),
    ((_x(4, 2, 8), _x(3, 2, 8), F), {}, "k must"),
    ((_x(4, 2, 8), _x(4, 2, 16), F), {}, "k must"),
    ((_x(4, 2, 8), _x(4, 2, 8, dtype=torch.float32), F), {}, "k must"),
    ((_x(4, 2, 8, dtype=torch.float16), None, F), {}, "bfloat16 or float32"),
    ((_x(4, 2, 8), None, F), dict(layout="pairs"), "layout"),
    ((_x(4, 2, 6), None, F), {}, "exceeds"),
    ((_x(4, 2, 8), None, F, torch.arange(3)), {}, "match"),
    ((_x(4, 2, 8), None, F, torch.zeros(4)), {}, "int32 or int64"),
    ((_x(2, 4, 2, 8), None, F, torch.zeros((4, 2), dtype=torch.int32)), {}, "match"),
    ((_x(4, 2, 8), None, F), {}, "GPU"),
])
def test_rotary(args, kw, match):
    with pytest.raises(ValueError, match=match):
        rotary(*args, **kw)


@pytest.mark.parametrize("args,kw", [((7,), {}), ((0,), {}), ((8,), dict(base=1.0)), ((8,), dict(factor=0.5)),
                                     ((8,), dict(scaling="dynamic")), ((2,), dict(scaling="ntk", factor=2.0)),
                                     ((8,), dict(scaling="by_parts", factor=2.0)),
                                     ((8,), dict(scaling="by_parts", factor=2.0, original_context=64, slow=4, fast=4))])
def test_frequencies_refused(args, kw):
    with pytest.raises(ValueError):
        rotary_frequencies(*args, device="cpu", **kw)


def test_frequency_vectors_refused():
    for t in (torch.zeros(4), torch.zeros(0, dtype=torch.float64), torch.zeros((2, 2), dtype=torch.float64)):
        with pytest.raises(ValueError):
            RotaryFrequencies(t)


def test_frequencies():
    def radians(*a, **kw):
        return rotary_frequencies(*a, device="cpu", **kw).turns * 2 * math.pi

    plain = radians(64)
    assert torch.allclose(plain, torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(radians(64, scaling="linear", factor=4.0), plain / 4, rtol=1e-14)
    ntk = radians(64, scaling="ntk", factor=8.0)
    assert abs(float(ntk[0] / plain[0]) - 1) < 1e-14 and abs(float(ntk[-1] * 8 / plain[-1]) - 1) < 1e-12
    parts = rotary_frequencies(64, scaling="by_parts", factor=8.0, original_context=4096, device="cpu")
    n = 4096 * plain / (2 * math.pi)
    ratio = parts.turns * 2 * math.pi / plain
    assert torch.allclose(ratio[n >= 32], torch.ones((), dtype=torch.float64)) and (n >= 32).any()
    assert torch.allclose(ratio[n <= 1], torch.full((), 1 / 8, dtype=torch.float64)) and (n <= 1).any()
    mid = (n > 1) & (n < 32)
    assert mid.any() and torch.allclose(ratio[mid], 1 / 8 + (n[mid] - 1) / 31 * (7 / 8), rtol=1e-12)
    assert abs(parts.amplitude - (0.1 * math.log(8) + 1)) < 1e-12 and rotary_frequencies(8, device="cpu").amplitude == 1.0


def test_c_refusals():
    L, p = _lib.lib(), 4096
    E, A = _lib.MSD_E_CONFIG, _lib.MSD_E_ARG
    fwd = dict(x=p, xs=8, r=None, rs=0, w=p, wt=0, n=4, d=8, t=0, eps=1e-5, y=p, s=None, rstd=None, c=None)
    for bad, code in ((dict(n=-1), E), (dict(d=0), E), (dict(d=16385), E), (dict(t=2), E), (dict(wt=5), E), (dict(n=1 << 31), E),
                      (dict(eps=-1.0), E), (dict(eps=math.nan), E), (dict(xs=-1), E), (dict(x=None), A), (dict(x=4097), A),
                      (dict(w=None), A), (dict(y=None), A), (dict(r=p), A), (dict(s=p), A), (dict(rstd=4098), A), (dict(c=4100), A)):
        assert L.msd_rms_forward(*{**fwd, **bad}.values(), None) == code, bad
    assert L.msd_rms_forward(*{**fwd, "n": 0, "x": None}.values(), None) == 0
    bwd = dict(s=p, ss=8, rstd=p, c=None, w=p, wt=0, dy=p, dys=8, ds=None, dss=0, n=4, d=8, t=0, dx=p, dw=p, ws=p)
    for bad, code in ((dict(d=0), E), (dict(t=7), E), (dict(dys=-8), E), (dict(s=None), A), (dict(rstd=None), A),
                      (dict(dy=None), A), (dict(dx=None), A), (dict(ws=None), A), (dict(c=4100), A), (dict(ds=4097), A)):
        assert L.msd_rms_backward(*{**bwd, **bad}.values(), None) == code, bad
    glu = dict(g=p, gs=8, u=p, us=8, n=4, d=8, t=0, y=p, c=None)
    for bad, code in ((dict(d=0), E), (dict(d=1 << 24), E), (dict(n=-1), E), (dict(n=1 << 40), E), (dict(t=3), E), (dict(us=-1), E),
                      (dict(g=None), A), (dict(u=4097), A), (dict(y=None), A), (dict(c=4104), A)):
        assert L.msd_swiglu_forward(*{**glu, **bad}.values(), None) == code, bad
    gb = dict(g=p, gs=8, u=p, us=8, c=None, dy=p, dys=8, n=4, d=8, t=0, dg=p, du=p)
    for bad, code in ((dict(d=0), E), (dict(g=None), A), (dict(dy=None), A), (dict(dg=None), A), (dict(du=None), A), (dict(c=8), A)):
        assert L.msd_swiglu_backward(*{**gb, **bad}.values(), None) == code, bad
    assert L.msd_checkpoint_bytes(-1, 8) == E and L.msd_checkpoint_bytes(4, 0) == E and L.msd_checkpoint_bytes(1 << 40, 8) == E
    assert L.msd_checkpoint_bytes(4, 130) >= 4 * 256 + 4 * 2 * 4
    assert L.msd_rms_workspace_bytes(1, 0) == E and L.msd_rms_workspace_bytes(100, 64) >= 64 * 4


def test_c_rope_refusals():
    L, p = _lib.lib(), 4096

    def call(q=p, k=p, pos=p, turns=p, q_out=p, k_out=p, **kw):
        r = _lib.MsdRope()
        base = dict(batch=1, tokens=4, n_heads=2, n_kv_heads=1, d_head=64, d_rot=64, interleaved=0, type=0, sign=1,
                    position_bytes=4, amplitude=1.0, start=0)
        for n, v in {**base, **{n: v for n, v in kw.items() if "stride" not in n}}.items():
            setattr(r, n, v)
        for n in ("q_stride", "k_stride"):
            getattr(r, n)[:] = kw.get(n, (512, 128, 64))
        return L.msd_rope_apply(ctypes.byref(r), q, k, pos, turns, q_out, k_out, None)

    E, A = _lib.MSD_E_CONFIG, _lib.MSD_E_ARG
    for kw in (dict(batch=-1), dict(tokens=-1), dict(d_head=0), dict(d_head=5000), dict(d_rot=0), dict(d_rot=3), dict(d_rot=66),
               dict(type=2), dict(sign=0), dict(position_bytes=2), dict(n_heads=5000), dict(n_heads=-1),
               dict(batch=1 << 30, tokens=1 << 20), dict(q_stride=(1, -1, 1))):
        assert call(**kw) == E, kw
    for kw in (dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=4097), dict(pos=None), dict(pos=4098), dict(turns=None),
               dict(turns=4100)):
        assert call(**kw) == A, kw
    assert call(tokens=0, q=None) == 0
    assert L.msd_rope_apply(None, p, p, p, p, p, p, None) == A
