"""Rotary positions, RMSNorm with the residual's addition and SwiGLU on the GPU, forward and gradients, against the
formulas in 64 bits.

Tolerances, element by element: u = half a step of the result's type (bf16 2^-8, f32 2^-24, relative) for the one rounding,
and for the 32-bit arithmetic before it e = 2^-19 of the sum of the magnitudes that enter: a row's sum goes through at
most 16 + 6 + 16 additions (2^-24 each, 2^-18.7, halved by the square root), the exponentials, quotients and products
that follow add some 8 roundings.  Sums over rows: at most 1 + rows / 256 + 4 + 32 + 16 additions, 2^-18 for up to 2000 rows.
Angles: reduced in f64, rounded to f32 as turns (2 pi 2^-25), cosine and sine to 2 ulp: below 2^-20.
"""
import math

import pytest
import torch

from transformer_amd.attention import attention
from transformer_amd.norm import rms_norm
from transformer_amd.rotary import RotaryFrequencies, rotary, rotary_frequencies
from transformer_amd.swiglu import swiglu

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
E, ROWS_E, ANGLE_E = 2.0 ** -19, 2.0 ** -18, 2.0 ** -20
BF, F32 = torch.bfloat16, torch.float32


def _rand(shape, seed, dtype=BF, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype).cuda()


def _near(got, ref, tol, what):
    got = got.double()
    assert torch.isfinite(got).all(), what
    over = (got - ref).abs() - tol - 1e-36
    if over.numel():
        i = int(over.argmax())
        assert float(over.max()) <= 0, (what, i, float(got.flatten()[i]), float(ref.flatten()[i]), float(tol.flatten()[i]))


def _int8(x):
    """The checkpoint's values of x (f32 arithmetic, as it is defined), one step of each, and whether a quotient lies so
    near the middle of two integers (2^-10) that 32 bits may round it to either."""
    n, d = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -d % 128)).reshape(n, -1, 128)
    top = b.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, 127)   # (a tensor: torch divides by or into a number through a rounded reciprocal)
    q = b * (most / torch.where(top < 2.0 ** -100, 1, top))
    step = torch.where(top < 2.0 ** -100, 0, top / most).expand_as(b)
    tie = (q - q.floor() - 0.5).abs() < 2.0 ** -10
    return [y.reshape(n, -1)[:, :d].double() for y in (torch.round(q) * step, step, tie)]


# ---- RMSNorm ----

def _rms(rows, d, dtype=BF, residual=True, keep=None, scale_dtype=None, seed=0, use_sum=True, spread=1.0):
    x, r = _rand((rows, d), seed, dtype, 0.5 * spread), _rand((rows, d), seed + 1, dtype, 2.0 * spread)
    w = (1 + 0.2 * _rand((d,), seed + 2, F32)).to(scale_dtype or dtype)
    dy, ds = _rand((rows, d), seed + 3, dtype), _rand((rows, d), seed + 4, dtype)
    x.requires_grad_(), w.requires_grad_(), r.requires_grad_()
    if residual:
        y, s = rms_norm(x, w, r, checkpoint=keep)
        outs, grads = ((y, s), (dy, ds)) if use_sum else ((y,), (dy,))
        dx, dr, dw = torch.autograd.grad(outs, (x, r, w), grads)
        assert torch.equal(dx, dr)
        assert torch.equal(s, (x.float() + r.float()).to(dtype))
        s = s.detach().double()
    else:
        y, use_sum = rms_norm(x, w, checkpoint=keep), False
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        s = x.detach().double()
    u, w64, dy = U[dtype], w.detach().double(), dy.double()
    rstd = 1 / ((s * s).mean(1, keepdim=True) + 1e-5).sqrt()
    n = s * rstd
    _near(y.detach(), n * w64, (u + E) * (n * w64).abs(), "y")
    off = torch.zeros_like(n)
    if keep:
        n, step, tie = _int8(n)
        off = step * tie + E * (n.abs() + step)
    t = dy * w64
    m = (t * n).mean(1, keepdim=True)
    add = ds.double() if use_sum else 0 * n
    ref = rstd * (t - n * m) + add
    tol = u * ref.abs() + E * (rstd * (t.abs() + n.abs() * (t * n).abs().mean(1, keepdim=True)) + add.abs())
    tol = tol + rstd * (off * m.abs() + n.abs() * (t.abs() * off).mean(1, keepdim=True))
    _near(dx, ref, tol, "dx")
    ref = (dy * n).sum(0)
    _near(dw, ref, U[w.dtype] * ref.abs() + ROWS_E * (dy * n).abs().sum(0) + (dy.abs() * off).sum(0), "dscale")
    plain = rms_norm(x.detach(), w.detach(), r.detach()) if residual else rms_norm(x.detach(), w.detach())
    assert torch.equal(plain[0] if residual else plain, y.detach())


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 7), (5, 8), (3, 64), (17, 511), (1, 512), (33, 513), (300, 768), (2000, 1024),
                                    (50, 1025), (40, 2048), (7, 3001), (12, 4096), (5, 4097), (9, 8192), (3, 16383), (2, 16384)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rms_norm(rows, d, dtype):
    _rms(rows, d, dtype, seed=d)


@pytest.mark.parametrize("rows,d", [(1, 1), (5, 130), (300, 1024), (7, 1000), (6, 2049), (3, 5000)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [True, False])
def test_rms_norm_int8_checkpoint(rows, d, dtype, residual):
    _rms(rows, d, dtype, residual, "int8", seed=d)


@pytest.mark.parametrize("kw", [dict(residual=False), dict(use_sum=False), dict(scale_dtype=F32), dict(spread=1e-4),
                                dict(spread=1e4), dict(dtype=F32, scale_dtype=BF)])
def test_rms_norm_forms(kw):
    _rms(37, 1000, seed=3, **kw)


def test_rms_norm_zero_rows_and_shapes():
    x = torch.zeros((2, 3, 64), dtype=BF, device="cuda").requires_grad_()
    w = torch.ones(64, dtype=BF, device="cuda").requires_grad_()
    y = rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert y.shape == dx.shape == x.shape and not y.any() and not dw.any()
    _near(dx, torch.full(x.shape, 1e-5 ** -0.5, dtype=torch.float64, device="cuda"), torch.full_like(dx.double(), 2.0), "dx")
    x = torch.zeros((0, 64), dtype=BF, device="cuda").requires_grad_()
    for keep in (None, "int8"):
        dx, dw = torch.autograd.grad(rms_norm(x, w, checkpoint=keep), (x, w), torch.zeros((0, 64), dtype=BF, device="cuda"))
        assert dx.shape == (0, 64) and not dw.any()
    for keep in (None, "int8"):   # rows of zeros among others keep their place in the checkpoint
        x = _rand((4, 200), 1)
        x[1:3] = 0
        x.requires_grad_()
        w = torch.ones(200, dtype=BF, device="cuda")
        dx, = torch.autograd.grad(rms_norm(x, w, checkpoint=keep), x, torch.ones((4, 200), dtype=BF, device="cuda"))
        assert torch.isfinite(dx).all()


def test_rms_norm_only_one_output_used():
    x, r = (_rand((5, 96), i).requires_grad_() for i in range(2))
    w = torch.ones(96, dtype=BF, device="cuda").requires_grad_()
    _, s = rms_norm(x, w, r)
    dx, dr, dw = torch.autograd.grad(s, (x, r, w), torch.ones_like(s), allow_unused=True)
    assert torch.equal(dx, torch.ones_like(x)) and torch.equal(dr, dx) and (dw is None or not dw.any())


def test_rms_norm_strided_and_unaligned():
    """Column slices, transposed batches, rows off any boundary: the bits of contiguous copies."""
    big = _rand((6, 5, 300), 1)
    w = _rand((101,), 2)
    for x in (big[:, :, 7:108], big.transpose(0, 1)[:, :, 3:104], big[:, 2, 1:102], big[..., 0:202:2]):
        r = torch.empty(x.numel() + 1, dtype=BF, device="cuda")[1:].view(x.shape).copy_(x * 2)
        dy = _rand((*x.shape[:-1], 202), 3)[..., ::2]
        got, want = [], []
        for to, f in ((got, lambda t: t), (want, lambda t: t.contiguous().clone())):
            leaves = [f(t).detach().requires_grad_() for t in (x, r, w)]
            y, s = rms_norm(leaves[0], leaves[2], leaves[1])
            to += [y, s, *torch.autograd.grad((y, s), leaves, (f(dy), f(dy)))]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rms_norm_frozen_scale_and_shared_scale():
    x, w, dy = _rand((9, 64), 1).requires_grad_(), _rand((64,), 2), _rand((9, 64), 3)
    a, = torch.autograd.grad(rms_norm(x, w), x, dy)
    w.requires_grad_()
    b, dw = torch.autograd.grad(rms_norm(x, w), (x, w), dy)
    assert torch.equal(a, b)
    two, = torch.autograd.grad((rms_norm(x, w), rms_norm(x, w)), w, (dy, dy))
    assert torch.equal(two, dw + dw)


def test_not_finite():
    """A NaN stays in its row (its 128 values of an 8-bit checkpoint) and reaches the scale's gradient."""
    x, w = _rand((4, 256), 1), _rand((256,), 2)
    x[2, 5] = math.nan
    for keep in (None, "int8"):
        leaf = x.clone().requires_grad_()
        y = rms_norm(leaf, w, checkpoint=keep)
        dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        for t in (y, dx):
            assert torch.isnan(t[2]).all() and torch.isfinite(t[[0, 1, 3]]).all()
    g, u = _rand((3, 300), 3), _rand((3, 300), 4)
    g[1, 130] = math.inf
    u[2, 299] = math.nan
    leaves = [t.clone().requires_grad_() for t in (g, u)]
    y = swiglu(*leaves, checkpoint="int8")
    dg, du = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert torch.isnan(dg[1, 128:256]).all() and torch.isnan(du[1, 128:256]).all() and torch.isfinite(dg[1, :128]).all()
    assert torch.isnan(dg[2, 256:]).all() and torch.isfinite(dg[0]).all() and torch.isfinite(du[2]).all()
    assert torch.isfinite(y[0]).all()


# ---- SwiGLU ----

def _glu(g, u, dy, keep=None):
    dtype = g.dtype
    leaves = [t.detach().requires_grad_() for t in (g, u)]
    y = swiglu(*leaves, checkpoint=keep)
    dg, du = torch.autograd.grad(y, leaves, dy)
    assert y.is_contiguous() and torch.equal(y.detach(), swiglu(g, u))
    e, h = U[dtype], E
    a, b, d = (t.double() for t in (g, u, dy))
    ref = a * torch.sigmoid(a) * b
    _near(y.detach(), ref, (e + h) * ref.abs(), "y")
    if keep:
        a, b = (_int8(t.reshape(-1, t.shape[-1]))[0].reshape(t.shape) for t in (g, u))
    s = torch.sigmoid(a)
    ref = d * b * (s + a * s * (1 - s))
    _near(dg, ref, e * ref.abs() + h * (d * b).abs() * s * (1 + a.abs()), "dgate")
    ref = d * a * s
    _near(du, ref, (e + h) * ref.abs(), "dup")
    return y.detach(), dg, du


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (1, 8), (509, 704), (5, 127), (2, 128), (9, 129), (64, 2816), (3, 10001),
                                    (700, 33)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("keep", [None, "int8"])
def test_swiglu(rows, d, dtype, keep):
    _glu(_rand((rows, d), d, dtype, 2.0), _rand((rows, d), d + 1, dtype), _rand((rows, d), d + 2, dtype), keep)


@pytest.mark.parametrize("keep", [None, "int8"])
def test_swiglu_large_and_small_gates(keep):
    """Gates whose exponential overflows, where 1 + exp(-g) is g's own size or 1; denormals; blocks of zeros."""
    g = torch.tensor([-1e4, -200.0, -89.0, -20.0, -1.28, -1e-3, -1e-38, 0.0, 1e-38, 1e-3, 1.0, 17.0, 100.0, 1e4], dtype=BF,
                     device="cuda").repeat(3, 20)
    g[1] = 0
    _glu(g, _rand(g.shape, 1), _rand(g.shape, 2), keep)


@pytest.mark.parametrize("keep", [None, "int8"])
def test_swiglu_halves_of_one_projection(keep):
    for shape, d in (((3, 50, 2 * 96), 96), ((40, 2 * 131), 131)):
        both, dy = _rand(shape, 1), _rand((*shape[:-1], d), 2)
        got = _glu(both[..., :d], both[..., d:], dy, keep)
        want = _glu(both[..., :d].contiguous(), both[..., d:].contiguous(), dy, keep)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = torch.zeros((0, 8), dtype=BF, device="cuda")
    leaf = empty.clone().requires_grad_()
    assert torch.autograd.grad(swiglu(leaf, empty, checkpoint=keep), leaf, empty)[0].shape == (0, 8)


def test_the_checkpoint_lets_go_of_the_activations():
    """With an 8-bit checkpoint, what a SwiGLU and a norm hold on to for the backward is half of bf16 and 1/32 more."""
    held = []
    for keep in (None, "int8"):
        g, u, r = (_rand((256, 4096), i).requires_grad_() for i in range(3))
        w = _rand((4096,), 4).requires_grad_()
        g, u, r, saved = g * 1, u * 1, r * 1, []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
            y = swiglu(g, u, checkpoint=keep)
            n, _ = rms_norm(r, w, r, checkpoint=keep)
        # (summed here: the allocator's own figure counts the whole of a block whose rest is too small to split off)
        held.append(sum(t.nbytes for t in saved))
    saved = 256 * 4096 * (2 - 1 - 4 / 128) * 3
    assert abs(held[0] - held[1] - saved) < 1e5, held


# ---- rotary positions ----

def _turn(x, pos, turns, amplitude, rot, layout, sign):
    """(rotated x, sum of the magnitudes that enter) in 64 bits; pos (..., tokens)."""
    x = x.double()
    a = (pos.double()[..., None] * turns) % 1.0 * (2 * math.pi) * sign
    c, s = a.cos().unsqueeze(-2) * amplitude, a.sin().unsqueeze(-2) * amplitude
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    y, m = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    m[..., i] = m[..., j] = amplitude * (x[..., i].abs() + x[..., j].abs())
    return y, m


def _rot(B, T, H, KV, D, rot, layout, dtype=BF, pos="start", seed=0, freq=None, strided=False, first=0):
    freq = freq or rotary_frequencies(rot)
    qkv = _rand((B, T, H + 2 * KV + 1, D), seed, dtype)
    q, k = qkv[:, :, :H], qkv[:, :, H:H + KV]
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    dq, dk = _rand((B, T, H, D), seed + 1, dtype), _rand((B, T, KV, D), seed + 2, dtype)
    g = torch.Generator().manual_seed(seed)
    p, at = None, torch.arange(first, first + T, device="cuda").expand(B, T)
    if pos != "start":
        kind = torch.int64 if pos.endswith("64") else torch.int32
        p = torch.randint(-1000, 2 ** 31 - 1 if pos.startswith("far") else 5000, (B, T), generator=g, dtype=torch.int64).to(kind).cuda()
        if pos.startswith("row"):
            p = p[0]
        at = p.expand(B, T)
    leaves = [t.detach().requires_grad_() for t in (q, k)]
    out = rotary(*leaves, freq, p, start=first, layout=layout)
    got = [*out, *torch.autograd.grad(out, leaves, (dq, dk))]
    u = U[dtype]
    for x, y, sign, what in ((q, got[0], 1, "q"), (k, got[1], 1, "k"), (dq, got[2], -1, "dq"), (dk, got[3], -1, "dk")):
        ref, m = _turn(x, at, freq.turns, freq.amplitude, rot, layout, sign)
        assert torch.equal(y[..., rot:], x[..., rot:]) and y.is_contiguous()
        _near(y.detach(), ref, u * ref.abs() + ANGLE_E * m, what)
    return got


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,T,H,KV,D,rot", [(1, 1, 1, 1, 2, 2), (2, 5, 3, 1, 64, 64), (1, 9, 4, 4, 128, 64), (3, 8, 2, 1, 80, 40),
                                            (1, 17, 2, 2, 96, 48), (2, 7, 5, 1, 33, 30), (1, 3, 1, 1, 6, 4), (1, 200, 16, 4, 64, 64),
                                            (1, 3, 2, 1, 512, 512)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary(B, T, H, KV, D, rot, layout, dtype):
    _rot(B, T, H, KV, D, rot, layout, dtype, seed=D)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("pos", ["near", "far", "far64", "row", "row64"])
def test_rotary_positions(layout, pos):
    """int32 and int64, per batch and shared, negative and up to 2^31: an f64 product of 2^31 with a turn of 1/6 is off by
    2^-23 of a turn's 2^-24."""
    _rot(3, 11, 4, 2, 64, 64, layout, F32, pos=pos, seed=7)
    _rot(3, 11, 4, 2, 64, 32, layout, BF, pos=pos, seed=8, strided=True)


def test_rotary_start_strides_and_no_k():
    _rot(2, 6, 4, 2, 64, 64, "half", first=100000)
    a = _rot(2, 6, 4, 2, 64, 64, "half", strided=True)
    b = _rot(2, 6, 4, 2, 64, 64, "half", strided=False)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    q, f = _rand((5, 3, 64), 1), rotary_frequencies(64)
    assert torch.equal(rotary(q, None, f), rotary(q, q, f)[0])
    assert torch.equal(rotary(q, None, f), rotary(q[None], None, f)[0])
    assert torch.equal(rotary(q, None, f), rotary(q, None, f, torch.arange(5, device="cuda")))
    odd = torch.empty(q.numel() + 1, dtype=BF, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(rotary(odd, None, f), rotary(q, None, f))
    turned = q.transpose(-1, -2).contiguous().transpose(-1, -2)
    assert torch.equal(rotary(turned, None, f), rotary(q, None, f))
    leaf = q.clone().requires_grad_()
    d, = torch.autograd.grad(rotary(leaf, None, f).sum(), leaf)
    assert d.shape == q.shape
    assert rotary(q[:0], q[:0], f)[0].shape == (0, 3, 64)
    one = _rand((1, 4, 64), 2).expand(5, -1, -1)
    assert torch.equal(rotary(one, None, f), rotary(one.contiguous(), None, f))
    x, y = (_rand((4, 2, 64), i).requires_grad_() for i in (3, 4))   # only one of the two is used, or wanted
    out = rotary(x, y, f)
    d, = torch.autograd.grad(out[0], x, torch.ones_like(out[0]))
    assert torch.isfinite(d).all()
    out = rotary(x, y.detach(), f)
    e, = torch.autograd.grad(out[0], x, torch.ones_like(out[0]))
    assert torch.equal(d, e)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
                                dict(scaling="by_parts", factor=8.0, original_context=2048), dict(base=500000.0)])
def test_rotary_scaled(kw):
    _rot(2, 9, 4, 2, 64, 64, "half", F32, pos="far", freq=rotary_frequencies(64, **kw))


def test_rotary_past_32_bit_offsets():
    """Tokens whose elements lie past 2^31 of a strided tensor."""
    big = torch.empty((40000, 60000), dtype=BF, device="cuda")
    q = big[:, 100:228].view(40000, 2, 64)
    q.copy_(_rand(q.shape, 1))
    assert torch.equal(rotary(q, None, rotary_frequencies(64)), rotary(q.contiguous(), None, rotary_frequencies(64)))
    w = torch.ones(128, dtype=BF, device="cuda")
    assert torch.equal(rms_norm(big[:, 100:228], w), rms_norm(big[:, 100:228].contiguous(), w))
    assert torch.equal(swiglu(big[:, 100:228], big[:, 100:228]), swiglu(*(big[:, 100:228].contiguous(),) * 2))


# ---- all of them ----

def _step(x, w, norm, freq, keep):
    from transformer_amd.attention import attention
    h = rms_norm(x, norm, checkpoint=keep)
    q, k, v = (h @ w["qkv"]).unflatten(-1, (8, 64)).split((4, 2, 2), -2)
    q, k = rotary(q, k, freq)
    a = attention(q, k, v).flatten(-2) @ w["o"]
    h, x = rms_norm(a, norm, x, checkpoint=keep)
    g, u = (h @ w["gu"]).chunk(2, -1)
    return rms_norm(swiglu(g, u, checkpoint=keep) @ w["down"], norm, x, checkpoint=keep)[0]


def _layer_inputs(seed):
    w = {n: _rand(s, seed + i, spread=0.05).requires_grad_()
         for i, (n, s) in enumerate(dict(qkv=(256, 512), o=(256, 256), gu=(256, 1408), down=(704, 256)).items())}
    norm = (1 + 0.1 * _rand((256,), seed + 9, F32)).to(BF).requires_grad_()
    return _rand((2, 70, 256), seed + 8).requires_grad_(), w, norm, _rand((2, 70, 256), seed + 7)


def _layer_grads(x, w, norm, dy, freq, keep):
    y = _step(x, w, norm, freq, keep)
    return [y.detach(), *torch.autograd.grad(y, (x, norm, *w.values()), dy)]


@pytest.mark.parametrize("keep", [None, "int8"])
def test_a_layer_of_them(keep):
    """Norm, rotary positions, attention and feed-forward of one layer and the loss on top, as a training step runs them:
    the gradients against the same layer in 64 bits, to 3 % of their norm (a chain of about 12 bf16 roundings of half a
    step each way, 24 * 2^-8 / sqrt(3) if all added up; 8-bit checkpoints 1/254 more at three places)."""
    from transformer_amd.xent import fused_output_and_loss
    freq = rotary_frequencies(64)
    x, w, norm, _ = _layer_inputs(1)
    emb, target = _rand((500, 256), 50, spread=0.05).requires_grad_(), torch.randint(0, 500, (2, 70), generator=torch.Generator().manual_seed(1))
    leaves = (x, norm, *w.values(), emb)
    loss = fused_output_and_loss(_step(x, w, norm, freq, keep), emb, target.cuda())
    got = torch.autograd.grad(loss, leaves)

    X, N, *W, M = (t.detach().double().requires_grad_() for t in leaves)
    W = dict(zip(w, W))

    def rms(t):
        return t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * N

    a = torch.arange(70, dtype=torch.float64, device="cuda")[:, None] * freq.turns * 2 * math.pi
    c, s = a.cos()[:, None], a.sin()[:, None]
    q, k, v = (rms(X) @ W["qkv"]).unflatten(-1, (8, 64)).split((4, 2, 2), -2)
    q, k = (torch.cat((t[..., :32] * c - t[..., 32:] * s, t[..., :32] * s + t[..., 32:] * c), -1) for t in (q, k))
    q, k, v = q.transpose(1, 2), *(t.transpose(1, 2).repeat_interleave(2, 1) for t in (k, v))
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) / 8
    p = torch.softmax(p.masked_fill(torch.ones(70, 70, device="cuda").triu(1).bool(), -math.inf), -1)
    R = X + torch.matmul(p, v.contiguous()).transpose(1, 2).flatten(-2) @ W["o"]
    g, u = (rms(R) @ W["gu"]).chunk(2, -1)
    z = rms(R + (g * torch.sigmoid(g) * u) @ W["down"]) @ M.T
    want = torch.nn.functional.cross_entropy(z.flatten(0, 1), target.flatten().cuda())
    assert abs(float(loss.detach()) - float(want.detach())) < 0.03 * float(want.detach())
    for a, b in zip(got, torch.autograd.grad(want, (X, N, *W.values(), M))):
        assert float((a.double() - b).norm()) <= 0.03 * float(b.norm())


@pytest.mark.parametrize("keep", [None, "int8"])
def test_streams_threads_and_repetition(keep):
    """Equal bits from call to call, on two streams at once and from two threads."""
    import threading
    freq = rotary_frequencies(64)
    xs = [_layer_inputs(100 * (i + 1)) for i in range(2)]
    alone = [_layer_grads(*x, freq, keep) for x in xs]
    torch.cuda.synchronize()
    got, errors = [[], []], []
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_layer_grads(*xs[i], freq, keep))
    torch.cuda.synchronize()

    def work(i):
        try:
            for _ in range(4):
                got[i].append(_layer_grads(*xs[i], freq, keep))
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(2):
        assert len(got[i]) == 8 and all(torch.equal(a, b) for r in got[i] for a, b in zip(r, alone[i]))


@pytest.mark.parametrize("keep", [None, "int8"])
def test_captured_and_replayed(keep):
    """The operators of a layer, forward and backward, in a graph, replayed over new inputs with eager work between."""
    freq = rotary_frequencies(64)

    def run(x, w, r, dy, q, k):
        leaves = [t.detach().requires_grad_() for t in (x, w, r, q, k)]
        y, s = rms_norm(leaves[0], leaves[1], leaves[2], checkpoint=keep)
        z = swiglu(y, s, checkpoint=keep)
        a, b = rotary(leaves[3], leaves[4], freq)
        return [y.detach(), s.detach(), *torch.autograd.grad((z, a, b), leaves, (dy, q, k))]

    def inputs(i):
        return [_rand(s, 10 * i + j) for j, s in enumerate(((90, 333), (333,), (90, 333), (90, 333), (20, 4, 64), (20, 2, 64)))]

    static = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*static)
    for i in range(1, 5):
        new = inputs(i)
        for s, t in zip(static, new):
            s.copy_(t)
        graph.replay()
        want = run(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_frequencies_object():
    f = rotary_frequencies(64)
    q = _rand((3, 2, 64), 1)
    assert torch.equal(rotary(q, None, f), rotary(q, None, RotaryFrequencies(f.turns)))


def _strided_calls():
    """(operator, its strided leaves): each reads them where they lie."""
    freq = rotary_frequencies(64)
    both, wide = _rand((40, 512), 1), _rand((6, 50, 8, 64), 2)
    q, k, v = wide[:, :, :4], wide[:, :, 4:6], wide[:, :, 6:]
    return [
        (lambda g, u: swiglu(g, u), (both[:, :256], both[:, 256:])),
        (lambda x, w: rms_norm(x, w), (both[:, :200], _rand((200,), 3))),
        (lambda x, w, r: sum(rms_norm(x, w, r, checkpoint="int8")), (both[:, :200], _rand((200,), 3), both[:, 300:500])),
        (lambda q, k, v: attention(q, k, v), (q, k, v)),
        (lambda q, k: sum(t.sum(2) for t in rotary(q, k, freq)), (q, k)),
    ]


@pytest.mark.parametrize("which", range(5))
def test_saved_tensors_that_hooks_move(which):
    """What is saved may come back with other strides (here by way of host memory): the same gradients."""
    f, leaves = _strided_calls()[which]
    leaves = [x.detach().requires_grad_() for x in leaves]
    want = torch.autograd.grad(f(*leaves).float().sin().sum(), leaves)
    with torch.autograd.graph.save_on_cpu():
        y = f(*leaves)
    got = torch.autograd.grad(y.float().sin().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", range(5))
def test_second_derivatives_are_refused(which):
    """Gradients may be recorded, and give the same values; differentiating them raises."""
    f, leaves = _strided_calls()[which]
    leaves = [x.detach().requires_grad_() for x in leaves]
    want = torch.autograd.grad(f(*leaves).float().sin().sum(), leaves)
    got = torch.autograd.grad(f(*leaves).float().sin().sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="differentiable once"):
        sum(x.float().sum() for x in got).backward()


@pytest.mark.parametrize("which", range(5))
def test_parts_of_the_gradients_and_twice(which):
    """Only some leaves want gradients; a graph that is kept gives them again; nothing is recorded without a wish for it."""
    f, leaves = _strided_calls()[which]
    whole = [x.detach().requires_grad_() for x in leaves]
    y = f(*whole).float().sin().sum()
    want = torch.autograd.grad(y, whole, retain_graph=True)
    again = torch.autograd.grad(y, whole)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, whole)
    for i in range(len(leaves)):
        some = [x.detach().requires_grad_(i == j) for j, x in enumerate(leaves)]
        got, = torch.autograd.grad(f(*some).float().sin().sum(), some[i:i + 1])
        assert torch.equal(got, want[i])
    with torch.no_grad():
        assert not f(*whole).requires_grad
    with torch.inference_mode():
        assert torch.equal(f(*leaves), f(*whole))


def test_rotary_heads_of_4096():
    """The most cosines and sines that a workgroup keeps."""
    q, freq = _rand((5, 1, 4096), 3), rotary_frequencies(4096)
    got = rotary(q, None, freq, start=7)
    pos = torch.arange(7, 12, dtype=torch.int64, device="cuda")
    turn = (pos.double()[:, None] * freq.turns) % 1.0 * (2 * math.pi)
    a, b = q[:, 0, :2048].double(), q[:, 0, 2048:].double()
    want = torch.cat((a * turn.cos() - b * turn.sin(), a * turn.sin() + b * turn.cos()), -1)
    # the result's rounding, and the f32 angle, cosine and products: a few 2^-24 of the pair
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * torch.cat((a.abs() + b.abs(),) * 2, -1)
    assert ((got[:, 0].double() - want).abs() <= tol).all()
