"""Calls of the layer operators that their first tests leave out: saved tensors with other strides, forward-mode
differentiation and traces, and norms of so many rows that the backward's workgroups take several each."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_layers_gpu import E, ROWS_E, U, _int8, _near
from transformer_amd.attention import attention
from transformer_amd.norm import rms_norm
from transformer_amd.rotary import rotary, rotary_frequencies
from transformer_amd.swiglu import swiglu

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_rotary_positions_whose_saved_copy_has_other_strides(kind):
    """Strided positions that go to host memory and back between forward and backward come back contiguous."""
    freq, (B, T) = rotary_frequencies(64), (3, 50)
    every = torch.randint(0, 5000, (B, 3 * T), generator=torch.Generator().manual_seed(1)).to(kind).cuda()
    x, dx = _rand((B, T, 4, 64), 2), _rand((B, T, 4, 64), 3)
    for positions in (every[:, ::3], every[:, :T], every[:1, ::3].expand(B, T), every[1, ::3], every.t()[:T, :B].t()):
        grads = []
        for moved in (False, True):
            leaf = x.clone().requires_grad_()
            if moved:
                with torch.autograd.graph.save_on_cpu():
                    y = rotary(leaf, None, freq, positions)
            else:
                y = rotary(leaf, None, freq, positions.contiguous())
            grads += torch.autograd.grad(y, leaf, dx)
        assert torch.equal(*grads)


def _calls():
    freq = rotary_frequencies(64)
    h, x = [_rand((2, 5, 2, 64), i) for i in range(3)], [_rand((5, 64), i) for i in range(3)]
    return [(attention, h), (lambda q, k: rotary(q, k, freq)[0], h[:2]), (lambda q: rotary(q, None, freq), h[:1]),
            (lambda s, w, r: rms_norm(s, w[0], r)[0], x), (lambda s, w: rms_norm(s, w[0], checkpoint="int8"), x[:2]), (swiglu, x[:2])]


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_and_traces_are_refused(which):
    """By the public calls and by the gradients, which then go on as before."""
    f, x = _calls()[which]
    want = f(*x)
    for recorded in (False, True):
        y = [t.detach().requires_grad_(recorded) for t in x]
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            f(fwd.make_dual(y[0], torch.ones_like(y[0])), *y[1:])
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, tuple(y), check_trace=False)
    out = f(*y)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(out, y, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(out, y, torch.ones_like(out)))
    with torch.no_grad():
        assert torch.equal(f(*x), want)


@pytest.mark.parametrize("rows,d", [(8195, 100), (24591, 8), (2051, 1100), (6147, 2049), (515, 4100), (1537, 5000), (513, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("keep", [None, "int8"])
def test_rms_norm_of_several_rows_a_group(rows, d, dtype, keep):
    """At most 512 workgroups of 16, 4 or 1 rows (d up to 1024, 4096, 16384): past 8192, 2048 and 512 rows each takes a second and
    third row, the last with groups that have none.  The scale's gradient then is sums of up to 4 rows a lane, 4 steps of a tree,
    32 parts a lane and 16 lanes: 56 additions of 2^-24 each are within the 2^-18 allowed.  The other tolerances are those of
    test_layers_gpu.py with one term more: a kept value that is off by o (a quotient between two integers, rounded to either) makes
    dx = rstd (t - n m) + ds, m = mean(t n), differ by rstd (o m + n mean(t o) + o mean(t o)), and in short f32 rows the last
    product counts (4e-6 of 4e-4 at 100 values)."""
    x, r = _rand((rows, d), d, dtype) * 0.5, _rand((rows, d), d + 1, dtype) * 2
    w = (1 + 0.2 * _rand((d,), d + 2, torch.float32)).to(dtype)
    dy, ds = _rand((rows, d), d + 3, dtype), _rand((rows, d), d + 4, dtype)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    y, s = rms_norm(*leaves, checkpoint=keep)
    dx, dw, dr = torch.autograd.grad((y, s), leaves, (dy, ds))
    assert torch.equal(dx, dr) and torch.equal(s, (x.float() + r.float()).to(dtype))
    u, w64, t, add = U[dtype], w.detach().double(), dy.double() * w.detach().double(), ds.double()
    rstd = 1 / (s.detach().double().square().mean(1, keepdim=True) + 1e-5).sqrt()
    n = s.detach().double() * rstd
    _near(y.detach(), n * w64, (u + E) * (n * w64).abs(), "y")
    off = torch.zeros_like(n)
    if keep:
        n, step, tie = _int8(n)
        off = step * tie + E * (n.abs() + step)
    m, shift = (t * n).mean(1, keepdim=True), (t.abs() * off).mean(1, keepdim=True)
    ref = rstd * (t - n * m) + add
    tol = u * ref.abs() + E * (rstd * (t.abs() + n.abs() * (t * n).abs().mean(1, keepdim=True)) + add.abs())
    _near(dx, ref, tol + rstd * (off * m.abs() + n.abs() * shift + off * shift), "dx")
    part = dy.double() * n
    _near(dw, part.sum(0), u * part.sum(0).abs() + ROWS_E * part.abs().sum(0) + (dy.double().abs() * off).sum(0), "dscale")


@pytest.mark.parametrize("which", range(7))
def test_saved_tensors_that_hooks_change(which):
    """Other types, shapes or devices raise instead of being read as what was saved; the same values elsewhere do."""
    freq, at = rotary_frequencies(64), torch.arange(10, dtype=torch.int32, device="cuda").reshape(2, 5)
    calls = _calls() + [(lambda q: rotary(q, None, freq, at), [_rand((2, 5, 2, 64), 1)])]
    f, x = calls[which]
    x = [t.detach().requires_grad_() for t in x]
    want = torch.autograd.grad(f(*x), x, torch.ones_like(f(*x)))
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        f(*x)
    for i in range(len(saved)):
        for change in (lambda t: t.cpu(), lambda t: t.reshape(-1)[:-1], lambda t: t.to(torch.float16), lambda t: t.clone(),
                       lambda t: t[None].expand(2, *t.shape).transpose(0, -1).contiguous().transpose(0, -1)[0]):
            n = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: n.append(t) or (len(n) - 1, t), lambda p: change(p[1]) if p[0] == i else p[1]):
                out = f(*x)
            same = (u := change(saved[i])).dtype == saved[i].dtype and u.shape == saved[i].shape and u.is_cuda
            if same:
                assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, x, torch.ones_like(out)), want))
            else:
                with pytest.raises(RuntimeError, match="saved tensor"):
                    torch.autograd.grad(out, x, torch.ones_like(out))


@pytest.mark.parametrize("which", range(7))
def test_inside_a_compiled_function(which):
    """torch.compile breaks its graph at the calls and runs them, with their gradients."""
    at = torch.arange(10, dtype=torch.int32, device="cuda").reshape(2, 5)
    f, x = (_calls() + [(lambda q: rotary(q, None, rotary_frequencies(64), at, layout="interleaved"), [_rand((2, 5, 2, 64), 1)])])[which]
    got = []
    torch._dynamo.reset()
    for g in (f, torch.compile(f, backend="eager")):
        leaves = [t.clone().requires_grad_() for t in x]
        y = g(*[t * 2 for t in leaves])
        got.append([y, *torch.autograd.grad(y, leaves, torch.ones_like(y))])
    assert all(torch.equal(a, b) for a, b in zip(*got))
