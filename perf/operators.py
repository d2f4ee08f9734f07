"""Performance cases of the training-layer operators: attention, rotary positions, RMSNorm with the
residual's addition and SwiGLU, each forward and backward, with 8-bit activation checkpoints where the
operator offers them, and attention's single-token form over a cache.

``run`` computes a case in plain torch operations in 32 bits, or (``own``) through the framework's
operators; ``exact`` restates the definitions in 64 bits.
"""
import math
import random

import torch

own = False
DEV = "cuda"
EPS = 1e-5
BLOCK = 128          # values of a row that share one scale of an 8-bit checkpoint


def listed():
    return [
        # one token each of four sequences against their cached rows: latency and the cache's bytes
        dict(name="attend_token", kind="attend", batch=4, q=1, k=2000, heads=16, kv=4, d=64, causal=True, cache=True,
             train=False, docs=0),
        # a training step of the 306M model's attention: full contexts
        dict(name="attend_306m", kind="attend", batch=8, q=512, k=512, heads=16, kv=4, d=64, causal=True, cache=False,
             train=True, docs=0),
        # the same heads over documents of uneven lengths packed without padding
        dict(name="attend_packed", kind="attend", batch=1, q=8191, k=8191, heads=16, kv=4, d=64, causal=True,
             cache=False, train=True, docs=23),
        # a long context with heads of 128
        dict(name="attend_long", kind="attend", batch=1, q=8192, k=8192, heads=16, kv=4, d=128, causal=True,
             cache=False, train=True, docs=0),
        # queries over another sequence (no causal mask), ragged lengths, a head size between the powers of two
        dict(name="attend_cross", kind="attend", batch=3, q=333, k=1021, heads=6, kv=2, d=96, causal=False,
             cache=False, train=True, docs=0),
        # rotary positions of a training step of the 306M model, q and k as parts of one projection
        dict(name="rotary_306m", kind="rotary", batch=8, tokens=512, heads=16, kv=4, d=64, rot=64, layout="half",
             scaling="none", far=0, type="bf16", train=True),
        # half of each head, interleaved, scaled to a context eight times the trained one
        dict(name="rotary_long", kind="rotary", batch=1, tokens=32767, heads=32, kv=8, d=128, rot=64,
             layout="interleaved", scaling="by_parts", far=1000000, type="bf16", train=True),
        # one token each of eight sequences
        dict(name="norm_token", kind="norm", rows=8, d=1024, residual=True, type="bf16", checkpoint="none", train=False),
        # a training step of the 306M model
        dict(name="norm_306m", kind="norm", rows=4096, d=1024, residual=True, type="bf16", checkpoint="none",
             train=True),
        # long, wide activations whose checkpoint is kept in 8 bits
        dict(name="norm_wide_int8", kind="norm", rows=16383, d=4096, residual=True, type="bf16", checkpoint="int8",
             train=True),
        # the 306M model's feed-forward of a ragged micro-batch
        dict(name="swiglu_509", kind="swiglu", rows=509, d=2816, type="bf16", fused=False, checkpoint="none",
             train=True),
        # wide activations, gate and up as halves of one projection, the checkpoint in 8 bits
        dict(name="swiglu_wide_int8", kind="swiglu", rows=16384, d=8192, type="bf16", fused=True, checkpoint="int8",
             train=True),
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi spread evenly over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "rotary", "norm", "swiglu"])
    if kind == "attend":
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        d = rng.choice([64, 64, 128, 128, 32, 80, 96])
        form = rng.choice(["token", "full", "full", "packed", "cross"])
        c = dict(kind=kind, batch=1, heads=heads, kv=kv, d=d, causal=True, cache=False, train=True, docs=0)
        if form == "token":
            c.update(batch=_log(rng, 1, 64), q=_log(rng, 1, 4), k=_log(rng, 4, 16000), cache=True, train=False)
        elif form == "packed":
            n = _log(rng, 100, 8191)
            c.update(q=n, k=n, docs=rng.randint(1, 10 ** 6))
        else:
            t = _log(rng, 16, 4096)
            c.update(batch=max(1, min(8, 4096 // t)), q=t, k=t)
            if form == "cross":
                c.update(k=_log(rng, 16, 4096), causal=rng.random() < 0.3)
        return c
    if kind == "rotary":
        d = rng.choice([64, 128, 80])
        return dict(kind=kind, batch=_log(rng, 1, 8), tokens=_log(rng, 1, 4095), heads=rng.choice([4, 12, 16, 32]),
                    kv=rng.choice([1, 2, 4]), d=d, rot=rng.choice([d, d, d // 2]),
                    layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "by_parts"]), far=rng.choice([0, 100000]),
                    type=rng.choice(["bf16", "bf16", "f32"]), train=rng.random() < 0.75)
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 16000), d=_log(rng, 64, 4096), residual=rng.random() < 0.7,
                    type=rng.choice(["bf16", "bf16", "f32"]), checkpoint=rng.choice(["none", "none", "int8"]),
                    train=rng.random() < 0.75)
    return dict(kind=kind, rows=_log(rng, 1, 8000), d=_log(rng, 64, 8192), type=rng.choice(["bf16", "bf16", "f32"]),
                fused=rng.random() < 0.5, checkpoint=rng.choice(["none", "int8"]), train=rng.random() < 0.75)


# ---- inputs --------------------------------------------------------------------------------

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rand(g, shape, spread=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device=DEV) * spread).to(dtype)


def _lengths(case):
    """Lengths of the documents packed into the case's rows, 16..2048 evenly over the logarithm."""
    rng, left, out = random.Random(case["docs"]), case["q"], []
    while left:
        out.append(min(left, _log(rng, 16, 2048)))
        left -= out[-1]
    return out


def _scaling(case):
    """Arguments of the scaled frequencies: a context eight times the trained one."""
    if case["scaling"] == "none":
        return {}
    return dict(scaling=case["scaling"], factor=8.0, **({"original_context": 4096} if case["scaling"] == "by_parts" else {}))


def _turns(case):
    """(turns per position of each rotated pair in 64 bits, amplitude)."""
    r, base, factor = case["rot"], 10000.0, 8.0
    if case["scaling"] == "ntk":
        base *= factor ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / (2 * math.pi)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "by_parts":
        keep = ((4096 * f - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 62))
    return globals()["_prepare_" + case["kind"]](case, g)


def _prepare_attend(case, g):
    B, Tq, Tk, H, KV, D = (case[n] for n in ("batch", "q", "k", "heads", "kv", "d"))
    s = dict(case=case, sequences=None, documents=None)
    if case["cache"]:   # the cache's own layout: kv head by kv head, with room behind the cached rows
        room = -(-Tk // 16) * 16
        k, v = (_rand(g, (B, KV, room, D)).transpose(1, 2)[:, :Tk] for _ in range(2))
    else:
        k, v = (_rand(g, (B, Tk, KV, D)) for _ in range(2))
    q, do = _rand(g, (B, Tq, H, D), 1.5), _rand(g, (B, Tq, H, D), 0.1)
    if case["docs"]:
        lens = _lengths(case)
        q, k, v, do = (x[0] for x in (q, k, v, do))
        s["documents"] = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(lens, device=DEV))
        if own:   # which rows are whose: known to the data loader, used by every layer of a step
            from transformer_amd.attention import Sequences
            s["sequences"] = Sequences(lens, device=DEV)
    s.update(q=q, k=k, v=v, do=do)
    if case["train"]:
        for n in ("q", "k", "v"):
            s[n] = s[n].detach().requires_grad_()
    return s


def _prepare_rotary(case, g):
    B, T, H, KV, D = (case[n] for n in ("batch", "tokens", "heads", "kv", "d"))
    t = TYPES[case["type"]]
    qkv = _rand(g, (B, T, H + 2 * KV, D), 1.0, t)
    first = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device=DEV, dtype=torch.int32)
    turns, amplitude = _turns(case)
    s = dict(case=case, q=qkv[:, :, :H], k=qkv[:, :, H:H + KV], turns=turns.to(DEV), amplitude=amplitude,
             positions=first + torch.arange(T, device=DEV, dtype=torch.int32),
             dq=_rand(g, (B, T, H, D), 0.1, t), dk=_rand(g, (B, T, KV, D), 0.1, t))
    if own:   # computed once for a model
        from transformer_amd.rotary import rotary_frequencies
        s["frequencies"] = rotary_frequencies(case["rot"], device=DEV, **_scaling(case))
    if case["train"]:
        s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
    return s


def _prepare_norm(case, g):
    n, d, t = case["rows"], case["d"], TYPES[case["type"]]
    s = dict(case=case, x=_rand(g, (n, d), 0.5, t), scale=(1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(t),
             residual=_rand(g, (n, d), 2.0, t) if case["residual"] else None, dy=_rand(g, (n, d), 0.1, t),
             ds=_rand(g, (n, d), 0.1, t))
    if case["train"]:
        for k in ("x", "scale", "residual"):
            if s[k] is not None:
                s[k].requires_grad_()
    return s


def _prepare_swiglu(case, g):
    n, d, t = case["rows"], case["d"], TYPES[case["type"]]
    both = _rand(g, (n, 2 * d), 1.0, t)
    gate, up = (both[:, :d], both[:, d:]) if case["fused"] else (both[:, :d].contiguous(), both[:, d:].contiguous())
    s = dict(case=case, gate=gate, up=up, dy=_rand(g, (n, d), 0.1, t))
    if case["train"]:
        s["gate"], s["up"] = gate.detach().requires_grad_(), up.detach().requires_grad_()
    return s


# ---- one pass ------------------------------------------------------------------------------

def run(state):
    if own:
        return globals()["_own_" + state["case"]["kind"]](state, **state["case"])
    with torch.no_grad():
        return globals()["_plain_" + state["case"]["kind"]](state, **state["case"])


def _own_attend(s, causal, train, **_):
    from transformer_amd.attention import attention
    out = attention(s["q"], s["k"], s["v"], causal=causal, sequences=s["sequences"])
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])) if train else out


def _own_rotary(s, layout, train, **_):
    from transformer_amd.rotary import rotary
    q, k = rotary(s["q"], s["k"], s["frequencies"], s["positions"], layout=layout)
    if not train:
        return q, k
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))


def _own_norm(s, residual, checkpoint, train, **_):
    from transformer_amd.norm import rms_norm
    keep = None if checkpoint == "none" else checkpoint
    if not residual:
        y = rms_norm(s["x"], s["scale"], eps=EPS, checkpoint=keep)
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["scale"]), s["dy"])) if train else y
    y, r = rms_norm(s["x"], s["scale"], s["residual"], eps=EPS, checkpoint=keep)
    if not train:
        return y, r
    return (y.detach(), r.detach(), *torch.autograd.grad((y, r), (s["x"], s["residual"], s["scale"]), (s["dy"], s["ds"])))


def _own_swiglu(s, checkpoint, train, **_):
    from transformer_amd.swiglu import swiglu
    y = swiglu(s["gate"], s["up"], checkpoint=None if checkpoint == "none" else checkpoint)
    return (y.detach(), *torch.autograd.grad(y, (s["gate"], s["up"]), s["dy"])) if train else y


def _visible(s, Tq, Tk, causal):
    """Which keys a query sees: those up to its own position, counted from the sequences' ends, of its document."""
    see = torch.ones(Tq, Tk, dtype=torch.bool, device=DEV)
    if causal:
        see = torch.arange(Tk, device=DEV)[None] <= torch.arange(Tk - Tq, Tk, device=DEV)[:, None]
    if s["documents"] is not None:
        see = see & (s["documents"][:, None] == s["documents"][None])
    return see


def _plain_attend(s, q, k, heads, kv, d, causal, train, **_):
    Tq, Tk, g, bf = q, k, heads // kv, torch.bfloat16
    packed = s["documents"] is not None

    def rows(x, n):   # (B, T, n g, d) as (B, n, g T, d) in 32 bits
        x = (x[None] if packed else x).float()
        B, T, h, _ = x.shape
        return x.reshape(B, T, n, h // n, d).permute(0, 2, 3, 1, 4).reshape(B, n, -1, d)

    def back(x, T):
        B, n = x.shape[:2]
        x = x.reshape(B, n, -1, T, d).permute(0, 3, 1, 2, 4).reshape(B, T, -1, d).to(bf)
        return x[0] if packed else x

    Q, K, V = rows(s["q"], kv), rows(s["k"], kv), rows(s["v"], kv)
    hide = ~_visible(s, Tq, Tk, causal).repeat(g, 1)
    p = torch.matmul(Q, K.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(d)).masked_fill_(hide, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1, total))
    out = back(torch.matmul(p, V), Tq)
    if not train:
        return out
    DO = rows(s["do"], kv)
    dV = torch.matmul(p.transpose(-1, -2).contiguous(), DO)
    dp = torch.matmul(DO, V.transpose(-1, -2).contiguous())
    ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(1 / math.sqrt(d))
    dQ, dK = torch.matmul(ds, K), torch.matmul(ds.transpose(-1, -2).contiguous(), Q)
    return out, back(dQ, Tq), back(dK, Tk), back(dV, Tk)


def _rotate(x, c, s, layout, rot, dtype):
    """The first ``rot`` values of each head of x rotated by the angles with cosines c and sines s."""
    h = rot // 2
    a, b = (x[..., :h], x[..., h:rot]) if layout == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    pair = (a * c - b * s, a * s + b * c)
    turned = torch.cat(pair, -1) if layout == "half" else torch.stack(pair, -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1).to(dtype)


def _plain_rotary(s, layout, rot, type, train, **_):
    turns = s["positions"].double()[..., None, None] * s["turns"]
    angle = (turns - turns.floor()) * (2 * math.pi)
    c, sn = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()
    t = TYPES[type]
    out = [_rotate(s[n].float(), c, sn, layout, rot, t) for n in ("q", "k")]
    if train:
        out += [_rotate(s[n].float(), c, -sn, layout, rot, t) for n in ("dq", "dk")]
    return tuple(out)


def _int8(x):
    """What x stands for after a checkpoint in 8 bits: a 32-bit scale for each 128 values of a row, from the largest."""
    n, d = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -d % BLOCK)).reshape(n, -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    small = top < 2.0 ** -100
    q = torch.round(x * (127 / torch.where(small, 1, top)))
    return torch.where(small, 0, q * (top / 127)).reshape(n, -1)[:, :d]


def _plain_norm(s, d, residual, type, checkpoint, train, **_):
    t = TYPES[type]
    r = s["x"]
    if residual:
        r = (s["x"].float() + s["residual"].float()).to(t)
    x, scale = r.float(), s["scale"].float()
    inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xh = x * inv
    out = ((xh * scale).to(t), r) if residual else ((xh * scale).to(t),)
    if not train:
        return out if residual else out[0]
    if checkpoint == "int8":
        xh = _int8(xh)
    dy = s["dy"].float()
    dxh = dy * scale
    dx = inv * (dxh - xh * (dxh * xh).mean(-1, keepdim=True))
    dscale = (dy * xh).sum(0).to(t)
    if not residual:
        return (*out, dx.to(t), dscale)
    dx = (dx + s["ds"].float()).to(t)
    return (*out, dx, dx.clone(), dscale)


def _plain_swiglu(s, type, checkpoint, train, **_):
    t = TYPES[type]
    g, u = s["gate"].float(), s["up"].float()
    y = (g / (1 + torch.exp(-g)) * u).to(t)
    if not train:
        return y
    if checkpoint == "int8":
        g, u = _int8(g), _int8(u)
    dy, sig = s["dy"].float(), 1 / (1 + torch.exp(-g))
    return y, (dy * u * sig * (1 + g * (1 - sig))).to(t), (dy * g * sig).to(t)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "attend":
        lens = [(n, n) for n in _lengths(c)] if c["docs"] else [(c["q"], c["k"])] * c["batch"]
        pairs = 0
        for q, k in lens:   # rows that see j keys: j = k - q + i + 1 where that is positive
            first = max(0, q - k)
            pairs += sum(range(k - q + 1 + first, k + 1)) if c["causal"] else q * k
        q, k = c["batch"] * c["q"] * c["heads"], c["batch"] * c["k"] * c["kv"]
        if c["train"]:   # q, k, v, dout read; out, dq, dk, dv written
            return dict(bytes=2 * c["d"] * (4 * q + 4 * k), flops=14 * c["d"] * c["heads"] * pairs)
        return dict(bytes=2 * c["d"] * (2 * q + 2 * k), flops=4 * c["d"] * c["heads"] * pairs)
    size = 4 if c["type"] == "f32" else 2
    if c["kind"] == "rotary":
        n = c["batch"] * c["tokens"] * (c["heads"] + c["kv"]) * c["d"]
        return dict(bytes=size * n * 2 * (2 if c["train"] else 1) + 4 * c["batch"] * c["tokens"],
                    flops=3 * n * (2 if c["train"] else 1))
    n = c["rows"] * c["d"]
    if c["kind"] == "norm":
        moved = (4 if c["residual"] else 2) + ((4 if c["residual"] else 2) if c["train"] else 0)
        moved -= 1 if c["train"] and c["residual"] else 0   # x and the residual have one gradient
        return dict(bytes=size * (n * moved + c["d"] * (2 if c["train"] else 1)), flops=n * (15 if c["train"] else 5))
    return dict(bytes=size * n * (6 if c["train"] else 3), flops=n * (25 if c["train"] else 8))


# ---- the definitions in 64 bits ------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return globals()["_exact_" + case["kind"]](s, **case)


def _exact_attend(s, batch, q, k, heads, kv, d, causal, train, docs, **_):
    Q, K, V, DO = (s[n].detach() if docs else s[n].detach().flatten(0, 1) for n in ("q", "k", "v", "do"))
    out, dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=DEV) for x in (Q, Q, K, V))
    lens = [(n, n) for n in _lengths(s["case"])] if docs else [(q, k)] * batch
    q0 = k0 = 0
    for nq, nk in lens:
        i, j = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        last = torch.arange(nq, device=DEV)[:, None] + (nk - nq)
        hidden = (torch.arange(nk, device=DEV)[None] > last) if causal else None
        for h in range(heads):
            a = h // (heads // kv)
            qh, kh, vh = Q[i, h].double(), K[j, a].double(), V[j, a].double()
            e = qh @ kh.T / math.sqrt(d)
            if hidden is not None:
                e = e.masked_fill(hidden, float("-inf"))
            p = torch.nan_to_num(torch.softmax(e, -1), nan=0.0)   # a row that sees nothing
            o = p @ vh
            out[i, h] = o
            if not train:
                continue
            do = DO[i, h].double()
            dv[j, a] += p.T @ do
            de = p * (do @ vh.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(d)
            dq[i, h] = de @ kh
            dk[j, a] += de.T @ qh
    def shaped(x, T):
        return x if docs else x.unflatten(0, (batch, T))
    return (shaped(out, q), shaped(dq, q), shaped(dk, k), shaped(dv, k)) if train else shaped(out, q)


def _exact_rotary(s, layout, rot, train, **_):
    angle = 2 * math.pi * torch.frac(s["positions"].double().unsqueeze(-1) * s["turns"]).unsqueeze(-2)

    def turn(x, way):
        z = x.detach().double()
        y = z.clone()
        first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        w = torch.complex(z[..., first], z[..., second]) * torch.polar(torch.full_like(angle, s["amplitude"]), way * angle)
        y[..., first], y[..., second] = w.real, w.imag
        return y

    out = (turn(s["q"], 1), turn(s["k"], 1))
    return out + (turn(s["dq"], -1), turn(s["dk"], -1)) if train else out


def _exact_int8(x):
    """The checkpoint's values: the scale and the quotient are 32-bit by its definition, the rest is not."""
    out = torch.empty_like(x)
    for j in range(0, x.shape[1], BLOCK):
        b = x[:, j:j + BLOCK].float()
        top = b.abs().amax(1, keepdim=True)
        q = (b * (127 / top)).round().double() * (top / 127).double()
        out[:, j:j + BLOCK] = torch.where(top < 2.0 ** -100, 0, q)
    return out


def _exact_norm(s, residual, type, checkpoint, train, **_):
    x, w, dy = s["x"].detach().double(), s["scale"].detach().double(), s["dy"].double()
    if residual:
        x = (x + s["residual"].detach().double()).to(TYPES[type]).double()   # the sum is kept in its type
    ms = (x * x).sum(1, keepdim=True) / x.shape[1] + EPS
    z = x / ms.sqrt()
    out = (z * w, x) if residual else (z * w,)
    if not train:
        return out if residual else out[0]
    if checkpoint == "int8":
        z = _exact_int8(z)
    t = dy * w
    dx = (t - z * ((t * z).sum(1, keepdim=True) / x.shape[1])) / ms.sqrt()
    dw = (dy * z).sum(0)
    if not residual:
        return (*out, dx, dw)
    return (*out, dx + s["ds"].double(), dx + s["ds"].double(), dw)


def _exact_swiglu(s, checkpoint, train, **_):
    g, u, dy = s["gate"].detach().double(), s["up"].detach().double(), s["dy"].double()
    y = g * torch.sigmoid(g) * u
    if not train:
        return y
    if checkpoint == "int8":
        g, u = _exact_int8(g), _exact_int8(u)
    sig = torch.sigmoid(g)
    return y, dy * u * (sig + g * sig * (1 - sig)), dy * g * sig
