"""Performance cases of the paged cache's operators: writing a step's keys and values into pages, attention of each
sequence's newest tokens (one, or a chunk of a prompt) over its pages, with or without the sums of the attention weight that
each cached position has received, and the eviction that keeps the most attended and the newest positions.

``run`` computes a case in plain torch operations in 32 bits, or (``own``) through the framework's
operators; ``exact`` restates the definitions in 64 bits.
"""
import math
import random

import torch

own = False
DEV = "cuda"
PAGE = 16            # positions of a page


def listed():
    return [
        # a decode step of four sequences in the middle of their answers: latency
        dict(name="step_token", kind="attend", batch=4, new=1, mixed=False, longest=2000, heads=16, kv=4, d=64,
             weights=False),
        # a decode step of the 306M model, which counts what each position receives
        dict(name="step_306m_weights", kind="attend", batch=8, new=1, mixed=False, longest=512, heads=16, kv=4, d=64,
             weights=True),
        # a decode step of a full server: many sequences of uneven lengths, the cache's bytes
        dict(name="step_many", kind="attend", batch=64, new=1, mixed=False, longest=16000, heads=32, kv=8, d=128,
             weights=False),
        # the same, counting, with heads that share no keys
        dict(name="step_many_weights", kind="attend", batch=24, new=1, mixed=False, longest=8000, heads=16, kv=16, d=128,
             weights=True),
        # prompts of the 306M model in chunks
        dict(name="chunk_306m", kind="attend", batch=8, new=128, mixed=False, longest=512, heads=16, kv=4, d=64,
             weights=False),
        # a step that serves single tokens, drafts and chunks together, ragged, with a head size between the powers of two
        dict(name="chunk_mixed", kind="attend", batch=13, new=333, mixed=True, longest=2900, heads=6, kv=2, d=96,
             weights=False),
        # a chunk of a long prompt
        dict(name="chunk_long", kind="attend", batch=1, new=2048, mixed=False, longest=16384, heads=32, kv=8, d=128,
             weights=False),
        # a chunk behind a cache that is evicted afterwards
        dict(name="chunk_long_weights", kind="attend", batch=1, new=511, mixed=False, longest=8191, heads=16, kv=4, d=128,
             weights=True),
        # the keys and values of a decode step
        dict(name="append_token", kind="append", batch=8, new=1, mixed=False, longest=512, heads=16, kv=4, d=64),
        # those of a step that is full of prompts
        dict(name="append_chunk", kind="append", batch=7, new=4095, mixed=False, longest=6000, heads=32, kv=8, d=128),
        # the 306M model's cache, all layers, cut to half its context
        dict(name="evict_306m", kind="evict", batch=8, longest=512, layers=24, kv=4, d=64, keep=256, recent=64),
        # long caches cut to a quarter
        dict(name="evict_long", kind="evict", batch=2, longest=30000, layers=4, kv=8, d=128, keep=8000, recent=1000),
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi spread evenly over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["step", "step", "chunk", "chunk", "append", "evict"])
    kv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 128, 128, 32, 80, 96])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    if kind == "step":   # one token, or a few drafts
        longest = _log(rng, 8, 16000)
        return dict(kind="attend", batch=_log(rng, 1, max(1, min(64, 400000 // longest))), new=rng.choice([1, 1, 1, 4]), mixed=rng.random() < 0.2,
                    longest=longest, heads=heads, kv=kv, d=d, weights=rng.random() < 0.4)
    if kind == "chunk":
        longest = _log(rng, 64, 12000)
        new = _log(rng, 8, min(longest, 2048))
        most = max(1, min(16, 2 ** 28 // (heads * new * longest)))
        return dict(kind="attend", batch=rng.randint(1, most), new=new, mixed=rng.random() < 0.4, longest=longest, heads=heads,
                    kv=kv, d=d, weights=rng.random() < 0.4)
    if kind == "append":
        new = _log(rng, 1, 4095)
        return dict(kind="append", batch=_log(rng, 1, max(1, min(64, 30000 // new))), new=new, mixed=rng.random() < 0.4,
                    longest=new + _log(rng, 1, 4000), heads=heads, kv=kv, d=d)
    longest, layers = _log(rng, 32, 30000), _log(rng, 1, 24)
    keep = max(16, int(longest * rng.uniform(0.1, 0.9)))
    return dict(kind="evict", batch=_log(rng, 1, max(1, min(32, 240000 // (longest * layers)))), longest=longest, layers=layers,
                kv=kv, d=d, keep=keep, recent=int(keep * rng.uniform(0.0, 0.5)))


# ---- inputs --------------------------------------------------------------------------------

def _rand(g, shape, spread=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * spread).to(torch.bfloat16)


def _lengths(case):
    """(new tokens, cached positions with them) of each sequence: one as long as the case says, the others from a quarter of that
    on; in a mixed step some have one new token, some none."""
    new, longest = case.get("new", 0), case["longest"]
    rng = random.Random(case["batch"] * 1000003 + longest * 101 + new)
    lens = [longest] + [rng.randint(max(new, longest // 4, 1), longest) for _ in range(case["batch"] - 1)]
    news = [new] + [rng.choice([0, 1, 1, rng.randint(1, new)]) if case.get("mixed") else new for _ in lens[1:]]
    return news, lens


def _pages(n, free):
    """The numbers of the pages that n positions take, from the list of the free ones."""
    return [free.pop() for _ in range(-(-n // PAGE))]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 62))
    return globals()["_prepare_" + case["kind"]](case, g, random.Random(int(seed)))


def _pool(case, rng, more=0):
    """Page numbers of every sequence, in no order, `more` positions of others for each, and how many pages the pool has."""
    lens = _lengths(case)[1]
    n = sum(-(-x // PAGE) for x in lens) + case["batch"] * -(-more // PAGE) + 3
    free = list(range(n))
    rng.shuffle(free)
    return [_pages(x, free) for x in lens], [_pages(more, free) for _ in lens], n


def _table(rows):
    """The lists as one table on the GPU, filled up with a page that exists."""
    width = max(1, *(len(r) for r in rows))
    return torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int64).to(DEV)


def _sequences(case, tables):
    """The step's plan, made once for all layers."""
    from transformer_amd.paged_attention import PagedSequences
    return PagedSequences(*_lengths(case), tables, case.get("heads", case["kv"]), case["kv"], device=DEV)


def _prepare_step(case, g, rng):
    """A layer's pages and the step's projections, whose heads lie as q, k, v in one tensor."""
    B, H, KV, D = (case[n] for n in ("batch", "heads", "kv", "d"))
    news, lens = _lengths(case)
    tables, _, n = _pool(case, rng)
    pool, qkv = _rand(g, (2, KV, n * PAGE, D)), _rand(g, (sum(news), H + 2 * KV, D), 1.5)
    first = [sum(news[:b]) for b in range(B)]
    s = dict(case=case, k_pages=pool[0], v_pages=pool[1], q=qkv[:, :H], k=qkv[:, H:H + KV], v=qkv[:, H + KV:])
    s.update(table=_table(tables), lens=torch.tensor(lens).to(DEV), news=torch.tensor(news).to(DEV), first=torch.tensor(first).to(DEV),
             sequence=torch.tensor([b for b in range(B) for _ in range(news[b])]).to(DEV))
    if own:
        s["sequences"] = _sequences(case, tables)
    return s


_prepare_append = _prepare_step


def _prepare_attend(case, g, rng):
    s = _prepare_step(case, g, rng)
    s["weights"] = None
    if case["weights"]:   # what earlier steps have left
        s["weights"] = torch.rand((case["batch"], case["kv"], case["longest"]), generator=g, device=DEV) * 3
    return s


def _prepare_evict(case, g, rng):
    Ly, B, KV, D = (case[n] for n in ("layers", "batch", "kv", "d"))
    tables, to, n = _pool(case, rng, case["keep"])
    k, v = _rand(g, (Ly, KV, n * PAGE, D)), _rand(g, (Ly, KV, n * PAGE, D))
    # few positions receive most of it; some have received the same, some nothing
    w = torch.exp(2 * torch.randn((Ly, B, KV, case["longest"]), generator=g, device=DEV) - 2)
    s = dict(case=case, k_pages=k, v_pages=v, weights=torch.round(w * 1024) / 1024, table=_table(tables), to=_table(to),
             lens=torch.tensor(_lengths(case)[1]).to(DEV))
    if own:
        from transformer_amd.paged_attention import PagedEviction
        s["eviction"] = PagedEviction(_sequences(case, tables), case["keep"], case["recent"], to)
    return s


# ---- one pass ------------------------------------------------------------------------------

def run(state):
    if own:
        return globals()["_own_" + state["case"]["kind"]](state)
    with torch.no_grad():
        return globals()["_plain_" + state["case"]["kind"]](state, **state["case"])


def _own_attend(s):
    from transformer_amd.paged_attention import paged_attention
    return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["sequences"], weights=s["weights"])


def _own_append(s):
    from transformer_amd.paged_attention import paged_append
    paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["sequences"])
    return s["k_pages"], s["v_pages"]


def _own_evict(s):
    from transformer_amd.paged_attention import paged_evict
    weights, kept = paged_evict(s["k_pages"], s["v_pages"], s["weights"], s["eviction"])
    return s["k_pages"], s["v_pages"], weights, kept


def _plain_attend(s, batch, longest, heads, kv, d, **_):
    B, L, g, top_new = batch, longest, heads // kv, s["case"]["new"]
    i, j = torch.arange(top_new, device=DEV), torch.arange(L, device=DEV)
    there = i < s["news"][:, None]
    rows = torch.where(there, s["first"][:, None] + i, 0)
    Q = s["q"][rows].float().reshape(B, top_new, kv, g, d).permute(0, 2, 3, 1, 4).reshape(B, kv, g * top_new, d)
    cells = s["table"][:, j // PAGE] * PAGE + j % PAGE
    K, V = (s[n][:, cells].transpose(0, 1).float() for n in ("k_pages", "v_pages"))
    see = j <= (s["lens"] - s["news"])[:, None, None] + i[:, None]   # (the newest token sees all)
    see = (see & there[..., None]).repeat(1, g, 1)[:, None]
    p = torch.matmul(Q, K.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(d)).masked_fill_(~see, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1, total))
    out = torch.matmul(p, V.contiguous()).reshape(B, kv, g, top_new, d).permute(0, 3, 1, 2, 4).reshape(B, top_new, heads, d)
    news_at = torch.arange(len(s["sequence"]), device=DEV) - s["first"][s["sequence"]]
    out = out[s["sequence"], news_at].to(torch.bfloat16)
    if s["weights"] is None:
        return out
    before = j < (s["lens"] - s["news"])[:, None, None]
    return out, torch.where(before, s["weights"], 0) + p.sum(-2)


def _plain_append(s, **_):
    at = torch.arange(len(s["sequence"]), device=DEV) - s["first"][s["sequence"]]
    at = at + (s["lens"] - s["news"])[s["sequence"]]
    cells = s["table"][s["sequence"], at // PAGE] * PAGE + at % PAGE
    s["k_pages"][:, cells] = s["k"].transpose(0, 1)
    s["v_pages"][:, cells] = s["v"].transpose(0, 1)
    return s["k_pages"], s["v_pages"]


def _plain_evict(s, batch, longest, layers, kv, keep, recent, **_):
    j, n = torch.arange(longest, device=DEV), torch.arange(keep, device=DEV)
    lens = s["lens"][:, None, None]
    w = torch.where(j >= lens - recent, math.inf, s["weights"])
    w = torch.where(j >= lens, -1.0, w)   # (no weight is negative)
    first = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :keep]
    first = torch.nn.functional.pad(first, (0, keep - first.shape[-1]))
    there = (n < lens).expand(first.shape)
    kept = torch.sort(torch.where(there, first, longest), dim=-1)[0]
    kept = torch.where(there, kept, 0)
    b = torch.arange(batch, device=DEV)[:, None, None]
    layer, head = torch.arange(layers, device=DEV)[:, None, None, None], torch.arange(kv, device=DEV)[:, None]
    source = s["table"][b, kept // PAGE] * PAGE + kept % PAGE
    cells = (s["to"][:, n // PAGE] * PAGE + n % PAGE)[:, None].expand(source.shape)
    for x in (s["k_pages"], s["v_pages"]):
        x[layer, head, cells] = torch.where(there[..., None], x[layer, head, source], x[layer, head, cells])
    weights = torch.where(there, torch.gather(s["weights"], -1, kept), 0)
    return s["k_pages"], s["v_pages"], weights, torch.where(there, kept, -1).to(torch.int32)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    news, lens = _lengths(case)
    if case["kind"] == "append":   # keys and values read, written
        return dict(bytes=sum(news) * case["kv"] * case["d"] * 8, flops=0)
    if case["kind"] == "evict":   # the kept rows read, written; the weights read; the kept ones and their places written
        held = sum(min(n, case["keep"]) for n in lens)
        heads = case["layers"] * case["kv"]
        return dict(bytes=heads * (held * (case["d"] * 8 + 8) + 4 * sum(lens)), flops=0)
    # queries read, outputs written, every cached key and value read once; weights read, written
    served = sum(n for n, q in zip(lens, news) if q)
    pairs = sum(q * (n - q) + q * (q + 1) // 2 for q, n in zip(news, lens))
    size = 4 * case["d"] * (sum(news) * case["heads"] + served * case["kv"])
    flops = 4 * case["d"] * case["heads"] * pairs
    if case["weights"]:
        size += 4 * case["kv"] * (2 * sum(lens) - sum(news))
        flops += case["heads"] * pairs
    return dict(bytes=size, flops=flops)


# ---- the definitions in 64 bits ------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    tables, lens = s["table"].tolist(), s["lens"].tolist()

    def held(x, b, count):   # a sequence's rows, page after page
        return torch.cat([x[..., PAGE * t:PAGE * t + PAGE, :] for t in tables[b][:-(-count // PAGE)]], -2)[..., :count, :]

    if case["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        sums = torch.zeros((case["batch"], case["kv"], case["longest"]), dtype=torch.float64, device=DEV)
        at, share = 0, case["heads"] // case["kv"]
        for b, (new, n) in enumerate(zip(s["news"].tolist(), lens)):
            if case["weights"]:
                sums[b, :, :n - new] = s["weights"][b, :, :n - new]
            if not new:
                continue
            keys, values = held(s["k_pages"], b, n).double(), held(s["v_pages"], b, n).double()
            hidden = torch.ones(new, n, dtype=torch.bool, device=DEV).triu(n - new + 1)
            for h in range(case["heads"]):
                e = (s["q"][at:at + new, h].double() @ keys[h // share].T.contiguous()) / case["d"] ** 0.5
                p = torch.softmax(e.masked_fill(hidden, float("-inf")), -1)
                out[at:at + new, h] = p @ values[h // share]
                sums[b, h // share, :n] += p.sum(0)
            at += new
        return (out, sums) if case["weights"] else out
    k, v = s["k_pages"].double(), s["v_pages"].double()
    if case["kind"] == "append":
        at = 0
        for b, (new, n) in enumerate(zip(s["news"].tolist(), lens)):
            cells = torch.tensor([PAGE * tables[b][x // PAGE] + x % PAGE for x in range(n - new, n)], dtype=torch.int64, device=DEV)
            for x, rows in ((k, s["k"]), (v, s["v"])):
                x[:, cells] = rows[at:at + new].transpose(0, 1).double()
            at += new
        return k, v
    weights = torch.zeros((case["layers"], case["batch"], case["kv"], case["keep"]), dtype=torch.float64)
    kept, w, to = torch.full(weights.shape, -1, dtype=torch.int32), s["weights"].cpu(), s["to"].tolist()
    for b, n in enumerate(lens):
        old = n - min(case["recent"], n)
        heavy = max(0, min(n, case["keep"]) - (n - old))
        cells = torch.tensor([PAGE * to[b][x // PAGE] + x % PAGE for x in range(min(n, case["keep"]))], dtype=torch.int64, device=DEV)
        for layer in range(case["layers"]):
            rows_k, rows_v = held(s["k_pages"][layer], b, n), held(s["v_pages"][layer], b, n)
            for h in range(case["kv"]):
                x = w[layer, b, h, :old].tolist()
                order = sorted(range(old), key=lambda i: -x[i])   # (in order of position where they are alike)
                chosen = torch.tensor(sorted(order[:heavy]) + list(range(old, n)), dtype=torch.int64)
                kept[layer, b, h, :len(chosen)] = chosen.to(torch.int32)
                weights[layer, b, h, :len(chosen)] = w[layer, b, h][chosen].double()
                k[layer, h][cells] = rows_k[h][chosen.to(DEV)].double()
                v[layer, h][cells] = rows_v[h][chosen.to(DEV)].double()
    return k, v, weights.to(DEV), kept.to(DEV)
