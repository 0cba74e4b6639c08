"""The batched operators of ane_amd beyond one kind of model, as timed cases.

``run`` is one pass through an operator: in plain torch where ``own`` is
false, through the framework's entry points where it is true.  ``listed``
names the cases, ``draw`` gives more of the same ranges, ``work`` says what a
pass cannot do without, and ``exact`` restates each operator in 64 bits.

Kinds and what they stand for:

linear   a batch's activations through an int8 weight matrix: each token
         quantized with a scale of its own (after an RMSNorm, where the layer
         has one there), the product in 8-bit integers, then the scales of
         token and output channel, a bias, a residual.
rotate   new tokens of packed sequences: RMSNorm of each q and k head, the
         position rotation (adjacent pairs or halves, whole heads or part of
         them, frequencies scaled for long contexts), k and v stored in the
         sequences' pages.
attend   attention of packed new tokens over the paged cache where the model
         is not plainly causal: scores capped by a tanh, a bias that grows
         with the distance, a window, documents, a prefix seen from both
         sides; one new token a sequence is the decode step.

The cache: fp16 keys and values in pages [layers][pages][kv heads][page size]
[head dim], one row of page numbers a sequence, a length a sequence.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's q, k and v products behind the attention norm: the latency a chat user sees
        {"name": "linear_one", "kind": "linear", "type": "f32", "out": "f32", "tokens": 1, "n": 6144, "k": 4096, "norm": True,
         "bias": False, "residual": False},
        # the next token of a serving batch through the down projection, added to the residual stream
        {"name": "linear_batch", "kind": "linear", "type": "f32", "out": "f32", "tokens": 32, "n": 4096, "k": 14336,
         "norm": False, "bias": False, "residual": True},
        # prompts through gate and up: the largest product of a layer
        {"name": "linear_prompt", "kind": "linear", "type": "f16", "out": "f16", "tokens": 4096, "n": 28672, "k": 4096,
         "norm": True, "bias": False, "residual": False},
        # sizes that fill no tile, a bias
        {"name": "linear_ragged", "kind": "linear", "type": "f32", "out": "f16", "tokens": 301, "n": 2003, "k": 1777,
         "norm": False, "bias": True, "residual": False},
        # the next token of every sequence of a batch, heads normalised, halves rotated
        {"name": "rotate_batch", "kind": "rotate", "type": "f32", "q_out": "f32", "seqs": 64, "new": 1, "cached": 3000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "norm": True, "half": True, "rot": 128, "stretch": 1.0, "mix": 1},
        # the prompts of a batch, queries handed on in 16 bits
        {"name": "rotate_prompt", "kind": "rotate", "type": "f32", "q_out": "f16", "seqs": 6, "new": 2400, "cached": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "norm": True, "half": True, "rot": 128, "stretch": 1.0, "mix": 2},
        # half of each head rotated, at far positions of a context stretched eightfold
        {"name": "rotate_far", "kind": "rotate", "type": "f16", "q_out": "f16", "seqs": 5, "new": 777, "cached": 60000,
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 48, "norm": False, "half": False, "rot": 32, "stretch": 8.0, "mix": 3},
        # one long document through a layer with a window and capped scores
        {"name": "attend_window", "kind": "attend", "type": "f16", "seqs": 1, "new": 8192, "cached": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "cap": 50.0, "slopes": False, "window": 1024, "docs": 0, "prefix": 0, "mix": 0},
        # prompts of different lengths, scores lowered with the distance
        {"name": "attend_distance", "kind": "attend", "type": "f32", "seqs": 9, "new": 1023, "cached": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "cap": 0.0, "slopes": True, "window": 0, "docs": 0, "prefix": 0, "mix": 4},
        # a smaller model: documents packed into sequences, the first part of each sequence seen from both sides
        {"name": "attend_documents", "kind": "attend", "type": "f16", "seqs": 5, "new": 777, "cached": 0, "heads": 12,
         "kv_heads": 4, "dim": 64, "page": 48, "cap": 0.0, "slopes": False, "window": 0, "docs": 3, "prefix": 200, "mix": 5},
        # the next chunk of two long prompts, scores capped and nothing masked but the future
        {"name": "attend_chunk", "kind": "attend", "type": "f32", "seqs": 2, "new": 96, "cached": 8000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "cap": 30.0, "slopes": False, "window": 0, "docs": 0, "prefix": 0, "mix": 6},
        # the next token of a batch of unrelated sequences, in a layer with a window
        {"name": "attend_tokens", "kind": "attend", "type": "f32", "seqs": 32, "new": 1, "cached": 4095, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "cap": 50.0, "slopes": False, "window": 1024, "docs": 0, "prefix": 0, "mix": 7},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["linear", "linear", "rotate", "attend", "attend"])
    c = {"kind": kind, "type": rng.choice(["f32", "f16"])}
    if kind == "linear":
        while True:
            c.update(tokens=1 if rng.random() < 0.15 else size(1, 8192), n=size(16, 28672), k=size(32, 14336))
            if c["tokens"] * c["n"] * c["k"] <= 4096 * 28672 * 4096:
                break
        if rng.random() < 0.6:  # whole groups of 64, as most models have
            c.update(n=-(-c["n"] // 64) * 64, k=-(-c["k"] // 64) * 64)
            c["tokens"] = max(1, min(c["tokens"], 4096 * 28672 * 4096 // (c["n"] * c["k"])))
        c.update(out=rng.choice(["f32", "f16"]), norm=rng.random() < 0.5, bias=rng.random() < 0.3, residual=rng.random() < 0.4)
        return c
    kv = rng.choice([1, 2, 3, 4, 8])
    c.update(kv_heads=kv, heads=kv * rng.choice([1, 2, 3, 4, 4, 5, 8]), dim=rng.choice([64, 128]), page=16 * size(1, 16),
             seqs=size(1, 64), mix=rng.randint(10, 10**6))
    if kind == "rotate":
        c.update(q_out=rng.choice(["f32", "f16"]), new=1 if rng.random() < 0.3 else size(1, 9000 // c["seqs"]),
                 cached=0 if rng.random() < 0.4 else size(1, min(60000, 300000 // c["seqs"])), norm=rng.random() < 0.6, half=rng.random() < 0.6,
                 rot=rng.choice([c["dim"], c["dim"], c["dim"] // 2, c["dim"] // 4]), stretch=rng.choice([1.0, 1.0, 4.0, 8.0]))
        return c
    while True:  # at most half the score plane of the longest listed prompt
        c.update(seqs=size(1, 32), new=1 if rng.random() < 0.3 else size(1, 6000),
                 cached=0 if rng.random() < 0.5 else size(1, 9000))
        if c["seqs"] * c["new"] * (c["new"] + c["cached"]) * c["heads"] <= 1 << 30:
            break
    c.update(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, window=0 if rng.random() < 0.5 else size(16, 4096),
             docs=0, prefix=0)
    if rng.random() < 0.4:
        c.update(docs=rng.randint(2, 6) if c["new"] > 8 else 0, prefix=size(1, c["new"] + c["cached"]) if rng.random() < 0.5 else 0)
    return c


def _lengths(c):
    """New and cached positions of each sequence (packed prompts differ in length; the first has the longest)."""
    r = random.Random(c["mix"])
    n = c["seqs"]
    new = [c["new"] if i == 0 or c["new"] == 1 else r.randint(max(1, c["new"] // 4), c["new"]) for i in range(n)]
    old = [c["cached"] if i == 0 or not c["cached"] else r.randint(c["cached"] // 4, c["cached"]) for i in range(n)]
    return new, old


def _masks(c):
    """First position of each new token's document, prefix length of each sequence (None: there are none)."""
    r = random.Random(c["mix"] + 1)
    new, old = _lengths(c)
    first = prefix = None
    if c["docs"]:
        first = []
        for n, m in zip(new, old):  # the first document holds the cached positions
            cuts = sorted({m + r.randrange(n) for _ in range(c["docs"] - 1)} - {0})
            at = 0
            for p in range(m, m + n):
                if p in cuts:
                    at = p
                first.append(at)
    if c["prefix"]:
        prefix = [c["prefix"] if i == 0 else r.randint(0, c["prefix"]) for i in range(c["seqs"])]
    return first, prefix


# ------------------------------------------------------------------ the inputs
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _randn(gen, shape, dtype, std):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    return x.normal_(0.0, std, generator=gen)


def _freqs(c):
    """Radians a position of each rotated pair: base 500000; stretched for a longer context, the slow ones divided by
    the stretch, the fast ones left as they are, in between by how often each turns within 8192 positions."""
    i = torch.arange(c["rot"] // 2, dtype=torch.float64)
    f = torch.pow(torch.tensor(500000.0, dtype=torch.float64), -2.0 * i / c["rot"])
    keep = ((8192 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
    return f * keep + f / c["stretch"] * (1.0 - keep)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "linear":
        t, n, k = c["tokens"], c["n"], c["k"]
        x = _randn(gen, (t, k), TYPES[c["type"]], 1.0)
        x *= torch.rand((t, 1), device=DEV, generator=gen).mul_(3).exp_().to(x.dtype)  # tokens of different size
        wide = -(-k // 16) * 16  # rows of the weights start on 16 bytes
        w = torch.zeros((n, wide), dtype=torch.int8, device=DEV)
        w[:, :k] = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=DEV, generator=gen)
        s.update(x=x, w=w[:, :k], w_scales=torch.rand(n, device=DEV, generator=gen).add_(0.1).mul_(1e-3),
                 norm=_randn(gen, (k,), torch.float32, 0.1).add_(1.0) if c["norm"] else None,
                 bias=_randn(gen, (n,), torch.float32, 1.0) if c["bias"] else None,
                 residual=_randn(gen, (t, n), TYPES[c["out"]], 1.0) if c["residual"] else None,
                 out=torch.empty((t, n), dtype=TYPES[c["out"]], device=DEV))
        return s
    r = random.Random(seed * 7919 + c["mix"])
    ps = c["page"]
    new, old = _lengths(c)
    lens = [a + b for a, b in zip(new, old)]
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + 3
    ids = r.sample(range(pages), sum(need))  # pages in no order
    rows = [[ids.pop() for _ in range(n)] + [-1] * (max(need) - n) for n in need]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    shape = (1, pages, c["kv_heads"], ps, c["dim"])
    s["k"], s["v"] = _randn(gen, shape, torch.float16, 1.0), _randn(gen, shape, torch.float16, 0.5)
    t, hq, hk, d = start[-1], c["heads"], c["kv_heads"], c["dim"]
    s.update(table=_i32(rows), lens=_i32(lens), start=_i32(start), max_len=max(lens), max_new=max(new))
    if c["kind"] == "rotate":
        qkv = _randn(gen, (t, hq + 2 * hk, d), TYPES[c["type"]], 1.0)  # as the product writes it
        s.update(q=qkv[:, :hq], new_k=qkv[:, hq:hq + hk], new_v=qkv[:, hq + hk:], freqs=_freqs(c).to(DEV),
                 factor=1.0 + 0.1 * math.log(c["stretch"]),
                 q_norm=_randn(gen, (d,), torch.float32, 0.1).add_(1.0) if c["norm"] else None,
                 k_norm=_randn(gen, (d,), torch.float32, 0.1).add_(1.0) if c["norm"] else None,
                 out=torch.empty((t, hq, d), dtype=TYPES[c["q_out"]], device=DEV))
        return s
    first, prefix = _masks(c)
    s["q"] = _randn(gen, (t, hq, d), TYPES[c["type"]], 1.5)
    s.update(out=torch.empty_like(s["q"]), first=None if first is None else _i32(first),
             prefix=None if prefix is None else _i32(prefix),
             slopes=torch.exp2(-8.0 * torch.arange(1, hq + 1, device=DEV) / hq).float() if c["slopes"] else None)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    import ane_amd as ane

    c = s["case"]
    if c["kind"] == "linear":
        if "work" not in s:  # kept by a serving program
            s["work"] = ane.linear_i8_workspace(c["tokens"], c["n"], c["k"])
        ane.linear_i8(s["x"], s["w"], s["w_scales"], s["out"], norm_w=s["norm"], eps=1e-5, bias=s["bias"],
                      residual=s["residual"], workspace=s["work"])
        return s["out"]
    if "cache" not in s:  # the cache's handle and what goes with it, which a serving program makes once
        s["cache"] = cache = ane.PagedCache(c["heads"], s["k"], s["v"], s["table"], s["lens"])
        if c["kind"] == "rotate":
            s["rope"] = ane.Rope(s["freqs"], half=c["half"], factor=s["factor"])
        else:
            s["rule"] = ane.AttentionRule(softcap=c["cap"], slopes=s["slopes"], window=c["window"], first=s["first"],
                                          prefix=s["prefix"])
            s["work"] = ane.attention_prompt_workspace(cache, c["seqs"], s["q"].shape[0], s["max_len"], rule=s["rule"])
    single = c["new"] == 1  # one new token a sequence: no starts are needed
    if c["kind"] == "rotate":
        ane.paged_norm_rope_append(s["cache"], 0, None if single else s["start"], s["q"], s["new_k"], s["new_v"], s["rope"],
                                   s["out"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    ane.attention_prompt(s["cache"], 0, None if single else s["start"], s["q"], s["out"], max_len=s["max_len"],
                         workspace=s["work"], rule=s["rule"])
    return s["out"]


def _plain_linear(s):
    x = s["x"].float()
    if s["norm"] is not None:  # (the sum in 64 bits: a value next to the border of two integers goes by it)
        ms = x.double().square().mean(dim=1, keepdim=True).float()
        x = x * (1.0 / torch.sqrt(ms + 1e-5)) * s["norm"]
    top = x.abs().amax(dim=1, keepdim=True)
    scale = torch.where(top == 0, torch.ones_like(top), top / 127.0)
    q = torch.round(x * torch.where(top == 0, 127.0, 127.0 / top)).clamp(-127, 127)
    y = (q @ s["w"].float().t()) * scale * s["w_scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    s["out"].copy_(y)
    return s["out"]


def _places(s):
    """Sequence, place among its new tokens and position of every packed token."""
    start = s["start"].long()
    t = s["q"].shape[0]
    seq = torch.bucketize(torch.arange(t, device=DEV), start[1:], right=True)
    i = torch.arange(t, device=DEV) - start[seq]
    return seq, i, s["lens"].long()[seq] - (start[1:] - start[:-1])[seq] + i


def _plain_rotate(s):
    c, ps = s["case"], s["case"]["page"]
    seq, _, pos = _places(s)
    angle = pos.double()[:, None] * s["freqs"]  # far positions need 64 bits
    co, si = (angle.cos() * s["factor"]).float()[:, None], (angle.sin() * s["factor"]).float()[:, None]
    rot = c["rot"]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-6) * w
        y = x[..., :rot]
        a, b = (y[..., :rot // 2], y[..., rot // 2:]) if c["half"] else (y[..., 0::2], y[..., 1::2])
        u, v = a * co - b * si, a * si + b * co
        y = torch.cat([u, v], dim=-1) if c["half"] else torch.stack([u, v], dim=-1).flatten(-2)
        return torch.cat([y, x[..., rot:]], dim=-1)

    s["out"].copy_(turn(s["q"], s["q_norm"]))
    page = s["table"][seq, pos // ps].long()
    at = (page, torch.arange(c["kv_heads"], device=DEV)[:, None], pos % ps)
    s["k"][0].index_put_(at, turn(s["new_k"], s["k_norm"]).to(torch.float16).transpose(0, 1))
    s["v"][0].index_put_(at, s["new_v"].to(torch.float16).transpose(0, 1))
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _plain_attend(s):
    c, ps = s["case"], s["case"]["page"]
    n, hk, d, m = c["seqs"], c["kv_heads"], c["dim"], s["max_new"]
    g = c["heads"] // hk
    seq, i, pos = _places(s)

    def padded(x, fill):  # [sequences][new tokens] from packed tokens
        y = torch.full((n, m), fill, dtype=torch.long, device=DEV)
        y[seq, i] = x
        return y[:, None, None, :, None]

    q = torch.zeros((n, m, c["heads"], d), device=DEV)
    q[seq, i] = s["q"].float()
    q = q.view(n, m, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * m, d)
    j = torch.arange(s["max_len"], device=DEV)
    page = s["table"][:, j // ps].long().clamp(min=0)
    k, v = (s[x][0][page, :, (j % ps)[None, :]].float().transpose(1, 2).contiguous() for x in "kv")
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(d)).view(n, hk, g, m, -1)
    p = padded(pos, -1)
    if c["cap"]:
        sc = sc.div_(c["cap"]).tanh_().mul_(c["cap"])
    if s["slopes"] is not None:
        sc -= s["slopes"].view(1, hk, g, 1, 1) * (p - j).abs()
    end = p + 1 if s["prefix"] is None else torch.maximum(p + 1, s["prefix"].long()[:, None, None, None, None])
    end = torch.where(p < 0, 0, torch.minimum(end, s["lens"].long()[:, None, None, None, None]))
    hidden = j >= end
    if c["window"]:
        hidden |= j <= p - c["window"]
    if s["first"] is not None:
        hidden |= j < padded(s["first"].long(), 0)
    sc.masked_fill_(hidden, -math.inf)
    top = sc.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    w = sc.sub_(top).exp_()
    total = w.sum(dim=-1, keepdim=True)
    o = torch.matmul(w.view(n, hk, g * m, -1), v).view(n, hk, g, m, d) / total.masked_fill(total == 0, 1.0)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, m, c["heads"], d)[seq, i])
    return s["out"]


def _plain(s):
    return {"linear": _plain_linear, "rotate": _plain_rotate, "attend": _plain_attend}[s["case"]["kind"]](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    size = 4 if c["type"] == "f32" else 2
    if c["kind"] == "linear":
        t, n, k = c["tokens"], c["n"], c["k"]
        out = 4 if c["out"] == "f32" else 2
        return {"bytes": t * k * size + n * k + 4 * n * (2 if c["bias"] else 1) + t * n * out * (2 if c["residual"] else 1)
                + (4 * k if c["norm"] else 0), "flops": 2 * t * n * k}
    new, old = _lengths(c)
    t = sum(new)
    if c["kind"] == "rotate":
        out = 4 if c["q_out"] == "f32" else 2
        return {"bytes": t * c["dim"] * (c["heads"] * (size + out) + 2 * c["kv_heads"] * (size + 2)),
                "flops": t * (c["heads"] + c["kv_heads"]) * (3 * c["rot"] + (4 * c["dim"] if c["norm"] else 0))}
    first, prefix = _masks(c)
    pairs = seen = at = 0
    for i, (n, m) in enumerate(zip(new, old)):
        least = m + n
        for p in range(m, m + n):
            lo = max(0, p + 1 - c["window"] if c["window"] else 0, first[at] if first else 0)
            end = min(m + n, max(p + 1, prefix[i] if prefix else 0))
            pairs += max(0, end - lo)
            least = min(least, lo)
            at += 1
        seen += m + n - least
    return {"bytes": 2 * t * c["heads"] * c["dim"] * size + 4 * c["kv_heads"] * c["dim"] * seen,
            "flops": 4 * c["dim"] * c["heads"] * pairs}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "linear":
        # the integers are defined by 32-bit steps: each is computed in 64 bits and rounded
        x = s["x"].double()
        if c["norm"]:
            mean = ((x * x).sum(dim=1) / c["k"]).float().double()
            inv = (1.0 / (mean + torch.tensor(1e-5, dtype=torch.float32).double()).float().double().sqrt().float().double()).float().double()
            x = ((x * inv[:, None]).float().double() * s["norm"].double()).float().double()
        out = torch.empty((c["tokens"], c["n"]), dtype=torch.float64, device=DEV)
        w = s["w"].double().t().contiguous()
        for a in range(0, c["tokens"], 1024):
            y = x[a:a + 1024]
            top = y.abs().max(dim=1).values
            step = (top / 127.0).float().double().masked_fill_(top == 0, 1.0)
            per = (127.0 / top).float().double().masked_fill_(top == 0, 127.0)
            ints = (y * per[:, None]).float().double().round().clamp(-127.0, 127.0)
            out[a:a + 1024] = ints @ w * step[:, None] * s["w_scales"].double()
        if c["bias"]:
            out += s["bias"].double()
        if c["residual"]:
            out += s["residual"].double()
        return out
    new, old = _lengths(c)
    ps, g = c["page"], c["heads"] // c["kv_heads"]
    out, at = s["q"].double().clone(), 0
    if c["kind"] == "rotate":
        k, v = s["k"].double(), s["v"].double()
        for i, (n, m) in enumerate(zip(new, old)):
            p = torch.arange(m, m + n, device=DEV)
            z = torch.polar(torch.full((n, 1, c["rot"] // 2), s["factor"], dtype=torch.float64, device=DEV),
                            (p.double()[:, None] * s["freqs"])[:, None])

            def turn(x, w):
                x = x.double()
                if w is not None:
                    x = x / ((x * x).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * w.double()
                part, rest = x[..., :c["rot"]], x[..., c["rot"]:]
                if c["half"]:
                    y = torch.complex(*(h.contiguous() for h in part.chunk(2, dim=-1))) * z
                    return torch.cat([y.real, y.imag, rest], dim=-1)
                y = torch.view_as_complex(part.reshape(*part.shape[:-1], -1, 2).contiguous()) * z
                return torch.cat([torch.view_as_real(y).flatten(-2), rest], dim=-1)

            rows = slice(at, at + n)
            at += n
            page = s["table"][i, p // ps].long()
            out[rows] = turn(s["q"][rows], s["q_norm"])
            k[0, page, :, p % ps] = turn(s["new_k"][rows], s["k_norm"])
            v[0, page, :, p % ps] = s["new_v"][rows].double()
        return {"q": out, "k": k, "v": v}
    first, prefix = _masks(c)
    for i, (n, m) in enumerate(zip(new, old)):
        j = torch.arange(m + n, device=DEV)
        page = s["table"][i, j // ps].long()
        p = torch.arange(m, m + n, device=DEV)[:, None]
        sees = j[None, :] <= p
        if prefix:
            sees = sees | (j[None, :] < prefix[i])
        if c["window"]:
            sees = sees & (p - j[None, :] < c["window"])
        if first:
            sees = sees & (j[None, :] >= torch.tensor(first[at:at + n], device=DEV)[:, None])
        for h in range(c["heads"]):
            k, v = (s[x][0, page, h // g, j % ps].double() for x in "kv")
            w = s["q"][at:at + n, h].double() @ k.t().contiguous() / math.sqrt(c["dim"])
            if c["cap"]:
                w = torch.tanh(w / c["cap"]) * c["cap"]
            if c["slopes"]:
                w = w - float(s["slopes"][h]) * (p - j[None, :]).abs()
            e = torch.exp(w - w.masked_fill(~sees, -1e300).amax(dim=1, keepdim=True)).masked_fill(~sees, 0.0)
            out[at:at + n, h] = e @ v / e.sum(dim=1, keepdim=True).clamp(min=1e-300)
        at += n
    return out
