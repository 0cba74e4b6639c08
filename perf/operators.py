"""The batched and paged attention operators of ane_amd, as timed cases.

``run`` is one pass through an operator: in plain torch where ``own`` is
false, through the framework's entry points where it is true.  ``listed``
names the cases, ``draw`` gives more of the same ranges, ``work`` says what a
pass cannot do without, and ``exact`` restates each operator in 64 bits.

The cache all of them work on: fp16 keys and values in pages
[layers][pages][kv heads][page size][head dim], one row of page numbers a
sequence, a length a sequence, a reference count a page.

Kinds and what they stand for:

append   new tokens of packed sequences: RoPE of q and k, k and v stored in
         the sequences' pages (a decode batch: one token each; a prompt:
         many).
prompt   causal attention of packed prompts with grouped heads; a sequence
         may have positions cached before its new tokens.
shared   one new token of each sequence of a batch, the sequences of a group
         sharing the pages of a long prefix; without groups, plain batched
         decode.
fork     the samples of the last step are freed and new ones forked from
         their prompts (each sample shares the prompt's whole pages and gets
         its own copy of the last, part-filled one).
compact  the live pages of a fragmented pool moved to its front.
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
        # the next token of every sequence of a serving batch, appended
        {"name": "append_batch", "kind": "append", "type": "f32", "q_out": "f32", "seqs": 64, "new": 1, "cached": 3000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "mix": 1},
        # the prompts of a batch, appended; queries handed on in 16 bits
        {"name": "append_prompt", "kind": "append", "type": "f32", "q_out": "f16", "seqs": 6, "new": 2400, "cached": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "mix": 2},
        # a chat turn: one short prompt, the latency before its first token
        {"name": "prompt_chat", "kind": "prompt", "type": "f32", "seqs": 1, "new": 128, "cached": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "mix": 0},
        # prompts of different lengths packed together, activations as the products give them
        {"name": "prompt_packed", "kind": "prompt", "type": "f32", "seqs": 9, "new": 1023, "cached": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "mix": 3},
        # one long document
        {"name": "prompt_long", "kind": "prompt", "type": "f16", "seqs": 1, "new": 8192, "cached": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "mix": 0},
        # the next chunk of two long prompts: few rows, many cached positions
        {"name": "prompt_chunk", "kind": "prompt", "type": "f32", "seqs": 2, "new": 96, "cached": 8000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "mix": 4},
        # a smaller model: 64-wide heads in groups of three, odd lengths
        {"name": "prompt_groups3", "kind": "prompt", "type": "f16", "seqs": 5, "new": 777, "cached": 333, "heads": 12,
         "kv_heads": 4, "dim": 64, "page": 48, "mix": 5},
        # one sequence, one token: the latency a chat user sees
        {"name": "decode_one", "kind": "shared", "type": "f32", "seqs": 1, "groups": 0, "prefix": 0, "own": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "mix": 0},
        # a serving batch of unrelated sequences of different lengths
        {"name": "decode_batch", "kind": "shared", "type": "f32", "seqs": 32, "groups": 0, "prefix": 0, "own": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "mix": 6},
        # many users behind one long system prompt
        {"name": "shared_system", "kind": "shared", "type": "f32", "seqs": 64, "groups": 1, "prefix": 8192, "own": 300,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "mix": 7},
        # eight samples drawn from each of eight prompts
        {"name": "fork_samples", "kind": "fork", "layers": 32, "prompts": 8, "samples": 7, "length": 330, "kv_heads": 8,
         "dim": 128, "page": 16, "mix": 8},
        # a pool half of whose pages were freed in no order
        {"name": "compact_half", "kind": "compact", "layers": 16, "pages": 512, "live": 0.5, "kv_heads": 8, "dim": 128,
         "page": 16, "mix": 9},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["append", "prompt", "prompt", "shared", "shared", "fork", "compact"])
    kv = rng.choice([1, 2, 3, 4, 8])
    c = {"kind": kind, "kv_heads": kv, "dim": rng.choice([64, 128]), "page": 16 * size(1, 16), "mix": rng.randint(10, 10**6)}
    if kind in ("append", "prompt", "shared"):
        c.update(heads=kv * rng.choice([1, 2, 3, 4, 4, 5, 8]), type=rng.choice(["f32", "f16"]), seqs=size(1, 64))
    if kind == "append":
        c.update(q_out=rng.choice(["f32", "f16"]), new=1 if rng.random() < 0.3 else size(1, 9000 // c["seqs"]),
                 cached=0 if rng.random() < 0.4 else size(1, 4000))
    elif kind == "prompt":
        while True:  # at most the score plane of the longest listed prompt
            c.update(seqs=size(1, 32), new=size(1, 6000), cached=0 if rng.random() < 0.5 else size(1, 9000))
            if c["seqs"] * c["new"] * (c["new"] + c["cached"]) * c["heads"] <= 1 << 30:
                break
    elif kind == "shared":
        groups = rng.choice([0, 0, 1, 1, rng.randint(1, 4)])
        while True:
            c.update(groups=min(groups, c["seqs"]), prefix=size(16, 8192) if groups else 0, own=size(1, 4096))
            if c["seqs"] * (c["prefix"] + c["own"]) * kv <= 64 * 8492 * 8:
                break
    elif kind == "fork":
        c.update(layers=size(1, 32), prompts=size(1, 16), samples=size(1, 16), length=size(1, 2000))
        per = -(-c["length"] // c["page"]) + c["samples"]
        while c["layers"] * c["prompts"] * per * kv * c["page"] * c["dim"] > 1 << 27:
            c["layers"] = max(1, c["layers"] // 2)
            c["prompts"] = max(1, c["prompts"] // 2)
    else:
        c.update(layers=size(1, 16), pages=size(16, 2048), live=round(rng.uniform(0.1, 0.95), 3))
        while c["layers"] * c["pages"] * kv * c["page"] * c["dim"] > 1 << 27:
            c["layers"] = max(1, c["layers"] // 2)
            c["pages"] = max(16, c["pages"] // 2)
    return c


def _lengths(c):
    """New and cached positions of each sequence (packed prompts differ in length; the first has the longest)."""
    r = random.Random(c["mix"])
    n = c["seqs"]
    new = [c["new"] if i == 0 or c["new"] == 1 else r.randint(max(1, c["new"] // 4), c["new"]) for i in range(n)]
    old = [c["cached"] if i == 0 or not c["cached"] else r.randint(c["cached"] // 4, c["cached"]) for i in range(n)]
    return new, old


def _groups(c):
    """Group bounds, prefix length of each group and own positions of each sequence of a shared case."""
    r = random.Random(c["mix"])
    n, g = c["seqs"], c["groups"]
    cuts = [0] + sorted(r.sample(range(1, n), g - 1)) + [n] if g else [0]
    prefix = [c["prefix"] if i == 0 else r.randint(max(1, c["prefix"] // 3), c["prefix"]) for i in range(g)]
    mine = [c["own"] if i == 0 else r.randint(max(1, c["own"] // 4), c["own"]) for i in range(n)]
    return cuts, prefix, mine


def _lives(c):
    """Which pages of a fragmented pool are live, and how many sequences hold each."""
    r = random.Random(c["mix"])
    return [r.choice([1, 1, 1, 2, 5]) if r.random() < c["live"] else 0 for _ in range(c["pages"])]


# ------------------------------------------------------------------ the inputs
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _randn(gen, shape, dtype, std):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    return x.normal_(0.0, std, generator=gen)


def _held(table, pages):
    """How many entries of the table name each page."""
    return torch.bincount(table[table >= 0], minlength=pages).to(torch.int32)


def _rope_table(n, dim):
    ang = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * torch.pow(
        500000.0, -2.0 * torch.arange(dim // 2, dtype=torch.float64, device=DEV) / dim)
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()


def _pool(gen, layers, pages, c):
    shape = (layers, pages, c["kv_heads"], c["page"], c["dim"])
    return _randn(gen, shape, torch.float16, 1.0), _randn(gen, shape, torch.float16, 0.5)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    r = random.Random(seed * 7919 + c["mix"])
    s = {"case": c}
    ps = c["page"]
    if c["kind"] in ("append", "prompt"):
        new, old = _lengths(c)
        lens = [a + b for a, b in zip(new, old)]
        need = [-(-n // ps) for n in lens]
        pages = sum(need) + 3
        ids = r.sample(range(pages), sum(need))  # pages in no order
        rows = [[ids.pop() for _ in range(n)] + [-1] * (max(need) - n) for n in need]
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        s["k"], s["v"] = _pool(gen, 1, pages, c)
        t, hq, hk, d = start[-1], c["heads"], c["kv_heads"], c["dim"]
        s.update(table=_i32(rows), lens=_i32(lens), start=_i32(start), max_len=max(lens), max_new=max(new))
        if c["kind"] == "append":
            qkv = _randn(gen, (t, hq + 2 * hk, d), TYPES[c["type"]], 1.0)  # as the product writes it
            s.update(q=qkv[:, :hq], new_k=qkv[:, hq:hq + hk], new_v=qkv[:, hq + hk:], rope=_rope_table(max(lens), d),
                     out=torch.empty((t, hq, d), dtype=TYPES[c["q_out"]], device=DEV))
        else:
            s["q"] = _randn(gen, (t, hq, d), TYPES[c["type"]], 1.5)
            s["out"] = torch.empty_like(s["q"])
        s["refs"] = _held(s["table"], pages)
    elif c["kind"] == "shared":
        cuts, prefix, mine = _groups(c)
        of = [next((g for g in range(c["groups"]) if cuts[g] <= i < cuts[g + 1]), -1) for i in range(c["seqs"])]
        lens = [(prefix[g] if g >= 0 else 0) + m for g, m in zip(of, mine)]
        whole = [p // ps for p in prefix]  # pages that every sequence of the group holds
        need = [-(-n // ps) - (whole[g] if g >= 0 else 0) for g, n in zip(of, lens)]
        pages = sum(whole) + sum(need) + 3
        ids = r.sample(range(pages), sum(whole) + sum(need))
        common = [[ids.pop() for _ in range(w)] for w in whole]
        rows = [(common[g] if g >= 0 else []) + [ids.pop() for _ in range(n)] for g, n in zip(of, need)]
        wide = max(map(len, rows))
        s["k"], s["v"] = _pool(gen, 1, pages, c)
        for g in range(c["groups"]):  # the last, part-filled page of the prefix: a copy in each sequence
            part = prefix[g] % ps
            first = cuts[g]
            if part:
                to = torch.tensor([rows[i][whole[g]] for i in range(first, cuts[g + 1])], device=DEV)
                for p in (s["k"], s["v"]):
                    p[0, to, :, :part] = p[0, rows[first][whole[g]], :, :part].clone()
        s.update(table=_i32([x + [-1] * (wide - len(x)) for x in rows]), lens=_i32(lens), max_len=max(lens),
                 cuts=_i32(cuts) if c["groups"] else None, prefix=_i32(prefix) if c["groups"] else None,
                 max_prefix=max(prefix, default=0))
        s["refs"] = _held(s["table"], pages)
        s["q"] = _randn(gen, (c["seqs"], c["heads"], c["dim"]), TYPES[c["type"]], 1.5)
        s["out"] = torch.empty_like(s["q"])
    elif c["kind"] == "fork":
        mix = random.Random(c["mix"])
        n, m = c["prompts"], c["samples"]
        lens = [c["length"] if i == 0 else mix.randint(max(1, c["length"] // 2), c["length"]) for i in range(n)]
        need = [-(-x // ps) for x in lens]
        pages = sum(need) + n * m + 2
        ids = r.sample(range(pages), sum(need))
        refs = [0] * pages
        rows = [[-1] * max(need) for _ in range(n * (m + 1))]
        for i, k in enumerate(need):
            for j in range(k):
                rows[i][j] = ids.pop()
                refs[rows[i][j]] = 1
        s["k"], s["v"] = _pool(gen, c["layers"], pages, c)
        s.update(table=_i32(rows), lens=_i32(lens + [0] * (n * m)), refs=_i32(refs), served=_i32([0] * (n * m)),
                 src=_i32([i for i in range(n) for _ in range(m)]), dst=_i32(range(n, n * (m + 1))))
    else:
        refs = _lives(c)
        held = [p for p, k in enumerate(refs) for _ in range(k)]
        r.shuffle(held)
        wide = -(-len(held) // 8)  # eight sequences hold them
        rows = [held[i * wide:(i + 1) * wide] for i in range(8)]
        s["k"], s["v"] = _pool(gen, c["layers"], c["pages"], c)
        s.update(table=_i32([x + [-1] * (max(1, wide) - len(x)) for x in rows]), lens=_i32([len(x) * ps for x in rows]),
                 refs=_i32(refs))
        s.update(table_out=torch.empty_like(s["table"]), refs_out=torch.empty_like(s["refs"]), live=_i32([0]))
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    import ane_amd as ane

    c = s["case"]
    kind = c["kind"]
    cache = s.get("cache")
    if cache is None:  # the cache's handle and a workspace, which a serving program makes once
        cache = s["cache"] = ane.PagedCache(c.get("heads", c["kv_heads"]), s["k"], s["v"], s["table"], s["lens"], s["refs"])
        s["work"] = (ane.attention_prompt_workspace(cache, s["start"].numel() - 1, s["q"].shape[0], s["max_len"])
                     if kind == "prompt" else
                     ane.attention_shared_workspace(cache, c["seqs"], c["groups"], s["max_prefix"], s["max_len"])
                     if kind == "shared" else ane.pages_workspace(cache))
    if kind == "append":
        ane.paged_rope_append(cache, 0, s["start"], s["q"], s["new_k"], s["new_v"], s["rope"], s["out"])
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if kind == "prompt":
        ane.attention_prompt(cache, 0, s["start"], s["q"], s["out"], max_len=s["max_len"], workspace=s["work"])
        return s["out"]
    if kind == "shared":
        ane.attention_shared(cache, 0, s["q"], s["out"], max_len=s["max_len"], group_start=s["cuts"],
                             prefix_len=s["prefix"], max_prefix=s["max_prefix"], workspace=s["work"])
        return s["out"]
    if kind == "fork":
        ane.pages_free(cache, s["dst"])
        ane.pages_fork(cache, s["src"], s["dst"], s["served"], workspace=s["work"])
        return {"k": s["k"], "v": s["v"], "table": s["table"], "lens": s["lens"], "refs": s["refs"], "served": s["served"]}
    ane.pages_compact(cache, table_out=s["table_out"], refs_out=s["refs_out"], n_live=s["live"], workspace=s["work"])
    return {"k": s["k"], "v": s["v"], "table": s["table_out"], "refs": s["refs_out"], "live": s["live"]}


def _gather(pool, table, n, ps):
    """[sequences][kv heads][n][dim] in 32 bits: the first n positions of every sequence, in order."""
    j = torch.arange(n, device=DEV)
    page = table[:, (j // ps).clamp(max=table.shape[1] - 1)].long().clamp(min=0)
    return pool[0][page, :, (j % ps)[None, :]].float().transpose(1, 2).contiguous()


def _attend(q, k, v, seen, scale):
    """Softmax attention of q [s][kv][rows][dim] on k, v [s][kv][n][dim], key j seen by a row where j < seen; rows that
    see nothing give zeros."""
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    j = torch.arange(k.shape[2], device=DEV)
    sc.masked_fill_(j >= seen[..., None], -math.inf)
    top = sc.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = sc.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)


def _plain(s):
    c = s["case"]
    kind, ps = c["kind"], c["page"]
    if kind in ("append", "prompt"):
        start = s["start"].long()
        t = s["q"].shape[0]
        seq = torch.bucketize(torch.arange(t, device=DEV), start[1:], right=True)
        i = torch.arange(t, device=DEV) - start[seq]
        pos = s["lens"].long()[seq] - (start[1:] - start[:-1])[seq] + i
    if kind == "append":
        rot = s["rope"][pos][:, None]

        def turn(x):
            x = x.float()
            a, b, co, si = x[..., 0::2], x[..., 1::2], rot[..., 0], rot[..., 1]
            return torch.stack([a * co - b * si, a * si + b * co], dim=-1).flatten(-2)

        page = s["table"][seq, pos // ps].long()
        s["out"].copy_(turn(s["q"]))
        at = (page, torch.arange(c["kv_heads"], device=DEV)[:, None], pos % ps)
        s["k"][0].index_put_(at, turn(s["new_k"]).to(torch.float16).transpose(0, 1))
        s["v"][0].index_put_(at, s["new_v"].to(torch.float16).transpose(0, 1))
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if kind == "prompt":
        n, g = c["seqs"], c["heads"] // c["kv_heads"]
        q = torch.zeros((n, s["max_new"], c["heads"], c["dim"]), device=DEV)
        q[seq, i] = s["q"].float()
        seen = torch.zeros((n, s["max_new"]), dtype=torch.long, device=DEV)
        seen[seq, i] = pos + 1
        q = q.view(n, s["max_new"], c["kv_heads"], g, c["dim"]).permute(0, 2, 3, 1, 4).reshape(n, c["kv_heads"], -1, c["dim"])
        seen = seen[:, None, None].expand(n, 1, g, s["max_new"]).reshape(n, 1, -1)
        k, v = (_gather(s[x], s["table"], s["max_len"], ps) for x in "kv")
        o = _attend(q, k, v, seen, 1.0 / math.sqrt(c["dim"]))
        o = o.view(n, c["kv_heads"], g, s["max_new"], c["dim"]).permute(0, 3, 1, 2, 4).reshape(n, s["max_new"], c["heads"], c["dim"])
        s["out"].copy_(o[seq, i])
        return s["out"]
    if kind == "shared":
        n, g = c["seqs"], c["heads"] // c["kv_heads"]
        q = s["q"].float().view(n, c["kv_heads"], g, c["dim"])
        k, v = (_gather(s[x], s["table"], s["max_len"], ps) for x in "kv")
        o = _attend(q, k, v, s["lens"].long()[:, None, None].expand(n, 1, g), 1.0 / math.sqrt(c["dim"]))
        s["out"].copy_(o.reshape(n, c["heads"], c["dim"]))
        return s["out"]
    if kind == "fork":
        table, lens, refs, src, dst = s["table"], s["lens"], s["refs"], s["src"].long(), s["dst"].long()
        held = table[dst]
        refs.index_add_(0, held[held >= 0].long(), torch.full_like(held[held >= 0], -1))
        table[dst] = -1
        lens[dst] = 0
        n = lens[src].long()
        whole, part = n // ps, n % ps
        free = torch.nonzero(refs == 0).flatten()
        fits = (part > 0).long().cumsum(0) <= free.numel()
        s["served"].copy_(fits)
        j = torch.arange(table.shape[1], device=DEV)
        row = table[src].masked_fill(j >= whole[:, None], -1)
        taken = torch.nonzero(fits & (part > 0)).flatten()
        fresh = free[:taken.numel()]
        origin = table[src[taken], whole[taken]].long()
        row[taken, whole[taken]] = fresh.to(torch.int32)
        table[dst] = row.masked_fill(~fits[:, None], -1)
        lens[dst] = n.masked_fill(~fits, 0).to(torch.int32)
        held = table[dst]
        refs.index_add_(0, held[held >= 0].long(), torch.ones_like(held[held >= 0]))
        used = torch.arange(ps, device=DEV) < part[taken][:, None]
        used = used[None, :, None, :, None]
        for pool in (s["k"], s["v"]):
            pool[:, fresh] = torch.where(used, pool[:, origin], pool[:, fresh])
        return {"k": s["k"], "v": s["v"], "table": table, "lens": lens, "refs": refs, "served": s["served"]}
    live = s["refs"] > 0
    n = live.sum()
    at = torch.arange(live.numel(), device=DEV)
    mover, hole = torch.nonzero(live & (at >= n)).flatten(), torch.nonzero(~live & (at < n)).flatten()
    to = at.clone()
    to[mover] = hole
    s["table_out"].copy_(torch.where(s["table"] >= 0, to[s["table"].long().clamp(min=0)].to(torch.int32), s["table"]))
    s["refs_out"].copy_(s["refs"])
    s["refs_out"][hole] = s["refs"][mover]
    s["refs_out"][mover] = 0
    s["live"].copy_(n)
    s["k"][:, hole] = s["k"][:, mover]
    s["v"][:, hole] = s["v"][:, mover]
    return {"k": s["k"], "v": s["v"], "table": s["table_out"], "refs": s["refs_out"], "live": s["live"]}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] in ("append", "prompt"):
        new, old = _lengths(c)
        t, size = sum(new), 4 if c["type"] == "f32" else 2
        if c["kind"] == "append":
            out = 4 if c["q_out"] == "f32" else 2
            rope = 4 * c["dim"] * max(a + b for a, b in zip(new, old))
            return {"bytes": t * c["dim"] * (c["heads"] * (size + out) + 2 * c["kv_heads"] * (size + 2))
                    + min(rope, 4 * c["dim"] * t), "flops": 3 * t * c["dim"] * (c["heads"] + c["kv_heads"])}
        pairs = sum(n * m + n * (n + 1) // 2 for n, m in zip(new, old))
        return {"bytes": 2 * t * c["heads"] * c["dim"] * size + 4 * c["kv_heads"] * c["dim"] * (t + sum(old)),
                "flops": 4 * c["dim"] * c["heads"] * pairs}
    if c["kind"] == "shared":
        cuts, prefix, mine = _groups(c)
        size = 4 if c["type"] == "f32" else 2
        pairs = sum(mine) + sum(p * (b - a) for p, a, b in zip(prefix, cuts, cuts[1:]))
        return {"bytes": 2 * c["seqs"] * c["heads"] * c["dim"] * size + 4 * c["kv_heads"] * c["dim"] * (sum(mine) + sum(prefix)),
                "flops": 4 * c["dim"] * c["heads"] * pairs}
    row = 4 * c["kv_heads"] * c["dim"] * c["layers"]  # one position's keys and values in all layers
    if c["kind"] == "fork":
        mix = random.Random(c["mix"])
        lens = [c["length"] if i == 0 else mix.randint(max(1, c["length"] // 2), c["length"]) for i in range(c["prompts"])]
        return {"bytes": 2 * row * c["samples"] * sum(n % c["page"] for n in lens)
                + 8 * sum(-(-n // c["page"]) for n in lens) * (c["samples"] + 1), "flops": 0}
    refs = _lives(c)
    n = sum(k > 0 for k in refs)
    moved = sum(k > 0 for k in refs[n:])
    return {"bytes": 2 * row * c["page"] * moved + 8 * (sum(refs) + len(refs)), "flops": 0}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c, ps = case, case["page"]
    if c["kind"] in ("append", "prompt"):
        new, old = _lengths(c)
    if c["kind"] == "append":
        out = s["q"].double().clone()
        k, v = s["k"].double(), s["v"].double()
        first = 0
        for i, (n, m) in enumerate(zip(new, old)):
            at = torch.arange(m, m + n, device=DEV)
            z = torch.view_as_complex(s["rope"][at].double())[:, None]

            def turn(x):
                x = torch.view_as_complex(x.double().reshape(x.shape[0], x.shape[1], -1, 2).contiguous())
                return torch.view_as_real(x * z).reshape(x.shape[0], x.shape[1], -1)

            rows = slice(first, first + n)
            first += n
            page = s["table"][i, at // ps].long()
            out[rows] = turn(s["q"][rows])
            k[0, page, :, at % ps] = turn(s["new_k"][rows])
            v[0, page, :, at % ps] = s["new_v"][rows].double()
        return {"q": out, "k": k, "v": v}
    if c["kind"] in ("prompt", "shared"):
        if c["kind"] == "shared":
            new, old = [1] * c["seqs"], [n - 1 for n in s["lens"].tolist()]
        g, out, first = c["heads"] // c["kv_heads"], s["q"].double().clone(), 0
        for i, (n, m) in enumerate(zip(new, old)):
            at = torch.arange(m + n, device=DEV)
            page = s["table"][i, at // ps].long()
            hidden = at[None, :] > torch.arange(m, m + n, device=DEV)[:, None]
            for h in range(c["heads"]):
                k, v = (s[x][0, page, h // g, at % ps].double() for x in "kv")
                w = s["q"][first:first + n, h].double() @ k.t().contiguous() / math.sqrt(c["dim"])
                out[first:first + n, h] = torch.softmax(w.masked_fill_(hidden, -math.inf), dim=-1) @ v
            first += n
        return out
    k, v = s["k"].double(), s["v"].double()
    if c["kind"] == "fork":
        table, lens, refs, served = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist(), []
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            n = lens[a]
            for j in range(n // ps):
                table[b][j] = table[a][j]
                refs[table[a][j]] += 1
            if n % ps:
                table[b][n // ps] = p = refs.index(0)
                refs[p] = 1
                for x in (k, v):
                    x[:, p, :, :n % ps] = x[:, table[a][n // ps], :, :n % ps]
            lens[b] = n
            served.append(1)
        return {"k": k, "v": v, "table": _i32(table), "lens": _i32(lens), "refs": _i32(refs), "served": _i32(served)}
    table, refs = s["table"].tolist(), s["refs"].tolist()
    n = sum(x > 0 for x in refs)
    to = {}
    for p in range(n, len(refs)):
        if refs[p]:
            to[p] = q = refs.index(0)
            refs[q], refs[p] = refs[p], 0
            for x in (k, v):
                x[:, q] = x[:, p]
    return {"k": k, "v": v, "table": _i32([[to.get(p, p) for p in row] for row in table]), "refs": _i32(refs), "live": _i32([n])}
