"""Attention under a rule (include/ane_decode.h: ane_hip_attention_rule;
ane_amd/csrc/paged_attention.hip): scores capped or lowered with the distance,
windows, documents, prefixes seen from both sides; element by element against
the formula in 64 bits.

The bound, u = 2^-24: a score is off by (hd + 8) u A_j as in test_paged.py, A_j =
scale sum |q k|; the cap passes errors on at most as they are (its slope is at
most 1) and adds its own, 2^-22 of a capped score (fp16: 2^-20), which is at most
A_j; the distance adds roundings of slope, product and sum, 4 u (A_j + B_j), B_j =
|slope (p - j)|.  With D_j the sum of these and w_j a row's weights, the weights'
relative errors, of which normalising takes the common part off, move the result
by at most 2 sum w_j D_j max|v|, first order; taken twice.  Exponential, its
argument, the parts of weights and the sums over n keys are as there: (2 n + 64) u
max|v|; 16-bit activations round weights and result, 2^-10 max|v| each.
"""
import ctypes
import math
import random
import shutil
import subprocess

import pytest

import ane_amd
from ane_amd import AneError, AttentionRule
from tests.test_paged import P, ROOT, dt, i32, make_cache, randq, raw_cache, seq_kv

U = 2.0 ** -24


# ------------------------------------------------------------------ CPU
def test_struct_layout_matches_c(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    src = tmp_path / "layout.c"
    names = ("softcap", "window", "slopes", "first", "prefix")
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ane_decode.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu ", offsetof(struct ane_attention_rule, {n}));\n' for n in names)
                   + 'printf("%zu\\n", sizeof(struct ane_attention_rule)); return 0; }\n')
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(AttentionRule, n).offset for n, _ in AttentionRule._fields_] + [ctypes.sizeof(AttentionRule)]


def raw_rule(cap=0.0, window=0, slopes=None, first=None, prefix=None):
    r = AttentionRule.__new__(AttentionRule)
    ctypes.Structure.__init__(r, cap, window, slopes, first, prefix)
    return r


def call(c=None, layer=0, n=2, qs=P, T=4, ml=0, rule=True, ty=0, q=P, qstr=1024, scale=0.1, out=P, ostr=1024, ws=P, wsb=1 << 40):
    c = raw_cache() if c is None else c
    rule = raw_rule() if rule is True else rule
    return ane_amd.lib().ane_hip_attention_rule(ctypes.byref(c), layer, None, n, qs, T, ml, ctypes.byref(rule) if rule else None,
                                                ty, q, qstr, scale, out, ostr, ws, wsb, None)


INVALID, POINTER, WORKSPACE = 1, 2, 8


@pytest.mark.parametrize("kw,st", [
    (dict(rule=None), POINTER), (dict(c=raw_cache(head_dim=96)), INVALID), (dict(layer=2), INVALID), (dict(ty=2), INVALID),
    (dict(scale=0.0), INVALID), (dict(qs=None, T=3), INVALID), (dict(rule=raw_rule(cap=-1.0)), INVALID),
    (dict(rule=raw_rule(cap=math.nan)), INVALID), (dict(rule=raw_rule(cap=math.inf)), INVALID),
    (dict(rule=raw_rule(cap=1e-7)), INVALID), (dict(rule=raw_rule(cap=2e6)), INVALID), (dict(rule=raw_rule(slopes=P + 2)), INVALID),
    (dict(rule=raw_rule(first=P + 1)), INVALID), (dict(rule=raw_rule(prefix=P + 3)), INVALID), (dict(q=None), POINTER),
    (dict(out=None), POINTER), (dict(q=P + 4), INVALID), (dict(qstr=1000), INVALID), (dict(n=0), 0), (dict(T=0), 0),
    (dict(T=(1 << 23) + 1), INVALID)])
def test_refusals(kw, st):
    assert call(**kw) == st


def test_workspace():
    f = ane_amd.lib().ane_hip_attention_rule_workspace_size
    c, none = raw_cache(max_pages=4096, page_size=64), ctypes.byref(raw_rule())
    plain = ane_amd.lib().ane_hip_attention_prompt_workspace_size(ctypes.byref(c), 1, 1, 8192)
    assert f(ctypes.byref(c), 1, 1, 8192, none) == plain > 0
    assert f(ctypes.byref(c), 1, 1, 8192, ctypes.byref(raw_rule(window=64))) < plain
    both = raw_rule(window=64, prefix=P)  # a window's keys, and what may lie ahead of a chunk's first token
    assert f(ctypes.byref(c), 1, 1, 8192, ctypes.byref(both)) < plain
    many = ane_amd.lib().ane_hip_attention_prompt_workspace_size(ctypes.byref(c), 1, 4000, 4040)
    assert f(ctypes.byref(c), 1, 4000, 4040, ctypes.byref(both)) == many
    assert call(c=c, n=1, qs=None, T=1, ml=8192, wsb=plain - 1) == WORKSPACE
    assert call(c=c, n=1, qs=None, T=1, ml=8192, ws=None) == WORKSPACE


def test_rule_wrapper_refuses_wrong_tensors():
    import torch

    for kw in (dict(slopes=torch.zeros(4, dtype=torch.float64)), dict(first=torch.zeros(4)), dict(prefix=torch.zeros(4)),
               dict(first=torch.zeros((2, 2), dtype=torch.int32)), dict(prefix=torch.zeros(8, dtype=torch.int32)[::2]),
               dict(window=-1), dict(window=1 << 32)):
        with pytest.raises(ValueError):
            AttentionRule(**kw)


# ------------------------------------------------------------------ the formula
def sees(pos, n, length, window, first, prefix):
    """[tokens][n] truth values."""
    import torch

    p, j = torch.as_tensor(pos, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    y = (j <= p) | (j < prefix)
    if window:
        y = y & (p - j < window)
    if first is not None:
        y = y & (j >= torch.as_tensor(first, device="cuda")[:, None])
    return y & (p >= 0) & (j < length)


def check(c, layer, s, q, got, pos, scale, cap=0.0, slopes=None, window=0, first=None, prefix=0):
    """Rows q [m][heads][hd] of sequence s at positions pos."""
    import torch

    G, hd = c.n_heads // c.n_kv_heads, c.head_dim
    n = int(c.kv_len[s])
    y = sees(pos, n, n, window, first, prefix)
    k, v = seq_kv(c, layer, s, n) if n else (None, None)
    dist = (torch.as_tensor(pos, device="cuda")[:, None] - torch.arange(n, device="cuda")[None]).abs().double()
    for h in range(c.n_heads):
        g = got[:, h].double()
        if n == 0:
            assert not g.any()
            continue
        kk, vv = (torch.nan_to_num(x[h // G], nan=0.0, posinf=0.0, neginf=0.0) for x in (k, v))
        raw = q[:, h].double() @ kk.t().contiguous() * scale
        A = q[:, h].double().abs() @ kk.abs().t().contiguous() * scale
        sc = torch.tanh(raw / cap) * cap if cap else raw
        B = dist * abs(float(slopes[h])) if slopes is not None else torch.zeros_like(dist)
        if slopes is not None:
            sc = sc - float(slopes[h]) * dist
        sc = sc.masked_fill(~y, -math.inf)
        w = torch.exp(sc - sc.amax(1, keepdim=True).clamp(min=-1e300))
        w = torch.nan_to_num(w / w.sum(1, keepdim=True).clamp(min=1e-300)).masked_fill(~y, 0.0)
        D = ((hd + 12) * A + (4 if q.dtype == torch.float32 else 16) * A * bool(cap) + 4 * (A + B)) * U
        vmax = vv.abs().amax(1)[None].masked_fill(~y, 0.0).amax(1)
        tol = (4 * (w * D).sum(1) + (2 * y.sum(1) + 64) * U) * vmax
        if q.dtype == torch.float16:
            tol = tol + 2 * 2.0 ** -10 * vmax + 2.0 ** -24
        err = (g - w @ vv).abs()
        assert bool((err <= tol[:, None]).all()), (s, h, float((err - tol[:, None]).max()), float(err.max()))


def run(c, new, ty, layer=0, seqs=None, cap=0.0, slopes=None, window=0, first=None, prefix=None, std=1.5, single=False, q=None,
        scale=None, **kw):
    import torch

    T = sum(new)
    q = randq(T, c.n_heads, c.head_dim, dt(ty), seed=T + window, std=std) if q is None else q
    out = torch.full_like(q, 5.0)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    rule = AttentionRule(cap, None if slopes is None else torch.tensor(slopes, device="cuda"), window,
                         None if first is None else i32(first), None if prefix is None else i32(prefix))
    ane_amd.attention_prompt(c, layer, None if single else i32(start), q, out, seqs=None if seqs is None else i32(seqs), rule=rule,
                             scale=scale, **kw)
    lens = c.kv_len.tolist()
    for i, n in enumerate(new):
        if n == 0:
            continue
        s = i if seqs is None else seqs[i]
        a, b = start[i], start[i + 1]
        check(c, layer, s, q[a:b], out[a:b], list(range(lens[s] - n, lens[s])), scale or c.head_dim ** -0.5, cap,
              None if slopes is None else torch.tensor(slopes), window, None if first is None else first[a:b],
              0 if prefix is None else min(prefix[i], lens[s]))
    return q, out, rule


def alibi(h):
    return [2.0 ** (-8.0 * (i + 1) / h) for i in range(h)]


def documents(new, old, n, seed):
    """The first position of each token's document: n random borders a sequence, the first document from 0."""
    r, out = random.Random(seed), []
    for m, o in zip(new, old):
        cuts = sorted(o + r.randrange(m) for _ in range(n)) if m else []
        at = 0
        for p in range(o, o + m):
            if p in cuts:
                at = p
            out.append(at)
    return out


RULES = {
    "none": {}, "cap": dict(cap=30.0), "cap_low": dict(cap=2.0), "slopes": dict(slopes=True), "window1": dict(window=1),
    "window16": dict(window=16), "window63": dict(window=63), "window64": dict(window=64), "window65": dict(window=65),
    "window700": dict(window=700), "docs": dict(first=4), "prefix": dict(prefix=True),
    "cap_slopes_window": dict(cap=50.0, slopes=True, window=100), "docs_prefix": dict(first=2, prefix=True),
    "all": dict(cap=20.0, slopes=True, window=200, first=3, prefix=True)}
SHAPES = [
    # type, hd, heads, kv, ps, new, old: 32-row tiles (in parts and not), 128-row tiles
    ("f32", 128, 8, 2, 16, [40, 1, 0, 3], [0, 99, 7, 300]),
    ("f16", 128, 4, 4, 48, [130, 17], [0, 1000]),
    ("f32", 64, 12, 4, 32, [70, 5], [513, 0]),
    ("f16", 64, 6, 2, 16, [2, 2, 2], [1, 700, 63]),
    ("f32", 128, 32, 8, 64, [700, 420, 33], [0, 200, 1000]),
    ("f16", 128, 32, 8, 16, [600, 601, 90], [64, 0, 900]),
    ("f32", 64, 24, 8, 48, [500, 777], [333, 0]),
    ("f16", 64, 40, 8, 16, [700, 640], [0, 100])]


@pytest.mark.gpu
@pytest.mark.parametrize("name", RULES)
@pytest.mark.parametrize("ty,hd,heads,kv,ps,new,old", SHAPES)
def test_rules(ane, ty, hd, heads, kv, ps, new, old, name):
    r = dict(RULES[name])
    c = make_cache([a + b for a, b in zip(new, old)], heads, kv, hd, ps, seed=len(name), layers=2)
    if "slopes" in r:
        r["slopes"] = alibi(heads)
    if "first" in r:
        r["first"] = documents(new, old, r["first"], heads)
    if "prefix" in r:
        r["prefix"] = [(37 * i + 200) % (a + b + 20) for i, (a, b) in enumerate(zip(new, old))]
    run(c, new, ty, layer=1, **r)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd", [("f32", 128), ("f16", 128), ("f32", 64), ("f16", 64)])
@pytest.mark.parametrize("name", ["cap", "slopes", "window64", "window700", "cap_slopes_window"])
@pytest.mark.parametrize("lens", [[1], [4000], [3, 1500, 64, 65, 2000], [100] * 300])
def test_single_tokens(ane, ty, hd, name, lens):
    r = dict(RULES[name])
    heads, kv = (8, 2) if len(lens) > 100 else (32, 8)
    if "slopes" in r:
        r["slopes"] = alibi(heads)
    c = make_cache(lens, heads, kv, hd, 16, seed=len(lens))
    run(c, [1] * len(lens), ty, single=True, max_len=max(lens), **r)
    if len(lens) == 5:
        run(c, [1] * 3, ty, single=True, seqs=[4, 1, 3], **r)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd", [("f32", 128), ("f16", 64)])
def test_prefix_ahead_of_a_window(ane, ty, hd):
    """Chunks far into a sequence whose prefix ends behind them, inside them, before them: keys in parts by the window."""
    new, old = [45, 300, 7, 90], [4744, 900, 3000, 0]
    c = make_cache([a + b for a, b in zip(new, old)], 4, 2, hd, 32, seed=4)
    for prefix in ([4789, 1200, 3003, 90], [4750, 1000, 10, 45], [120, 950, 3010, 1]):
        for window in (953, 60, 3000):
            run(c, new, ty, prefix=prefix, window=window, cap=30.0)
    run(c, [1] * 4, ty, single=True, prefix=[4789, 5, 3007, 90], window=953)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd", [("f32", 128), ("f16", 128), ("f32", 64), ("f16", 64)])
@pytest.mark.parametrize("kw", [dict(cap=20.0), dict(slopes=True), dict(window=90), dict(window=300, cap=3.0), dict(prefix=True),
                                dict(first=True)], ids=str)
def test_many_single_tokens(ane, ty, hd, kw):
    """Batches of which every (token, kv head) gets a wave: lengths from none to 400, a bound or a window of at most 512."""
    heads, kv, n = 12, 4, 270
    r = random.Random(hd)
    lens = [r.choice([0, 1, 31, 32, 33, 64, r.randint(1, 400)]) for _ in range(n)]
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = alibi(heads)
    if "first" in kw:
        kw["first"] = [r.choice([0, max(0, m - 1), m, m // 2, 1 << 20]) for m in lens]
    if "prefix" in kw:
        kw["prefix"] = [r.randint(0, 500) for _ in lens]
    c = make_cache(lens, heads, kv, hd, 16, seed=n)
    run(c, [1] * n, ty, single=True, max_len=400, **kw)
    if "window" in kw:
        run(c, [1] * n, ty, single=True, max_len=None, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("many", [False, True])
def test_tokens_that_see_nothing(ane, ty, many):
    """Documents that begin behind their tokens, behind every length and past 31 bits; negative positions under a prefix."""
    import torch

    heads, kv, n = (32, 8, 700) if many else (4, 2, 40)
    c = make_cache([n + 20, 30, 5], heads, kv, 128, 16)
    new = [n, 12, 9]  # the last one: four tokens before position 0
    r = random.Random(3)
    first = [r.choice([0, p, p + 1, p + 9, 1 << 20, -1, -(1 << 31)]) for a, b in zip(new, (20, 18, -4)) for p in range(b, a + b)]
    q = randq(sum(new), heads, 128, dt(ty), seed=5)
    out = torch.full_like(q, 5.0)
    ane.attention_prompt(c, 0, i32([0, n, n + 12, n + 21]), q, out,
                         rule=AttentionRule(10.0, first=i32(first), prefix=i32([n + 100, 4, 3])))
    at = 0
    for i, (a, b) in enumerate(zip(new, (20, 18, -4))):
        f = [x if x >= 0 else x + (1 << 32) for x in first[at:at + a]]
        check(c, 0, i, q[at:at + a], out[at:at + a], list(range(b, a + b)), 128 ** -0.5, 10.0, first=f,
              prefix=min([n + 100, 4, 3][i], [n + 20, 30, 5][i]))
        at += a
    assert not out[n + 12:n + 16].any()


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd", [("f32", 128), ("f16", 128), ("f32", 64), ("f16", 64)])
@pytest.mark.parametrize("heads,kv,n", [(4, 2, 90), (32, 8, 900)])
def test_masked_places_hold_anything(ane, ty, hd, heads, kv, n):
    """Infinities and NaN in keys and values touch the rows that see them and no other: before the window, before the
    document, at one place that some rows see.  (fp32: what stands in masked places decides whether a tile's small weights
    get a second round, so the others are as near to the formula as ever, not the same bits.)"""
    import torch

    for kw in (dict(window=50), dict(window=50, cap=5.0), dict(window=20, slopes=alibi(heads)),
               dict(first=[p // 40 * 40 for p in range(n)])):
        c = make_cache([n], heads, kv, hd, 16, seed=n)
        q, clean, rule = run(c, [n], ty, **kw)
        j = torch.arange(n, device="cuda")
        y = sees(list(range(n)), n, n, kw.get("window", 0), kw.get("first"), 0)
        for bad, at in ((math.nan, 0), (math.inf, 17), (-math.inf, n // 2)):
            for pages in (c.k_pages, c.v_pages):
                row = (0, int(c.page_table[0, at // 16]), slice(None), at % 16)
                keep = pages[row].clone()
                pages[row] = bad
                out = torch.full_like(q, 5.0)
                ane.attention_prompt(c, 0, i32([0, n]), q, out, rule=rule)
                pages[row] = keep
                blind = ~y[:, at]
                assert bool(blind.any()) and bool(torch.isfinite(out[blind]).all())
                if ty == "f16":
                    assert torch.equal(out[blind], clean[blind])
                rows = [p for p in range(n) if bool(blind[p])]
                check(c, 0, 0, q[rows], out[rows], rows, hd ** -0.5, kw.get("cap", 0.0),
                      torch.tensor(kw["slopes"]) if "slopes" in kw else None, kw.get("window", 0),
                      [kw["first"][p] for p in rows] if "first" in kw else None)
                if pages is c.v_pages:
                    assert not torch.isfinite(out[~blind]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,n", [(4, 2, 60), (32, 8, 800)])
def test_caps_and_slopes_at_the_ends(ane, heads, kv, n):
    """Caps far below and far above the scores, slopes that leave one key, negative ones, zeros, queries at the ends."""
    c = make_cache([n], heads, kv, 128, 16, seed=1)
    for cap in (2.0 ** -20, 0.01, 1.0, 2.0 ** 20):
        run(c, [n], "f32", cap=cap)
        run(c, [n], "f16", cap=cap)
    run(c, [n], "f32", slopes=[0.0, 1e4, -0.01, 3.0] * (heads // 4))
    run(c, [n], "f32", cap=30.0, std=60.0)
    run(c, [n], "f32", cap=50.0, std=1e-30)
    q = randq(n, heads, 128, dt("f32"), std=1e30)
    run(c, [n], "f32", cap=50.0, q=q)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,n", [(4, 2, 60), (32, 8, 800)])
def test_least_cap_over_largest_scores(ane, heads, kv, n):
    """|score| <= 2^-20: each weight is 1 / keys within a factor of e^(2^-19), whatever q."""
    import torch

    c = make_cache([n], heads, kv, 128, 16, seed=2)
    v = seq_kv(c, 0, 0, n)[1].double()
    for ty, std, scale in (("f32", 3e37, None), ("f32", 3e37, 9e29), ("f16", 3000.0, 9e29)):
        q = randq(n, heads, 128, dt(ty), seed=3).clamp(-4, 4) * std
        out = torch.full_like(q, 5.0)
        ane.attention_prompt(c, 0, i32([0, n]), q, out, scale=scale, rule=AttentionRule(2.0 ** -20))
        keys = torch.arange(1, n + 1, device="cuda", dtype=torch.float64)[:, None]
        for h in range(heads):
            x = v[h // (heads // kv)]
            top = x.abs().amax()
            tol = (1.01 * 2.0 ** -19 + (2 * n + 64) * U + 2 * 2.0 ** -10 * (ty == "f16")) * top
            assert bool(((out[:, h].double() - x.cumsum(0) / keys).abs() <= tol).all()), (ty, scale, h)


@pytest.mark.gpu
def test_no_rule_at_all_is_the_plain_call(ane):
    """An empty rule gives attention_prompt's bits."""
    import torch

    for heads, kv, new in ((8, 2, [50, 3]), (32, 8, [800, 500])):
        for ty in ("f32", "f16"):
            c = make_cache([n + 30 for n in new], heads, kv, 128, 16)
            q, out, _ = run(c, new, ty)
            plain = torch.zeros_like(q)
            ane.attention_prompt(c, 0, i32([0, new[0], sum(new)]), q, plain)
            assert torch.equal(out, plain)


@pytest.mark.gpu
def test_far_positions(ane):
    """Positions of which a cache has 2^30: the window and the distance at the far end, only the pages near it read."""
    import torch

    from ane_amd import PagedCache

    ps = 1 << 20
    k, v = (torch.full((1, 2, 2, ps, 64), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.full((1, 1024), -1, dtype=torch.int32, device="cuda")
    table[0, 1023] = 1
    length = (1 << 30) - 7
    gen = torch.Generator(device="cuda").manual_seed(1)
    tail = ps - 7
    for x in (k, v):
        x[0, 1, :, tail - 3000:tail] = torch.randn((2, 3000, 64), generator=gen, device="cuda").half()
    c = PagedCache(4, k, v, table, i32([length]))
    near = [x[:, 1:2, :, tail - 3000 - 8:tail].contiguous() for x in (k, v)]  # the same at small positions
    small = PagedCache(4, near[0], near[1], i32([[0]]), i32([3008]))
    for n in (1, 40):
        q = randq(n, 4, 64, dt("f32"))
        a, b = torch.zeros_like(q), torch.zeros_like(q)
        sl = torch.tensor(alibi(4), device="cuda")
        ane.attention_prompt(c, 0, i32([0, n]), q, a, rule=AttentionRule(20.0, sl, 2000))
        ane.attention_prompt(small, 0, i32([0, n]), q, b, rule=AttentionRule(20.0, sl, 2000))
        # (positions past 2^24: a distance is formed in whole numbers before it is rounded)
        assert bool(torch.isfinite(a).all()) and float((a - b).abs().max()) <= 2e-5 * float(b.abs().max())


@pytest.mark.gpu
def test_wrapper_refusals(ane):
    import torch

    c = make_cache([40, 20], 4, 2, 64, 16, fill_rest=0.0)
    q = randq(3, 4, 64, dt("f32"))
    for rule in (AttentionRule(first=i32([0, 0])), AttentionRule(prefix=i32([1])), AttentionRule(slopes=torch.zeros(3, device="cuda")),
                 AttentionRule(first=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ane.attention_prompt(c, 0, i32([0, 2, 3]), q, q.clone(), rule=rule)
    with pytest.raises(AneError):
        ane.attention_prompt(c, 0, i32([0, 2, 3]), q, q.clone(), rule=AttentionRule(-1.0))


@pytest.mark.gpu
def test_captured_calls_follow_their_tensors(ane):
    """A captured call follows lengths, documents, prefixes and slopes of each replay; eager calls between them."""
    import torch

    c = make_cache([900, 700], 8, 2, 128, 16, fill_rest=0.0)
    q = randq(60, 8, 128, dt("f32"))
    start, first, prefix = i32([0, 40, 60]), i32([0] * 60), i32([10, 0])
    sl = torch.tensor(alibi(8), device="cuda")
    rule = AttentionRule(25.0, sl, 300, first, prefix)
    work = ane.attention_prompt_workspace(c, 2, 60, 900, rule)
    out, eager = torch.zeros_like(q), torch.zeros_like(q)
    ane.attention_prompt(c, 0, start, q, out, max_len=900, workspace=work, rule=rule)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ane.attention_prompt(c, 0, start, q, out, max_len=900, workspace=work, rule=rule)
    for i in range(3):
        c.kv_len.copy_(i32([850 - 100 * i, 700 - i]))
        first.copy_(i32([(i * 300 + t) % 800 for t in range(60)]))
        prefix.copy_(i32([500 * i, 30]))
        sl.mul_(0.5)
        out.zero_()
        g.replay()
        ane.attention_prompt(c, 0, start, q, eager, max_len=900, rule=rule)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and bool(out.any())
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    out.zero_()
    torch.cuda.synchronize()
    ane.attention_prompt(c, 0, start, q, out, max_len=900, rule=rule, stream=st)
    st.synchronize()
    assert torch.equal(out, eager)


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_stay(ane):
    import torch

    c = make_cache([300, 80], 8, 2, 64, 16)
    q = randq(50, 8, 64, dt("f16"))
    out = torch.full_like(q, 5.0)
    ane.attention_prompt(c, 0, i32([2, 12, 40]), q, out, rule=AttentionRule(window=30))
    assert bool((out[:2] == 5).all()) and bool((out[40:] == 5).all()) and not bool((out[2:40] == 5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd", [("f32", 128), ("f16", 128), ("f32", 64), ("f16", 64)])
def test_negative_prefixes_are_none(ane, ty, hd):
    """-1 for a sequence without a prefix: no token sees past itself, in 32- and 128-row tiles, alone and in large batches."""
    import torch

    for new, old, heads, kv in (([40, 3, 9], [0, 300, 20], 8, 2), ([700, 420, 33], [0, 200, 1000], 32, 8)):
        c = make_cache([a + b for a, b in zip(new, old)], heads, kv, hd, 16, seed=5)
        q = randq(sum(new), heads, hd, dt(ty), seed=6)
        for window in (0, 90):
            outs = []
            for prefix in ([-1, 200, -(1 << 31)], [0, 200, 0]):
                out = torch.full_like(q, 5.0)
                ane.attention_prompt(c, 0, i32([sum(new[:i]) for i in range(len(new) + 1)]), q, out,
                                     rule=AttentionRule(30.0, window=window, prefix=i32(prefix)))
                outs.append(out)
            assert torch.equal(*outs)
            at = 0
            for i, (a, b) in enumerate(zip(new, old)):
                check(c, 0, i, q[at:at + a], outs[0][at:at + a], list(range(b, a + b)), hd ** -0.5, 30.0, window=window,
                      prefix=min([0, 200, 0][i], a + b))
                at += a
    for lens in ([1, 70, 900], [100] * 300):
        c = make_cache(lens, 8, 4, hd, 16, seed=7)
        q = randq(len(lens), 8, hd, dt(ty), seed=8)
        outs = [torch.full_like(q, 5.0) for _ in range(2)]
        for out, v in zip(outs, (-1, 0)):
            ane.attention_prompt(c, 0, None, q, out, max_len=max(lens), rule=AttentionRule(30.0, prefix=i32([v] * len(lens))))
        assert torch.equal(*outs)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("heads,kv,n", [(4, 2, 90), (32, 8, 900)])
def test_what_a_row_does_not_see_leaves_its_bits(ane, hd, heads, kv, n):
    """fp16, a cap far above the scores: a key outside the window or document that no score of its tile compares to (finite
    or not) chooses how the tile's tanh is formed, and changes no bit of a row that does not see it."""
    import torch

    for cap in (50.0, 20.0):
        for kw in (dict(window=50), dict(first=[p // 40 * 40 for p in range(n)])):
            c = make_cache([n], heads, kv, hd, 16, seed=n)
            q, clean, rule = run(c, [n], "f16", cap=cap, **kw)
            y = sees(list(range(n)), n, n, kw.get("window", 0), kw.get("first"), 0)
            for at in (0, 17, n // 2, n // 2 + 21):
                for bad in (math.inf, math.nan, 900.0):
                    row = (0, int(c.page_table[0, at // 16]), slice(None), at % 16)
                    keep = c.k_pages[row].clone()
                    c.k_pages[row] = bad
                    out = torch.full_like(q, 5.0)
                    ane.attention_prompt(c, 0, i32([0, n]), q, out, rule=rule)
                    c.k_pages[row] = keep
                    blind = ~y[:, at]
                    assert bool(blind.any()) and torch.equal(out[blind], clean[blind]), (cap, at, bad)
