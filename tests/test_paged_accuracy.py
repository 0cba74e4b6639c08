"""fp32 attention over the paged cache keeps fp32 accuracy.

tests/test_paged.py bounds the worst case of all roundings, which a kernel that
keeps 11 bits of q or of the weights still meets.  Here the error is measured as
such roundings leave it: for each row of each head, the root mean square of
(result - formula in 64 bits) over that of the result, and of those the root mean
square over all rows.  With values of random signs both are sums over the keys of
w_k v_k, the error's terms times the weight's relative error, so the ratio is the
size of that error whatever the number of keys.

What it may be (`allowed`), in units of 2^-24:
- a score is a sum of head_dim products, each of a part of q with a key: at most
  N = 2 head_dim + 8 roundings, each off by at most 1 of a partial sum.  Of scores
  around 3 (the keys that carry the weight), independent and uniform:
  3 sqrt(264) / sqrt(3) = 28;
- the exponential's argument is at most 2^4 and rounded once: 16 ln 2 / sqrt(3) =
  6.4; q in two parts 4 / sqrt(3) = 2.3, the weights as much (those that carry the
  result; the others are allowed 2^-18); together with the scores below 32;
- O takes n / 8 additions over n keys (two parts, 16 keys each), each off by at most
  1 of a sum that grows to the result: sqrt(n / 8) / sqrt(3) < sqrt(n) / 2;
- a key `margin` above the others: its score, the reference and the argument of the
  others' exponentials are of that size, each rounded once or twice: 6 margin.  Keys
  that carry the weight with scores around 8 instead of 3, of queries three times
  as large: 28 8 / 3 + 6.4, below 32 + 6 8.
Rounding the weights, or q, to fp16 once is off by 2^-12 / sqrt(3) and more: 2000 of
these units and more.
"""
import math

import pytest

from ane_amd import PagedCache
from tests.test_paged import formula, i32, make_cache, randq, share


def allowed(n, margin=0.0):
    return (32 + math.sqrt(n) / 2 + 6 * margin) * 2.0 ** -24


def ratio(got, want):
    """Root mean square, over rows, of each row's relative error (rows [..., head_dim])."""
    err = (got.double() - want).square().mean(-1)
    return float((err / want.square().mean(-1)).mean().sqrt())


# ------------------------------------------------------------------ the measure itself, on the CPU
def parts(x, n=2):
    """fp32 values as the sum of n fp16 parts, kept apart."""
    import torch

    out = []
    for _ in range(n):
        out.append(x.half().float())
        x = x - out[-1]
    return out


def model(q, k, v, q_parts=2, w_parts=2, lift=11.0, again=True):
    """The kernels' arithmetic over one tile: scores of q in parts, weights 2^lift
    large in parts, what is left of those below 2^-3 in two more."""
    import torch

    s = sum(p @ k.t() for p in parts(q * 8192, q_parts)) / 8192  # (q up to fp16's range, as the kernels scale it)
    s = s * (q.shape[-1] ** -0.5 * math.log2(math.e))
    x = torch.exp2(s - s.amax(-1, keepdim=True) + lift)
    ps = parts(x, w_parts)
    o = sum(p @ v for p in ps)
    if again:
        rest = torch.where(x < 0.125, x - sum(ps), torch.zeros(())) * 2.0 ** 38
        o = o + sum(p @ v for p in parts(rest)) * 2.0 ** -38
    return o / x.sum(-1, keepdim=True)


def planted(n, hd, rows, margin, seed):
    """q [rows][hd], k, v [n][hd] as fp32; margin: key n // 3 scores that much above
    the mean of the others, with a value of zeros."""
    import torch

    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn((m, hd), generator=g) for m in (rows, n, n))
    k, v = k.half().float(), v.half().float()
    if margin:
        q[:, 0], k[:, 0] = 4.0, 0.0
        k[n // 3], v[n // 3] = 0.0, 0.0
        k[n // 3, 0] = float(torch.tensor(margin * hd ** 0.5 / 4).half())
    else:
        q = q * 1.5
    return q, k, v


@pytest.mark.parametrize("hd,n,margin", [(128, 7, 0), (128, 128, 0), (128, 4096, 0), (64, 300, 0), (64, 33, 14), (128, 700, 18),
                                         (128, 4096, 22), (64, 20, 30)])
def test_the_measure_tells_parts_apart(hd, n, margin):
    """The model meets it; without the low part of q or of the weights, or of small
    weights below a large one, it does not."""
    import torch

    q, k, v = planted(n, hd, 24, margin, 3)
    s = q.double() @ k.double().t() * hd ** -0.5
    want = torch.softmax(s, -1) @ v.double()
    assert ratio(model(q, k, v), want) < allowed(n, margin)
    assert ratio(model(q, k, v, q_parts=1), want) > 2 * allowed(n, margin)
    assert ratio(model(q, k, v, w_parts=1, again=False), want) > 2 * allowed(n, margin)
    if margin >= 18:
        assert ratio(model(q, k, v, lift=6.0, again=False), want) > 2 * allowed(n, margin)


# ------------------------------------------------------------------ prompts
PROMPTS = [
    # head_dim, heads, kv heads, page, new tokens, cached positions: 32 rows a
    # workgroup, with the keys whole and in parts; then 128 rows
    (128, 8, 2, 16, [128], [0]),
    (128, 4, 1, 64, [33, 1, 200], [0, 700, 40]),
    (64, 6, 2, 48, [130, 50], [14, 333]),
    (128, 4, 1, 16, [9, 2], [5000, 7001]),
    (64, 8, 2, 32, [5], [9000]),
    (128, 32, 8, 16, [1500, 30, 700], [0, 5, 300]),
    (64, 32, 8, 48, [1300, 900], [14, 333]),
    (128, 32, 8, 16, [256] * 9, [0, 3, 0, 17, 0, 0, 200, 0, 1]),
]


def check_heads(c, layer, s, q, got, seen, margin=0.0):
    """Rows q [m][heads][hd], row i seeing seen[i] positions; some heads of many."""
    heads = sorted({0, 1, c.n_heads // 2, c.n_heads - 1} & set(range(c.n_heads)))
    G = c.n_heads // c.n_kv_heads
    for h in heads:
        g = h // G
        view = PagedCache(1, c.k_pages[:, :, g:g + 1].contiguous(), c.v_pages[:, :, g:g + 1].contiguous(), c.page_table,
                          c.kv_len)
        want, _ = formula(view, layer, s, q[:, h:h + 1], seen, c.head_dim ** -0.5)
        r = ratio(got[:, h:h + 1], want)
        assert r < allowed(max(seen), margin), (s, h, r, r / allowed(max(seen), margin))


@pytest.mark.gpu
@pytest.mark.parametrize("std,margin", [(1.5, 0), (3.0, 8)])
@pytest.mark.parametrize("hd,heads,kv,ps,new,old", PROMPTS)
def test_prompts(ane, hd, heads, kv, ps, new, old, std, margin):
    import torch

    c = make_cache([a + b for a, b in zip(new, old)], heads, kv, hd, ps, seed=11)
    q = randq(sum(new), heads, hd, torch.float32, std=std)
    out = torch.zeros_like(q)
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    ane.attention_prompt(c, 0, i32(start), q, out, max_len=max(a + b for a, b in zip(new, old)))
    for i, n in enumerate(new):
        at = sorted({0, n // 2, n - 1} | set(range(0, n, 1 + n // 60)))
        rows = torch.tensor([start[i] + t for t in at], device="cuda")
        check_heads(c, 0, i, q[rows], out[rows], [old[i] + t + 1 for t in at], margin)


# ------------------------------------------------------------------ single tokens
SINGLE = [
    # head_dim, heads, kv heads, page, lengths, group bounds, prefixes
    (128, 32, 8, 64, [4096], None, None),
    (128, 8, 2, 16, [300, 17, 1000, 256], None, None),
    (64, 12, 4, 48, [64, 777, 4000], None, None),
    (128, 32, 8, 16, [20 + 3 * i for i in range(130)], None, None),  # a wave each
    (64, 24, 8, 16, [20 + 3 * i for i in range(130)], None, None),
    (128, 8, 1, 32, [3000 + i for i in range(40)], [0, 40], [2990]),
    (64, 6, 2, 48, [400, 100, 1300, 1200, 1250, 60], [1, 2, 5], [50, 1111]),
    (128, 32, 8, 16, [130 + i for i in range(131)], [0, 131], [120]),  # a wave each beside a prefix
    (128, 128, 16, 16, [153 + i % 40 for i in range(300)], [0, 300], [150]),  # a prefix on 128 rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("std,margin", [(1.5, 0), (3.0, 8)])
@pytest.mark.parametrize("hd,heads,kv,ps,lens,bounds,prefixes", SINGLE)
def test_single_tokens(ane, hd, heads, kv, ps, lens, bounds, prefixes, std, margin):
    import torch

    c = make_cache(lens, heads, kv, hd, ps, seed=12)
    kw = {}
    if bounds:
        share(c, bounds, prefixes)
        kw = dict(group_start=i32(bounds), prefix_len=i32(prefixes), max_prefix=max(prefixes))
    q = randq(len(lens), heads, hd, torch.float32, std=std)
    out = torch.zeros_like(q)
    ane.attention_shared(c, 0, q, out, max_len=max(lens), **kw)
    for s in sorted({0, 1, len(lens) // 2, len(lens) - 1} & set(range(len(lens)))):
        check_heads(c, 0, s, q[s:s + 1], out[s:s + 1], [lens[s]], margin)


# ------------------------------------------------------------------ one key far above the others
def with_sink(c, s, at, margin, value=0.0):
    """Position `at` of sequence s scores `margin` above the mean of the others, for
    queries whose dimension 0 is 4, and its value is made `value` times as large."""
    n, ps = int(c.kv_len[s]), c.page_size
    for j in range(-(-n // ps)):
        c.k_pages[:, int(c.page_table[s, j]), :, :min(ps, n - j * ps), 0] = 0
    page, row = int(c.page_table[s, at // ps]), at % ps
    c.k_pages[:, page, :, row] = 0
    c.k_pages[:, page, :, row, 0] = margin * c.head_dim ** 0.5 / 4
    c.v_pages[:, page, :, row] *= value


SINKS = [
    # head_dim, heads, kv heads, new tokens, cached positions
    (128, 8, 2, 4, 16), (64, 8, 2, 3, 30), (128, 4, 1, 30, 700), (64, 4, 1, 9, 5000), (128, 32, 8, 1, 4095),
    (128, 32, 8, 1100, 70), (64, 32, 8, 2100, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("margin", [12, 14, 16, 18, 20, 22, 30])
@pytest.mark.parametrize("hd,heads,kv,new,old", SINKS)
def test_one_key_far_above_the_others(ane, hd, heads, kv, new, old, margin):
    """The weights that carry the result are e^-margin of the largest, whose value is
    zeros; the large key is the first, one in the middle or the last that every row
    sees."""
    import torch

    for at in sorted({0, old // 2, old}):
        c = make_cache([old + new], heads, kv, hd, 16, seed=13 + at)
        with_sink(c, 0, at, margin)
        q = randq(new, heads, hd, torch.float32, seed=at, std=1.0)
        q[:, :, 0] = 4.0
        out = torch.zeros_like(q)
        ane.attention_prompt(c, 0, i32([0, new]), q, out, max_len=old + new)
        rows = torch.arange(0 if old else 1, new, 1 + new // 50, device="cuda")  # (a row that sees it alone is zeros)
        check_heads(c, 0, 0, q[rows], out[rows], [old + int(t) + 1 for t in rows], margin)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [1e-6, 1e-4, 1e-2])
@pytest.mark.parametrize("margin", [10, 14, 18])
@pytest.mark.parametrize("hd,heads,kv,new,old", [(128, 8, 2, 4, 16), (64, 4, 1, 9, 700), (128, 32, 8, 1100, 0)])
def test_one_key_far_above_the_others_of_a_small_value(ane, hd, heads, kv, new, old, margin, value):
    """Its share of the result is smaller, as large and larger than the others'."""
    import torch

    c = make_cache([old + new], heads, kv, hd, 16, seed=16)
    with_sink(c, 0, 0, margin, value)
    q = randq(new, heads, hd, torch.float32, seed=17, std=1.0)
    q[:, :, 0] = 4.0
    out = torch.zeros_like(q)
    ane.attention_prompt(c, 0, i32([0, new]), q, out, max_len=old + new)
    rows = torch.arange(0 if old else 1, new, 1 + new // 50, device="cuda")
    check_heads(c, 0, 0, q[rows], out[rows], [old + int(t) + 1 for t in rows], margin)


@pytest.mark.gpu
@pytest.mark.parametrize("margin", [14, 18, 22, 30])
@pytest.mark.parametrize("hd,heads,kv,n,prefix", [(128, 8, 2, 9, 300), (64, 8, 2, 5, 2000), (128, 32, 8, 140, 100),
                                                  (128, 128, 16, 300, 150)])
def test_one_key_far_above_the_others_in_a_prefix(ane, hd, heads, kv, n, prefix, margin):
    """The large key at the start of a shared prefix, as a model's first token often
    is: the prefix's sums and each row's own are joined."""
    import torch

    c = make_cache([prefix + 20 + i % 30 for i in range(n)], heads, kv, hd, 16, seed=14)
    share(c, [0, n], [prefix])
    for s in range(n):
        with_sink(c, s, 0, margin)
    q = randq(n, heads, hd, torch.float32, seed=15, std=1.0)
    q[:, :, 0] = 4.0
    out = torch.zeros_like(q)
    ane.attention_shared(c, 0, q, out, group_start=i32([0, n]), prefix_len=i32([prefix]), max_len=prefix + 50,
                         max_prefix=prefix)
    for s in (0, n // 2, n - 1):
        check_heads(c, 0, s, q[s:s + 1], out[s:s + 1], [prefix + 20 + s % 30], margin)
