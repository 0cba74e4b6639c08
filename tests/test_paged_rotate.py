"""RMSNorm of q and k heads, rotation and append in one pass (include/ane_decode.h;
ane_amd/csrc/paged_rotate.hip), element by element against the formula in 64 bits.

The bound, u = 2^-24: a sum of 8 squares in a lane and four additions across
lanes, all terms positive, is off by at most 12 u of itself; mean + eps, square
root and reciprocal bring the factor to 6 + 1/2 + 1 + 1 < 9 u, times value and
weight 11 u.  Cosine and sine are rounded once (the series leaves 1e-16), each
product and the sum once more: 14 u (|a| + |b|) |factor| < 16 u.  fp16 results
round by 2^-11 of themselves, at least 2^-25.  Without norm and rotation nothing
but that last rounding happens.
"""
import ctypes
import math
import shutil
import subprocess

import numpy as np
import pytest

import ane_amd
from ane_amd import AneError, PagedCache, Rope
from tests.test_paged import P, ROOT, dt, i32, make_cache, randq, raw_cache

U = 2.0 ** -24


# ------------------------------------------------------------------ CPU
def test_struct_layout_matches_c(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    src = tmp_path / "layout.c"
    names = ("rot_dim", "halves", "freqs", "factor")
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ane_decode.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu ", offsetof(struct ane_rope, {n}));\n' for n in names)
                   + 'printf("%zu\\n", sizeof(struct ane_rope)); return 0; }\n')
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(Rope, n).offset for n, _ in Rope._fields_] + [ctypes.sizeof(Rope)]


def raw_rope(rot=128, halves=1, freqs=P, factor=1.0):
    r = Rope.__new__(Rope)
    ctypes.Structure.__init__(r, rot, halves, freqs, factor)
    return r


def call(c=None, layer=0, n=2, qs=P, T=4, it=0, q=P, qstr=1024, k=P, v=P, kvstr=256, rope=None, qn=None, kn=None, eps=1e-6,
         qt=0, qo=P, qostr=1024):
    c = raw_cache() if c is None else c
    return ane_amd.lib().ane_hip_paged_norm_rope_append(
        ctypes.byref(c), layer, None, n, qs, T, it, q, qstr, k, v, kvstr, ctypes.byref(rope) if rope else None, qn, kn, eps, qt,
        qo, qostr, None)


INVALID, POINTER = 1, 2


@pytest.mark.parametrize("kw,st", [
    (dict(c=raw_cache(head_dim=96)), INVALID), (dict(layer=2), INVALID), (dict(T=(1 << 23) + 1), INVALID), (dict(it=2), INVALID),
    (dict(qt=2), INVALID), (dict(qs=None, T=3), INVALID), (dict(rope=raw_rope(rot=24)), INVALID),
    (dict(rope=raw_rope(rot=144)), INVALID), (dict(rope=raw_rope(factor=0.0)), INVALID),
    (dict(rope=raw_rope(factor=math.nan)), INVALID), (dict(rope=raw_rope(factor=math.inf)), INVALID),
    (dict(rope=raw_rope(freqs=None)), POINTER), (dict(rope=raw_rope(freqs=P + 4)), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=math.nan), INVALID), (dict(k=None), POINTER), (dict(v=None), POINTER), (dict(q=None), POINTER),
    (dict(qo=None), POINTER), (dict(q=P + 8), INVALID), (dict(qn=P + 2), INVALID), (dict(kn=P + 1), INVALID),
    (dict(qs=P + 2), INVALID), (dict(qstr=1020), INVALID), (dict(qstr=1026), INVALID), (dict(qostr=1022), INVALID),
    (dict(kvstr=252), INVALID), (dict(kvstr=258), INVALID), (dict(n=0), 0), (dict(T=0), 0)])
def test_refusals(kw, st):
    assert call(**kw) == st


def test_rope_wrapper_refuses_wrong_tensors():
    import torch

    for f in (torch.zeros(8), torch.zeros((2, 8), dtype=torch.float64), torch.zeros(16, dtype=torch.float64)[::2]):
        with pytest.raises(ValueError):
            Rope(f)


@pytest.mark.parametrize("rot,base", [(128, 500000.0), (32, 10000.0), (16, 1e6)])
def test_frequencies(rot, base):
    i = np.arange(rot // 2)
    plain = base ** (-2.0 * i / rot)

    def close(a, b):
        assert np.allclose(a, b, rtol=1e-13, atol=0)

    f, m = ane_amd.rope_freqs(rot, base)
    close(f, plain)
    assert m == 1.0
    close(ane_amd.rope_freqs(rot, base, 8.0, "linear")[0], plain / 8)
    f = ane_amd.rope_freqs(rot, base, 8.0, "base")[0]
    close(f[[0, -1]], [1.0, plain[-1] / 8])
    assert (np.diff(f) < 0).all()
    f, m = ane_amd.rope_freqs(rot, base, 8.0, "turns", context=8192, low=1, high=4)
    turns = 8192 * plain / (2 * math.pi)
    close(f[turns >= 4], plain[turns >= 4])
    close(f[turns <= 1], plain[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 4)
    t = (turns[mid] - 1) / 3
    close(f[mid], (1 - t) * plain[mid] / 8 + t * plain[mid])
    assert m == 1.0
    f, m = ane_amd.rope_freqs(rot, base, 8.0, "index", context=4096, low=1, high=32)
    assert m == 0.1 * math.log(8.0) + 1
    turns = 4096 * plain / (2 * math.pi)
    close(f[0], plain[0])
    assert (f <= plain * (1 + 1e-13)).all() and (f >= plain / 8 * (1 - 1e-13)).all()
    close(f[turns < 1][2:], plain[turns < 1][2:] / 8)  # the border is rounded outwards, by less than two pairs
    for bad in (dict(rot_dim=7), dict(factor=0.0), dict(scaling="x"), dict(scaling="turns", low=4, high=1), dict(base=0.0)):
        with pytest.raises(ValueError):
            ane_amd.rope_freqs(**{**dict(rot_dim=rot, base=base), **bad})


# ------------------------------------------------------------------ the formula
def want(x, pos, freqs, factor, halves, w, eps, out):
    """(result, bound) in 64 bits for x [tokens][heads][hd] (numpy, as given) at positions pos."""
    y = x.astype(np.float64)
    hd = y.shape[-1]
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(eps))) * w.astype(np.float64)
        tol = np.abs(y) * 11 * U
    else:
        tol = np.zeros_like(y)
    rot = 0 if freqs is None else 2 * len(freqs)
    if rot:
        a, b = (np.arange(rot // 2), np.arange(rot // 2, rot)) if halves else (np.arange(0, rot, 2), np.arange(1, rot, 2))
        ang = pos.astype(np.float64)[:, None] * freqs
        c, s = (np.cos(ang) * factor)[:, None], (np.sin(ang) * factor)[:, None]
        z, t = y.copy(), tol.copy()
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
        t[..., a] = t[..., b] = 16 * U * factor * (np.abs(y[..., a]) + np.abs(y[..., b]))
        y, tol = z, t
    if out == "f16":
        tol = tol + np.abs(y) * 2.0 ** -11 * (1 + 2.0 ** -10) + 2.0 ** -25
    z = pos < 0
    y[z], tol[z] = 0.0, 0.0
    return y, tol


def near(got, w, what):
    y, tol = w
    err = np.abs(got.astype(np.float64) - y)
    assert (err <= tol).all(), (what, float((err - tol).max()), float(err.max()))


def run(c, new, old, ty, qt, rot, halves, qn, kn, factor=1.0, layer=0, seqs=None, in_place=False, behind=2, base=10000.0, **kw):
    """One call on cache c, checked whole: q rows, the pages' new rows, everything else as it was."""
    import torch

    heads, kv, hd, ps = c.n_heads, c.n_kv_heads, c.head_dim, c.page_size
    T = sum(new)
    qkv = torch.cat([randq(T + behind, heads + 2 * kv, hd, dt(ty), seed=3 + T),
                     torch.zeros(T + behind, 1, hd, dtype=dt(ty), device="cuda")], 1)  # a stride past the heads
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:heads + 2 * kv]
    gen = torch.Generator(device="cuda").manual_seed(9)
    qw, kw_ = (torch.randn(hd, generator=gen, device="cuda") * 0.3 + 1 if u else None for u in (qn, kn))
    f = ane_amd.rope_freqs(rot, base)[0] if rot else None
    rope = Rope(torch.from_numpy(f).cuda(), half=halves, factor=factor) if rot else None
    out = q if in_place else torch.full((T + behind, heads, hd), 5.0, dtype=dt(qt), device="cuda")
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    qf, kf, vf, keep = (x.cpu().numpy().copy() for x in (q, k, v, out))
    kb, vb = c.k_pages.clone(), c.v_pages.clone()
    ane_amd.paged_norm_rope_append(c, layer, i32(start), q, k, v, rope, out, q_norm=qw, k_norm=kw_, eps=1e-6,
                                   seqs=None if seqs is None else i32(seqs), **kw)
    torch.cuda.synchronize()
    pos = np.concatenate([np.arange(m, m + n) for n, m in zip(new, old)] + [np.zeros(0, int)]).astype(np.int64)
    qw, kw_ = (None if x is None else x.cpu().numpy() for x in (qw, kw_))
    got = out.cpu().numpy()
    near(got[:T], want(qf[:T], pos, f, factor, halves, qw, 1e-6, qt), "q")
    assert np.array_equal(got[T:], keep[T:])
    table = c.page_table.cpu().numpy()
    s = np.concatenate([np.full(n, i if seqs is None else seqs[i]) for i, n in enumerate(new)] + [np.zeros(0, int)]).astype(int)
    live = pos >= 0
    page = torch.from_numpy(table[s[live], pos[live] // ps].astype(np.int64)).cuda()
    row = torch.from_numpy(pos[live] % ps).cuda()
    gk, gv = (x[layer, page, :, row].cpu().numpy() for x in (c.k_pages, c.v_pages))
    y, tol = want(kf[:T], pos, f, factor, halves, kw_, 1e-6, "f16")
    near(gk, (y[live], tol[live]), "k")
    assert np.array_equal(gv, vf[:T][live].astype(np.float16))
    for x, b in ((c.k_pages, kb), (c.v_pages, vb)):  # nothing else is written
        b[layer, page, :, row] = x[layer, page, :, row]
        assert torch.equal(x.view(torch.int16), b.view(torch.int16))


# ------------------------------------------------------------------ GPU
CASES = [
    # type, q_out, hd, heads, kv, ps, new, old, rot, halves, q norm, k norm, factor
    ("f32", "f32", 128, 32, 8, 16, [1] * 9, [0, 15, 16, 17, 100, 3, 31, 32, 63], 128, True, True, True, 1.0),
    ("f32", "f16", 128, 8, 2, 48, [33, 1, 0, 70], [0, 47, 5, 11], 128, True, True, True, 1.0),
    ("f16", "f32", 64, 3, 1, 16, [5, 129, 2], [40, 0, 1], 64, True, True, True, 1.2),
    ("f16", "f16", 64, 40, 4, 64, [64, 65], [0, 63], 32, True, True, False, 1.0),
    ("f32", "f32", 128, 64, 64, 16, [3], [14], 128, False, False, True, 1.0),
    ("f32", "f32", 128, 5, 5, 16, [7, 2], [1, 2], 64, False, True, True, 0.7),
    ("f16", "f16", 64, 12, 4, 48, [50], [60], 16, False, False, False, 1.2),
    ("f16", "f32", 128, 4, 4, 32, [50], [0], 16, True, False, False, 1.0),
    ("f32", "f16", 64, 7, 1, 16, [9, 9], [3, 30], 48, True, True, True, 1.0),
    ("f32", "f32", 128, 2, 1, 16, [20], [0], 112, True, False, True, 1.0),
    ("f32", "f32", 64, 2, 2, 16, [20, 1], [0, 0], 0, False, True, True, 1.0),
    ("f16", "f16", 128, 128, 1, 16, [4], [0], 0, False, False, False, 1.0),
    ("f32", "f32", 64, 128, 128, 16, [3], [100], 64, True, True, True, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("ty,qt,hd,heads,kv,ps,new,old,rot,halves,qn,kn,factor", CASES)
def test_rotate(ane, ty, qt, hd, heads, kv, ps, new, old, rot, halves, qn, kn, factor):
    c = make_cache([a + b for a, b in zip(new, old)], heads, kv, hd, ps, fill_rest=7.0, layers=2)
    run(c, new, old, ty, qt, rot, halves, qn, kn, factor, layer=1)


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("ty", ["f32", "f16"])
def test_in_place_and_chosen_sequences(ane, ty, halves):
    c = make_cache([50, 7, 33, 90], 8, 2, 128, 16, fill_rest=7.0)
    run(c, [3, 20, 1], [87, 30, 6], ty, ty, 96, halves, True, True, seqs=[3, 0, 1], in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
def test_far_positions(ane, halves):
    """Positions up to the last that a cache can have, 2^30 - 1: angles of 1e9 radians."""
    import torch

    ps = 1 << 20
    k, v = (torch.zeros((1, 3, 1, ps, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.full((2, 1024), -1, dtype=torch.int32, device="cuda")
    table[0, 1022], table[0, 1023], table[1, 700] = 2, 0, 1
    c = PagedCache(4, k, v, table, i32([1 << 30, 700 * ps + 12345]))
    run(c, [ps // 65536 + 5, 9], [(1 << 30) - 21, 700 * ps + 12336], "f32", "f32", 64, halves, False, False, base=500000.0)


@pytest.mark.gpu
def test_what_has_no_place(ane):
    """Negative positions, broken pages, unknown sequences; k and v alone; single tokens without starts."""
    import torch

    c = make_cache([40, 40, 2], 4, 2, 64, 16, fill_rest=7.0)
    c.page_table[1, 2] = c.n_pages  # position 32.. of sequence 1
    before = c.k_pages.clone(), c.v_pages.clone()
    q, k, v = randq(10, 4, 64, dt("f32")), randq(10, 2, 64, dt("f32"), 2), randq(10, 2, 64, dt("f32"), 3)
    out = torch.full_like(q, 5.0)
    rope = Rope(torch.from_numpy(ane.rope_freqs(64)[0]).cuda(), half=True)
    ones = torch.ones(64, device="cuda")
    ane.paged_norm_rope_append(c, 0, i32([0, 3, 8, 10]), q, k, v, rope, out, q_norm=ones, k_norm=ones, seqs=i32([1, 2, 77]))
    row = int(c.page_table[2, 0])
    for x, b in zip((c.k_pages, c.v_pages), before):
        same = x == b
        same[0, row, :, :2] = True
        assert bool(same.all())
    assert bool((c.v_pages[0, row, :, :2] == v[6:8].half().transpose(0, 1)).all())
    assert not out[3:6].any() and not out[8:].any() and out[:3].abs().sum() > 0 and out[6:8].abs().sum() > 0
    c2 = make_cache([5, 17], 4, 2, 64, 16)
    ane.paged_norm_rope_append(c2, 0, None, None, k[:2], v[:2], None, None)
    for s, p in ((0, 4), (1, 16)):
        page = int(c2.page_table[s, p // 16])
        assert bool((c2.k_pages[0, page, :, p % 16] == k[s].half()).all())
    with pytest.raises(ValueError):
        ane.paged_norm_rope_append(c2, 0, None, q[:2], k[:2], v[:2], rope, None)
    with pytest.raises(ValueError):
        ane.paged_norm_rope_append(c2, 0, None, q[:2], k[:2], v[:2], rope, out, q_norm=torch.ones(63, device="cuda"))
    with pytest.raises(ValueError, match="device"):
        ane.paged_norm_rope_append(c2, 0, None, q[:2], k[:2], v[:2], Rope(torch.zeros(16, dtype=torch.float64)), out)
    with pytest.raises(AneError):
        ane.paged_norm_rope_append(c2, 0, None, q[:2], k[:2], v[:2], Rope(torch.zeros(36, dtype=torch.float64, device="cuda")), out)


@pytest.mark.gpu
def test_same_as_the_table_where_both_apply(ane):
    """Adjacent pairs of whole heads without a norm: the bits of paged_rope_append with a table of the same angles."""
    import torch

    lens = [70, 3, 200]
    a, b = (make_cache(lens, 8, 2, 128, 16, fill_rest=0.0) for _ in range(2))
    qkv = randq(100, 12, 128, dt("f32"))
    start = i32([0, 60, 63, 100])
    oa, ob = (torch.zeros((100, 8, 128), device="cuda") for _ in range(2))
    ane.paged_rope_append(a, 0, start, qkv[:, :8], qkv[:, 8:10], qkv[:, 10:],
                          torch.from_numpy(ane.rope_table(200, 128, 500000.0)).cuda(), oa)
    rope = Rope(torch.from_numpy(ane.rope_freqs(128, 500000.0)[0]).cuda())
    ane.paged_norm_rope_append(b, 0, start, qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], rope, ob)
    assert torch.equal(oa, ob) and torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)


@pytest.mark.gpu
def test_captured_and_on_another_stream(ane):
    """A captured call follows the lengths and tables of each replay, eager work between them; then a stream of its own."""
    import torch

    c, d = (make_cache([100, 60], 8, 4, 64, 16, fill_rest=0.0) for _ in range(2))
    qkv = randq(12, 16, 64, dt("f16"))
    q, k, v = qkv[:, :8], qkv[:, 8:12], qkv[:, 12:]
    start = i32([0, 5, 12])
    rope = Rope(torch.from_numpy(ane.rope_freqs(32)[0]).cuda(), half=True, factor=1.1)
    w = torch.rand(64, device="cuda") + 0.5
    o, e = torch.zeros((12, 8, 64), device="cuda"), torch.zeros((12, 8, 64), device="cuda")
    ane.paged_norm_rope_append(c, 0, start, q, k, v, rope, o, q_norm=w, k_norm=w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ane.paged_norm_rope_append(c, 0, start, q, k, v, rope, o, q_norm=w, k_norm=w)
    for i in range(3):
        for x in (c, d):
            x.kv_len.copy_(i32([90 - 7 * i, 50 + i]))
        qkv.mul_(-1.5)
        o.zero_()
        g.replay()
        ane.paged_norm_rope_append(d, 0, start, q, k, v, rope, e, q_norm=w, k_norm=w)
        torch.cuda.synchronize()
        assert torch.equal(o, e) and bool(o.any())
    d.k_pages.copy_(c.k_pages), d.v_pages.copy_(c.v_pages)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    ane.paged_norm_rope_append(c, 0, start, k=k, v=v, q=q, rope=rope, q_out=o, q_norm=w, k_norm=w, stream=st)
    st.synchronize()
    ane.paged_norm_rope_append(d, 0, start, q, k, v, rope, e, q_norm=w, k_norm=w)
    assert torch.equal(o, e) and torch.equal(c.k_pages, d.k_pages) and torch.equal(c.v_pages, d.v_pages)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 65, 1000, 4097])
def test_wide_batch(ane, n):
    r = np.random.default_rng(n)
    new = [int(x) for x in r.integers(0, 4, n)]
    new[-1] = 1
    old = [int(x) for x in r.integers(0, 30, n)]
    c = make_cache([max(a + b, 1) for a, b in zip(new, old)], 4, 2, 64, 16, fill_rest=7.0)
    old = [max(a + b, 1) - a for a, b in zip(new, old)]
    run(c, new, old, "f16", "f16", 64, True, True, True)


@pytest.mark.gpu
def test_special_values(ane):
    """Infinities and NaN stay in their own heads; zeros with eps stay zeros; tiny and large heads are normalised."""
    import torch

    c = make_cache([6], 3, 3, 128, 16, fill_rest=0.0)
    q = randq(6, 3, 128, dt("f32"))
    q[0, 1, 5], q[1, 2, 127] = math.inf, math.nan
    q[2] = 0
    q[3, 0] *= 1e-3
    q[3, 1] *= 1e15
    out = torch.zeros_like(q)
    rope = Rope(torch.from_numpy(ane.rope_freqs(128)[0]).cuda(), half=True)
    one = torch.ones(128, device="cuda")
    ane.paged_norm_rope_append(c, 0, i32([0, 6]), q, q, q, rope, out, q_norm=one, k_norm=one)
    o = out.cpu().numpy()
    bad = ~np.isfinite(o).all(-1)
    assert bad[0, 1] and bad[1, 2] and bad.sum() == 2 and not o[2].any()
    pos = np.arange(6)
    f = ane.rope_freqs(128)[0]
    y, tol = want(q.cpu().numpy()[3:], pos[3:], f, 1.0, True, np.ones(128, np.float32), 1e-6, "f32")
    near(o[3:], (y, tol), "q")


@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,kv", [(128, 3, 3), (64, 4, 2)])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_heads_at_the_ends_of_the_range(ane, hd, heads, kv, eps):
    """Heads whose squares leave fp32's range, upwards and downwards: normalised like any other.  (A head of denormals
    beside an eps stays one: six roundings of 2^-150 each on the way, weights and rotation at most double them: below 2^-146.)"""
    import torch

    powers = [2.0 ** e for e in (66, 80, 100, 120, -66, -76, -100, -126, -140)]
    n = len(powers)
    c = make_cache([n], heads, kv, hd, 16, fill_rest=0.0)
    qkv = randq(n, heads + 2 * kv, hd, dt("f32"), seed=21) * torch.tensor(powers, device="cuda")[:, None, None]
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    gen = torch.Generator(device="cuda").manual_seed(9)
    qw, kw = (torch.randn(hd, generator=gen, device="cuda") * 0.3 + 1 for _ in range(2))
    out = torch.full((n, heads, hd), 5.0, device="cuda")
    f = ane.rope_freqs(hd)[0]
    ane.paged_norm_rope_append(c, 0, i32([0, n]), q, k, v, Rope(torch.from_numpy(f).cuda(), half=True), out, q_norm=qw, k_norm=kw,
                               eps=eps)
    pos = np.arange(n)
    y, tol = want(q.cpu().numpy(), pos, f, 1.0, True, qw.cpu().numpy(), eps, "f32")
    near(out.cpu().numpy(), (y, tol + 2.0 ** -146), "q")
    page = int(c.page_table[0, 0])
    near(c.k_pages[0, page, :, :n].transpose(0, 1).cpu().numpy(),
         want(k.cpu().numpy(), pos, f, 1.0, True, kw.cpu().numpy(), eps, "f16"), "k")
