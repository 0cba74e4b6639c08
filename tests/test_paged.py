"""The paged K/V cache and the attention over it (include/ane_decode.h;
ane_amd/csrc/paged.hip, paged_attention.hip).

The append and the page calls are compared bit for bit, the page calls with a
model of the cache in plain Python.  Attention is compared element by element
with its formula in 64 bits, within `bound` below: the worst case of the
roundings, written out there.
"""
import ctypes
import math
import random
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import ane_amd
from ane_amd import AneError, NO_PAGE, PagedCache

ROOT = Path(__file__).resolve().parents[1]
FIELDS = ("n_layers", "n_heads", "n_kv_heads", "head_dim", "page_size", "n_pages", "n_seqs", "max_pages")


# ------------------------------------------------------------------ CPU
def test_struct_layout_matches_c(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    src = tmp_path / "layout.c"
    names = FIELDS + ("k_pages", "v_pages", "page_table", "kv_len", "page_refs")
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ane_decode.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu ", offsetof(struct ane_paged_cache, {n}));\n' for n in names)
                   + 'printf("%zu\\n", sizeof(struct ane_paged_cache)); return 0; }\n')
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(PagedCache, n).offset for n, _ in PagedCache._fields_] + [ctypes.sizeof(PagedCache)]
    assert got == want


P = 0x10000  # an address no refused call touches


def raw_cache(**kw):
    c = PagedCache.__new__(PagedCache)
    v = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, page_size=16, n_pages=64, n_seqs=4, max_pages=8,
             k_ptr=P, v_ptr=P, table_ptr=P, len_ptr=P, refs_ptr=P)
    v.update(kw)
    ctypes.Structure.__init__(c, *v.values())
    return c


def c_append(c, layer=0, n=2, qs=P, T=4, it=0, q=P, qstr=1024, k=P, v=P, kvstr=256, rope=P, rl=100, qt=0, qo=P, qostr=1024):
    return ane_amd.lib().ane_hip_paged_rope_append(ctypes.byref(c) if c else None, layer, None, n, qs, T, it, q, qstr,
                                                   k, v, kvstr, rope, rl, qt, qo, qostr, None)


def c_prompt(c, layer=0, n=2, qs=P, T=4, ml=0, ty=0, q=P, qstr=1024, scale=0.1, out=P, ostr=1024, ws=0x10000, wsb=1 << 40):
    return ane_amd.lib().ane_hip_attention_prompt(ctypes.byref(c) if c else None, layer, None, n, qs, T, ml, ty, q, qstr,
                                                  scale, out, ostr, ws, wsb, None)


def c_shared(c, layer=0, n=4, ng=1, gs=P, pl=P, mp=0, ml=0, ty=0, q=P, qstr=1024, scale=0.1, out=P, ostr=1024,
             ws=0x10000, wsb=1 << 40):
    return ane_amd.lib().ane_hip_attention_shared(ctypes.byref(c) if c else None, layer, None, n, ng, gs, pl, mp, ml, ty,
                                                  q, qstr, scale, out, ostr, ws, wsb, None)


BAD_CACHES = [dict(n_layers=0), dict(n_heads=0), dict(n_heads=9), dict(n_heads=2 * 129), dict(n_kv_heads=0),
              dict(head_dim=96), dict(head_dim=0), dict(page_size=0), dict(page_size=24), dict(page_size=(1 << 20) + 16),
              dict(n_pages=0), dict(n_pages=1 << 31), dict(n_seqs=0), dict(max_pages=0), dict(max_pages=1 << 27),
              dict(k_ptr=P + 8), dict(v_ptr=P + 2)]


@pytest.mark.parametrize("kw", BAD_CACHES, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
def test_every_call_refuses_a_bad_cache(kw):
    """The description is checked before anything is launched (the addresses
    are never touched: no GPU is needed)."""
    L, c = ane_amd.lib(), raw_cache(**kw)
    b = ctypes.byref(c)
    assert c_append(c) == 1 and c_prompt(c) == 1 and c_shared(c) == 1
    assert L.ane_hip_pages_reserve(b, 1, P, P, None, P, 1 << 40, None) == 1
    assert L.ane_hip_pages_fork(b, 1, P, P, None, P, 1 << 40, None) == 1
    assert L.ane_hip_pages_free(b, 1, P, None) == 1
    assert L.ane_hip_pages_copy(b, 1, P, P, None) == 1
    assert L.ane_hip_pages_compact(b, None, None, None, P, 1 << 40, None) == 1
    assert L.ane_hip_pages_workspace_size(b) == 0
    assert L.ane_hip_attention_prompt_workspace_size(b, 2, 4, 0) == 0
    assert L.ane_hip_attention_shared_workspace_size(b, 2, 0, 0, 0) == 0


@pytest.mark.parametrize("kw", [dict(table_ptr=P + 2), dict(len_ptr=P + 1), dict(refs_ptr=P + 2),
                                dict(max_pages=(1 << 26) + 1)], ids=["table", "lengths", "counts", "positions"])
def test_misaligned_arrays_and_too_many_positions_are_refused(kw):
    """Counts and lengths are changed by atomics, which need whole words; keys
    are numbered in 31 bits with room for the tiles past the last."""
    test_every_call_refuses_a_bad_cache(kw)
    assert ane_amd.lib().ane_hip_pages_workspace_size(ctypes.byref(raw_cache(max_pages=1 << 26))) > 0


@pytest.mark.parametrize("ptr", ["k_ptr", "v_ptr", "table_ptr", "len_ptr"])
def test_missing_cache_arrays_are_refused(ptr):
    c = raw_cache(**{ptr: 0})
    assert c_append(c) == 2 and c_prompt(c) == 2 and c_shared(c) == 2
    assert c_append(None) == 2 and c_prompt(None) == 2 and c_shared(None) == 2
    assert ane_amd.lib().ane_hip_pages_free(ctypes.byref(raw_cache(refs_ptr=0)), 1, P, None) == 2


def test_argument_refusals():
    L, c = ane_amd.lib(), raw_cache()
    b = ctypes.byref(c)
    for kw, want in [(dict(layer=2), 1), (dict(T=(1 << 23) + 1), 1), (dict(it=2), 1), (dict(qt=-1), 1), (dict(qs=None), 1),
                     (dict(rl=0), 1), (dict(k=None), 2), (dict(v=None), 2), (dict(q=None), 2), (dict(qo=None), 2),
                     (dict(q=P + 4), 1), (dict(k=P + 8), 1), (dict(v=P + 2), 1), (dict(qo=P + 4), 1), (dict(rope=P + 4), 1),
                     (dict(kvstr=252), 1), (dict(kvstr=258), 1), (dict(qstr=1026), 1), (dict(qstr=1020), 1),
                     (dict(qostr=1020), 1), (dict(it=1, kvstr=260), 1), (dict(n=0), 0), (dict(T=0), 0)]:
        assert c_append(c, **kw) == want, kw
    for call in (c_prompt, c_shared):
        for kw, want in [(dict(layer=2), 1), (dict(ty=2), 1), (dict(scale=0.0), 1), (dict(scale=-0.1), 1),
                         (dict(scale=math.inf), 1), (dict(scale=math.nan), 1), (dict(scale=2e30), 1), (dict(q=None), 2), (dict(out=None), 2),
                         (dict(q=P + 8), 1), (dict(out=P + 8), 1), (dict(qstr=1022), 1), (dict(qstr=1020), 1),
                         (dict(ostr=1020), 1), (dict(ostr=1026), 1), (dict(n=0), 0)]:
            assert call(c, **kw) == want, (call.__name__, kw)
    assert c_prompt(c, qs=None) == 1 and c_prompt(c, T=0) == 0 and c_prompt(c, T=(1 << 23) + 1) == 1
    assert c_shared(c, ng=5) == 1 and c_shared(c, gs=None) == 2 and c_shared(c, pl=None) == 2
    for f in (lambda n, x, y, ws, wsb: L.ane_hip_pages_reserve(b, n, x, y, None, ws, wsb, None),
              lambda n, x, y, ws, wsb: L.ane_hip_pages_fork(b, n, x, y, None, ws, wsb, None)):
        assert f(65537, P, P, P, 1 << 40) == 1 and f(1, None, P, P, 1 << 40) == 2 and f(1, P, None, P, 1 << 40) == 2
        need = L.ane_hip_pages_workspace_size(b)
        assert f(1, P, P, None, 1 << 40) == 8 and f(1, P, P, P + 64, 1 << 40) == 8 and f(1, P, P, P, need - 1) == 8
        assert f(0, None, None, None, 0) == 0
    assert L.ane_hip_pages_free(b, 65537, P, None) == 1 and L.ane_hip_pages_free(b, 1, None, None) == 2
    assert L.ane_hip_pages_copy(b, 65537, P, P, None) == 1 and L.ane_hip_pages_copy(b, 1, P, None, None) == 2
    assert L.ane_hip_pages_copy(b, 0, None, None, None) == 0
    assert L.ane_hip_pages_compact(b, None, None, None, None, 0, None) == 8


def test_attention_workspace_is_checked():
    """Where a call needs a workspace it takes none that is missing, short or
    misaligned."""
    L, c = ane_amd.lib(), raw_cache(max_pages=4096)
    b = ctypes.byref(c)
    for call, need in ((c_prompt, L.ane_hip_attention_prompt_workspace_size(b, 2, 4, 0)),
                       (c_shared, L.ane_hip_attention_shared_workspace_size(b, 4, 1, 0, 0))):
        if need:
            assert call(c, ws=None) == 8 and call(c, ws=P + 64) == 8 and call(c, wsb=need - 1) == 8


def test_wrappers_refuse_wrong_tensors():
    import torch

    k = torch.zeros(1, 4, 2, 16, 64, dtype=torch.float16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        PagedCache(4, k.float(), k, table, lens)
    with pytest.raises(ValueError):
        PagedCache(4, k, k, table.long(), lens)
    with pytest.raises(ValueError):
        PagedCache(4, k, k, table, lens[:2])
    with pytest.raises(ValueError):
        PagedCache(4, k, k[:, :3], table, lens)
    with pytest.raises(ValueError):
        PagedCache(4, k, k, table, lens, torch.zeros(3, dtype=torch.int32))
    c = PagedCache(4, k, k, table, lens, torch.zeros(4, dtype=torch.int32))
    q, qs = torch.zeros(5, 4, 64), torch.tensor([0, 2, 4, 5], dtype=torch.int32)
    for bad in (q[:, :3], q[..., :32], q.double(), q.transpose(1, 2), q[0]):
        with pytest.raises(ValueError):
            ane_amd.attention_prompt(c, 0, qs, bad, bad)
    with pytest.raises(ValueError):
        ane_amd.attention_prompt(c, 0, qs, q, q.half())
    with pytest.raises(ValueError):
        ane_amd.attention_prompt(c, 0, qs.long(), q, q)
    with pytest.raises(ValueError):
        ane_amd.attention_shared(c, 0, q[:3], q[:3], group_start=qs[:2])
    with pytest.raises(ValueError):
        ane_amd.paged_rope_append(c, 0, qs, q, q[:, :2], q[:4, 2:], None, q)
    with pytest.raises(ValueError):
        ane_amd.paged_rope_append(c, 0, qs, q, q[:, :2], q[:, 2:], None, None)
    with pytest.raises(ValueError):
        ane_amd.pages_fork(c, lens, lens[:2])


def test_wrappers_refuse_a_cache_in_host_memory():
    """An address of host memory never reaches a kernel."""
    import torch

    k = torch.zeros(1, 4, 2, 16, 64, dtype=torch.float16)
    ints = [torch.zeros(n, dtype=torch.int32) for n in (3, 4)]
    c = PagedCache(4, k, k, torch.zeros(3, 2, dtype=torch.int32), *ints)
    q, qs = torch.zeros(5, 4, 64), torch.tensor([0, 2, 4, 5], dtype=torch.int32)
    for call in (lambda: ane_amd.attention_prompt(c, 0, qs, q, q), lambda: ane_amd.attention_shared(c, 0, q, q),
                 lambda: ane_amd.paged_rope_append(c, 0, qs, None, q[:, :2], q[:, 2:], None, None),
                 lambda: ane_amd.pages_reserve(c, qs, qs), lambda: ane_amd.pages_fork(c, qs, qs),
                 lambda: ane_amd.pages_free(c, qs), lambda: ane_amd.pages_copy(c, qs, qs),
                 lambda: ane_amd.pages_compact(c)):
        with pytest.raises(ValueError, match="not in GPU memory"):
            call()


# ------------------------------------------------------------------ helpers
def i32(v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_cache(lens, heads, kv, hd, ps, seed=0, layers=1, extra=3, fill_rest=math.nan):
    """Sequences of these lengths on pages in no order; every row that holds no
    position of any sequence is filled with fill_rest."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + extra
    ids = random.Random(seed).sample(range(pages), sum(need))
    wide = max(need + [1])
    rows = [[ids.pop() for _ in range(n)] + [NO_PAGE] * (wide - n) for n in need]
    k, v = (torch.full((layers, pages, kv, ps, hd), fill_rest, dtype=torch.float16, device="cuda") for _ in range(2))
    for row, n in zip(rows, lens):
        for j in range(-(-n // ps)):
            m = min(ps, n - j * ps)
            for x in (k, v):
                x[:, row[j], :, :m] = torch.randn((layers, kv, m, hd), generator=gen, device="cuda").half()
    refs = [0] * pages
    for row in rows:
        for p in row:
            if p != NO_PAGE:
                refs[p] += 1
    return PagedCache(heads, k, v, i32(rows), i32(lens), i32(refs))


def seq_kv(c, layer, s, n):
    """fp64 K and V [kv][n][hd] of the first n positions of sequence s."""
    import torch

    j = torch.arange(n, device="cuda")
    page = c.page_table[s, j // c.page_size].long()
    return [x[layer, page, :, j % c.page_size].double().transpose(0, 1).contiguous() for x in (c.k_pages, c.v_pages)]


def formula(c, layer, s, q, seen, scale):
    """(result, bound) in fp64 for rows q [m][heads][hd] of sequence s, row i
    seeing its first seen[i] positions.

    The bound: the score of a key is a sum of hd products, each rounded at most
    once, plus a few roundings for the scale, so it is off by at most
    (hd + 8) 2^-24 A with A = scale sum |q k|; a weight e^s then by twice that
    relative to the maximum's, and by 16 2^-24 for the exponential, its argument
    (|s| <= A) and the parts it is split into; the sums over n keys by n 2^-24
    each.  With all that relative to the largest value seen:
    (4 (hd + 12) A + 2 n + 64) 2^-24 max|v|.  16-bit activations round weights
    and result too: 2^-11 each, again of at most max|v|, twice for the pair."""
    import torch

    G = c.n_heads // c.n_kv_heads
    n = max([int(x) for x in seen] + [0])
    m = q.shape[0]
    out = torch.zeros((m, c.n_heads, c.head_dim), dtype=torch.float64, device="cuda")
    tol = torch.zeros((m, c.n_heads, 1), dtype=torch.float64, device="cuda")
    if n <= 0:
        return out, tol
    k, v = seq_kv(c, layer, s, n)
    seen = torch.as_tensor([max(0, int(x)) for x in seen], device="cuda")
    dead = torch.arange(n, device="cuda")[None, :] >= seen[:, None]
    for h in range(c.n_heads):
        kk, vv = torch.nan_to_num(k[h // G], nan=0.0, posinf=0.0, neginf=0.0), v[h // G]
        sc = (q[:, h].double() @ kk.t().contiguous() * scale).masked_fill(dead, -math.inf)
        A = (q[:, h].double().abs() @ kk.abs().t().contiguous() * scale).masked_fill(dead, 0.0).amax(1)
        p = torch.exp(sc - sc.amax(1, keepdim=True).clamp(min=-1e300))
        p = torch.nan_to_num(p / p.sum(1, keepdim=True).clamp(min=1e-300)).masked_fill(dead, 0.0)
        vz = torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
        out[:, h] = p @ vz
        vmax = (vz.abs().amax(1)[None, :].masked_fill(dead, 0.0)).amax(1)
        t = (4 * (c.head_dim + 12) * A + 2 * seen + 64) * 2.0 ** -24 * vmax
        if q.dtype == torch.float16:
            t = t + 2 * 2.0 ** -10 * vmax + 2.0 ** -24
        tol[:, h, 0] = t
    return out, tol


def check_rows(c, layer, s, q, got, seen, scale):
    want, tol = formula(c, layer, s, q, seen, scale)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (s, float((err - tol).max()), float(err.max()))


def run_prompt(c, new, q, out, layer=0, seqs=None, **kw):
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    ane_amd.attention_prompt(c, layer, i32(start), q, out, seqs=None if seqs is None else i32(seqs), **kw)
    return start


def check_prompt(c, new, q, out, start, layer=0, seqs=None, scale=None):
    lens = c.kv_len.tolist()
    for i, n in enumerate(new):
        s = i if seqs is None else seqs[i]
        seen = [lens[s] - n + t + 1 for t in range(n)]
        check_rows(c, layer, s, q[start[i]:start[i + 1]], out[start[i]:start[i + 1]], seen, scale or c.head_dim ** -0.5)


def randq(T, heads, hd, dtype, seed=1, std=1.5):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((T, heads, hd), generator=gen, device="cuda") * std).to(dtype)


def dt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16}[name]


# ------------------------------------------------------------------ append
def np_turn(x, cs):
    a, b, c, s = x[..., 0::2], x[..., 1::2], cs[..., 0], cs[..., 1]
    out = np.empty_like(x)
    out[..., 0::2] = (a * c).astype(np.float32) - (b * s).astype(np.float32)
    out[..., 1::2] = (a * s).astype(np.float32) + (b * c).astype(np.float32)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("ty,qt,hd,heads,kv,ps,new,old,rope", [
    ("f32", "f32", 128, 32, 8, 16, [1] * 9, [0, 15, 16, 17, 100, 3, 31, 32, 63], True),
    ("f32", "f16", 128, 8, 2, 48, [33, 1, 0, 70], [0, 47, 5, 11], True),
    ("f16", "f32", 64, 3, 1, 16, [5, 129, 2], [40, 0, 1], True),
    ("f16", "f16", 64, 40, 4, 64, [64, 65], [0, 63], False),
    ("f32", "f32", 128, 64, 64, 16, [3], [14], True)])
def test_append(ane, ty, qt, hd, heads, kv, ps, new, old, rope):
    import torch

    lens = [a + b for a, b in zip(new, old)]
    c = make_cache(lens, heads, kv, hd, ps, fill_rest=7.0, layers=2)
    T, behind = sum(new), 2
    qkv = torch.cat([randq(T + behind, heads + 2 * kv, hd, dt(ty), seed=3),
                     torch.zeros(T + behind, 1, hd, dtype=dt(ty), device="cuda")], 1)  # a stride past the heads
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:heads + 2 * kv]
    table = ane.rope_table(max(lens), hd) if rope else None
    out = torch.full((T + behind, heads, hd), 5.0, dtype=dt(qt), device="cuda")
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    want_k, want_v = c.k_pages.cpu().numpy().copy(), c.v_pages.cpu().numpy().copy()
    rows = c.page_table.cpu().numpy()
    qf, kf, vf = (x.float().cpu().numpy() for x in (q, k, v))
    want_q = np.full((T + behind, heads, hd), 5.0, np.float32)
    for i, n in enumerate(new):
        for t in range(n):
            p, r = old[i] + t, start[i] + t
            cs = table[p][None] if rope else None
            want_q[r] = np_turn(qf[r], cs) if rope else qf[r]
            page = rows[i, p // ps]
            want_k[1, page, :, p % ps] = (np_turn(kf[r], cs) if rope else kf[r]).astype(np.float16)
            want_v[1, page, :, p % ps] = vf[r].astype(np.float16)
    ane.paged_rope_append(c, 1, i32(start), q, k, v, None if table is None else torch.from_numpy(table).cuda(), out)
    assert np.array_equal(out.cpu().numpy(), want_q.astype(np.float32 if qt == "f32" else np.float16))
    assert np.array_equal(c.k_pages.cpu().numpy(), want_k) and np.array_equal(c.v_pages.cpu().numpy(), want_v)


@pytest.mark.gpu
def test_append_leaves_what_has_no_place(ane):
    """Negative positions, positions past the RoPE table, broken pages and
    unknown sequences: nothing is written to the pages, q_out rows are zeros
    where there is no position; k and v alone; a batch of single tokens."""
    import torch

    c = make_cache([40, 40, 2, 300], 4, 2, 64, 16, fill_rest=7.0)
    c.page_table[1, 2] = c.n_pages  # position 32.. of sequence 1
    before = c.k_pages.clone(), c.v_pages.clone()
    q, k, v = randq(12, 4, 64, dt("f32")), randq(12, 2, 64, dt("f32"), 2), randq(12, 2, 64, dt("f32"), 3)
    out = torch.full_like(q, 5.0)
    table = torch.from_numpy(ane.rope_table(100, 64)).cuda()
    # rows: sequence 1's last 3 (broken page), sequence 2's last 5 (2 positions), sequence 3 (past the table), unknown
    ane.paged_rope_append(c, 0, i32([0, 3, 8, 10, 12]), q, k, v, table, out, seqs=i32([1, 2, 3, 77]))
    row = int(c.page_table[2, 0])
    for x, b in zip((c.k_pages, c.v_pages), before):
        same = x == b
        same[0, row, :, :2] = True
        assert bool(same.all())
    assert bool((c.v_pages[0, row, :, :2] == v[6:8].half().transpose(0, 1)).all())
    assert not out[3:6].any() and not out[8:12].any() and out[:3].abs().sum() > 0 and out[6:8].abs().sum() > 0
    c2 = make_cache([5, 17], 4, 2, 64, 16)
    ane.paged_rope_append(c2, 0, None, None, k[:2], v[:2], None, None)
    for s, p in ((0, 4), (1, 16)):
        page = int(c2.page_table[s, p // 16])
        assert bool((c2.k_pages[0, page, :, p % 16] == k[s].half()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("over", [0, 1, 3, 10, 50, 2 ** 31 - 1 - 80])
@pytest.mark.parametrize("rope", [True, False])
def test_append_and_attention_count_an_overlong_length_alike(ane, over, rope):
    """A length past max_pages * page_size counts as that many positions, for
    the append as for the attention: the new tokens are the last of those, and
    each sees itself."""
    import torch

    cap, new = 80, 10
    c = make_cache([cap], 4, 2, 64, 16, fill_rest=0.0)
    qkv = randq(new, 8, 64, dt("f32"), seed=over % 97)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    rot, out = torch.full((new, 4, 64), 5.0, device="cuda"), torch.zeros((new, 4, 64), device="cuda")
    cs = ane.rope_table(cap, 64)
    before = c.k_pages.clone(), c.v_pages.clone()
    c.kv_len[0] = cap + over
    ane.paged_rope_append(c, 0, i32([0, new]), q, k, v, torch.from_numpy(cs).cuda() if rope else None, rot)
    ane.attention_prompt(c, 0, i32([0, new]), rot, out)
    row = c.page_table[0, cap // 16 - 1]
    at = [cap - new + t for t in range(new)]  # within the last page
    turn = (lambda x: np_turn(x.cpu().numpy(), cs[at][:, None])) if rope else lambda x: x.cpu().numpy()
    for x, old, want in ((c.k_pages, before[0], turn(k)), (c.v_pages, before[1], v.cpu().numpy())):
        old[0, row, :, 16 - new:] = torch.from_numpy(want.astype(np.float16)).cuda().transpose(0, 1)
        assert bool((x == old).all())
    assert np.array_equal(rot.cpu().numpy(), turn(q))
    check_rows(c, 0, 0, rot, out, [p + 1 for p in at], 64 ** -0.5)


def wide_batch(n, most, seed):
    """New tokens and cached positions of n sequences, some with none of either."""
    r = random.Random(seed)
    return [r.choice([0, 1, 1, r.randrange(most + 1)]) for _ in range(n)], [r.choice([0, 5, r.randrange(60)]) for _ in range(n)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 65, 130, 1000, 4097])
def test_append_wide_batch(ane, n):
    """More sequences than a wave looks through in one step (64) and in two (4096)."""
    import torch

    new, old = wide_batch(n, 4, n)
    c = make_cache([a + b for a, b in zip(new, old)], 2, 1, 64, 16, seed=n, fill_rest=0.0)
    T, lead, behind = sum(new), 3, 2  # rows before the first sequence and behind the last
    qkv = randq(lead + T + behind, 4, 64, dt("f32"), seed=n)
    q, k, v = qkv[:, :2], qkv[:, 2:3], qkv[:, 3:]
    out = torch.full((lead + T + behind, 2, 64), 5.0, device="cuda")
    start = lead + np.concatenate([[0], np.cumsum(new)])
    cs = ane.rope_table(80, 64)
    seq = np.repeat(np.arange(n), new)
    pos = np.asarray(old)[seq] + np.arange(T) - (start[:-1] - lead)[seq]
    want_k, want_v = c.k_pages.cpu().numpy().copy(), c.v_pages.cpu().numpy().copy()
    page, live = c.page_table.cpu().numpy()[seq, pos // 16], slice(lead, lead + T)
    qf, kf, vf = (x.cpu().numpy() for x in (q, k, v))
    want_k[0, page, 0, pos % 16] = np_turn(kf[live, 0], cs[pos]).astype(np.float16)
    want_v[0, page, 0, pos % 16] = vf[live, 0].astype(np.float16)
    ane.paged_rope_append(c, 0, i32(start.tolist()), q, k, v, torch.from_numpy(cs).cuda(), out)
    got = out.cpu().numpy()
    assert np.array_equal(got[live], np_turn(qf[live], cs[pos][:, None]))
    assert (got[:lead] == 5.0).all() and (got[lead + T:] == 5.0).all()
    assert np.array_equal(c.k_pages.cpu().numpy(), want_k) and np.array_equal(c.v_pages.cpu().numpy(), want_v)


# ------------------------------------------------------------------ prompts
SHAPES = [
    # type, hd, heads, kv, page, new tokens, cached positions
    ("f32", 128, 8, 2, 16, [1], [0]),
    ("f32", 128, 8, 2, 16, [128], [0]),
    ("f32", 128, 4, 1, 64, [33, 1, 0, 200, 65], [0, 700, 40, 3, 0]),
    ("f16", 128, 8, 2, 16, [300, 7], [0, 129]),
    ("f16", 128, 32, 8, 64, [97, 64, 63], [0, 1, 1000]),
    ("f32", 64, 6, 2, 48, [130, 50], [14, 333]),
    ("f16", 64, 12, 4, 48, [777, 301], [333, 2]),
    ("f16", 64, 5, 1, 16, [31, 32, 33], [5, 0, 31]),
    ("f32", 64, 2, 2, 80, [513], [0]),
    ("f16", 128, 16, 1, 112, [40, 9], [0, 300]),
    ("f32", 128, 128, 1, 32, [3, 2], [0, 77]),
    ("f32", 128, 8, 8, 1024, [90], [800]),
    ("f32", 128, 4, 1, 16, [9, 2], [5000, 7001]),
    ("f16", 64, 8, 2, 32, [5], [9000]),
    # enough rows for the kernel of 128 a workgroup (over 1024 a sequence, over 32768 in all)
    ("f32", 128, 32, 8, 16, [1500, 30, 700], [0, 5, 300]),
    ("f16", 128, 32, 8, 64, [2100], [0]),
    ("f32", 64, 32, 8, 48, [1300, 900], [14, 333]),
    ("f16", 64, 40, 8, 32, [1700, 3], [1, 0]),
    ("f16", 128, 36, 12, 16, [1001], [4200]),
    ("f32", 128, 32, 8, 16, [256] * 9, [0, 3, 0, 17, 0, 0, 200, 0, 1]),
    ("f16", 64, 32, 8, 16, [200] * 11, [0, 3, 0, 17, 0, 0, 200, 0, 1, 0, 0]),
    ("f32", 64, 32, 8, 32, [33, 1, 30] * 8, [0, 700, 64] * 8),
    ("f16", 128, 32, 8, 16, [16, 17] * 32, [100, 0] * 32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd,heads,kv,ps,new,old", SHAPES)
def test_prompt(ane, ty, hd, heads, kv, ps, new, old):
    import torch

    c = make_cache([a + b for a, b in zip(new, old)], heads, kv, hd, ps, layers=2, seed=5)
    q = randq(sum(new) + 3, heads, hd, dt(ty))
    out = torch.full_like(q, 5.0)
    start = run_prompt(c, new, q, out, layer=1)
    check_prompt(c, new, q, out, start, layer=1)
    assert bool((out[sum(new):] == 5.0).all())  # rows behind the last sequence


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd,heads,kv,n,most", [
    ("f32", 128, 4, 2, 64, 40), ("f32", 64, 4, 1, 65, 70), ("f16", 128, 8, 2, 130, 40), ("f32", 128, 2, 1, 1000, 9),
    ("f16", 64, 2, 2, 4097, 4), ("f32", 128, 32, 8, 130, 250), ("f16", 64, 40, 8, 200, 300)])  # the last two: 128 rows a workgroup
def test_prompt_wide_batch(ane, ty, hd, heads, kv, n, most):
    """More sequences than a wave looks through in one step (64) and in two (4096),
    empty ones among them, rows before the first and behind the last left as they were."""
    import torch

    new, old = wide_batch(n, most, n)
    new[n // 2], new[-1], old[-1] = most, 3, 0
    c = make_cache([a + b for a, b in zip(new, old)], heads, kv, hd, 16, seed=n)
    T, lead, behind = sum(new), 3, 2
    q = randq(lead + T + behind, heads, hd, dt(ty), seed=n)
    out = torch.full_like(q, 5.0)
    start = [lead]
    for m in new:
        start.append(start[-1] + m)
    ane.attention_prompt(c, 0, i32(start), q, out, max_len=max(a + b for a, b in zip(new, old)))
    assert bool((out[:lead] == 5.0).all()) and bool((out[lead + T:] == 5.0).all()) and not (out[lead:lead + T] == 5.0).all(2).any()
    for i in sorted({0, 1, 31, 32, 62, 63, 64, n // 2, n - 2, n - 1} & set(range(n)) | set(range(0, n, 1 + n // 25))):
        check_rows(c, 0, i, q[start[i]:start[i + 1]], out[start[i]:start[i + 1]], [old[i] + t + 1 for t in range(new[i])],
                   hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "f16"])
def test_prompt_strides_order_scale_and_bound(ane, ty):
    """Views of a wider tensor, sequences in another order (one of them twice),
    a scale of one's own, a length bound below the lengths, in place."""
    import torch

    c = make_cache([300, 77, 500, 64], 8, 2, 128, 16, seed=9)
    new, seqs = [70, 64, 20, 33], [2, 3, 0, 2]
    wide = randq(sum(new), 13, 128, dt(ty))
    q = wide[:, 2:10]
    big = torch.zeros((sum(new), 9, 128), dtype=dt(ty), device="cuda")
    out = big[:, 1:]
    start = run_prompt(c, new, q, out, seqs=seqs, scale=0.03)
    check_prompt(c, new, q, out, start, seqs=seqs, scale=0.03)
    assert not big[:, 0].any()
    run_prompt(c, new, q, big[:, 1:], seqs=seqs, scale=0.03, max_len=16)
    check_prompt(c, new, q, out, start, seqs=seqs, scale=0.03)
    keep = q.clone()
    run_prompt(c, new, q, q, seqs=seqs)
    check_prompt(c, new, keep, q, start, seqs=seqs)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd", [("f32", 128), ("f16", 128), ("f32", 64), ("f16", 64)])
@pytest.mark.parametrize("heads,kv,new,old", [(8, 2, [200], [0]), (8, 2, [40, 90], [300, 10]), (8, 2, [2, 3], [600, 700]),
                                              (32, 8, [1100, 90], [70, 10]), (32, 8, [1040], [0])])
def test_prompt_masked_places_hold_anything(ane, ty, hd, heads, kv, new, old):
    """NaN and infinities in keys and values a row does not see never reach it;
    make_cache fills every unused row of every page with NaN as well."""
    import torch

    lens = [a + b for a, b in zip(new, old)]
    c = make_cache(lens, heads, kv, hd, 16, seed=3)
    for s, (n, bad) in enumerate(zip(lens, (math.nan, -math.inf))):
        for j, val in ((n - 1, bad), (n - 2, math.inf)):  # seen by the last tokens only
            page = int(c.page_table[s, j // 16])
            c.v_pages[0, page, 0, j % 16, 3:40] = val
            c.k_pages[0, page, 1, j % 16, 5] = val
    q = randq(sum(new), heads, hd, dt(ty))
    out = torch.zeros_like(q)
    start = run_prompt(c, new, q, out)
    for i, n in enumerate(new):
        m = max(0, n - 2)
        a = start[i]
        check_rows(c, 0, i, q[a:a + m], out[a:a + m], [old[i] + t + 1 for t in range(m)], hd ** -0.5)
        last = out[a + n - 1].float()
        assert not torch.isfinite(last[:4, 3:40]).any()  # kv head 0: the values are seen
        assert bool(torch.isfinite(last[:4, :3]).all()) and bool(torch.isfinite(last[:4, 40:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,many", [(4, 1, 60), (32, 8, 5300)])
def test_prompt_rows_without_keys(ane, ty, heads, kv, many):
    """More new tokens than positions, empty sequences and unknown ones: zeros."""
    import torch

    c = make_cache([3, 0, 40], heads, kv, 128, 16)
    q = randq(many + 40, heads, 128, dt(ty))
    out = torch.full_like(q, 5.0)
    start = [0, many, many + 10, many + 10, many + 20, many + 40]
    ane.attention_prompt(c, 0, i32(start), q, out, seqs=i32([0, 1, 2, 99, 2]))
    assert not out[:many - 3].any() and not out[many:many + 20].any()
    check_rows(c, 0, 0, q[many - 3:many], out[many - 3:many], [1, 2, 3], 128 ** -0.5)
    check_rows(c, 0, 2, q[many + 20:], out[many + 20:], [21 + t for t in range(20)], 128 ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,new", [(4, 1, [4]), (4, 1, [150]), (40, 8, [1200])])
def test_broken_page_numbers_read_as_zeros(ane, heads, kv, new):
    import torch

    c = make_cache([max(500, new[0])], heads, kv, 128, 16, extra=1)
    zero = max(set(range(c.n_pages)) - set(c.page_table[0].tolist()))
    c.k_pages[0, zero] = 0
    c.v_pages[0, zero] = 0
    q = randq(new[0], heads, 128, dt("f32"))
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    for j, bad in ((3, c.n_pages), (17, NO_PAGE), (30, 0x7fffffff)):
        c.page_table[0, j] = zero
    run_prompt(c, new, q, a)
    for j, bad in ((3, c.n_pages), (17, NO_PAGE), (30, 0x7fffffff)):
        c.page_table[0, j] = bad
    run_prompt(c, new, q, b)
    assert bool((a == b).all()) and a.abs().sum() > 0
    c.kv_len[0] = 10 ** 9  # counts as max_pages * page_size
    run_prompt(c, new, q, b)
    ane.attention_shared(c, 0, q[:1], b[:1], max_len=500)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,n", [(4, 2, 40), (40, 8, 1100)])
def test_extreme_queries(ane, heads, kv, n):
    """fp32 queries far outside fp16's range, and tiny ones, keep fp32 accuracy."""
    import torch

    c = make_cache([n + 260], heads, kv, 128, 16, seed=2)
    q = randq(n, heads, 128, dt("f32"))
    q[:10] *= 1e6
    q[10:20] *= 1e-6
    q[20:30, :, ::2] *= 1e4
    out = torch.zeros_like(q)
    start = run_prompt(c, [n], q, out, scale=1e-2)
    check_prompt(c, [n], q, out, start, scale=1e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,n", [(4, 1, 40), (32, 8, 1100), (96, 8, 600)])
def test_scales_at_the_ends(ane, heads, kv, n):
    """Queries of zeros or of tiny values under a tiny scale, and large ones of
    keys that are zeros under a large scale: every score is 0 (or as good as 0),
    and masked keys stay masked."""
    c = make_cache([n + 30], heads, kv, 64, 16, seed=n)
    q = randq(n, heads, 64, dt("f32"), seed=2) * 1e-38
    q[::2] = 0
    out = q.new_empty(q.shape)
    for scale in (1e-12, 1e-37):
        start = run_prompt(c, [n], q, out, scale=scale)
        check_prompt(c, [n], q, out, start, scale=scale)
    c.k_pages.nan_to_num_(nan=0.0).mul_(0.0)
    q = randq(n, heads, 64, dt("f32"), seed=3) * 2.0 ** 110
    start = run_prompt(c, [n], q, out, scale=9e29)
    check_prompt(c, [n], q, out, start, scale=9e29)


@pytest.mark.gpu
def test_pages_past_32_bit_offsets(ane):
    """A pool of more than 4 GiB: the pages in use sit at its end."""
    import torch

    ps, kv, hd = 16, 8, 128
    pages = (1 << 32) // (ps * kv * hd * 2) + 40
    k, v = (torch.empty((1, pages, kv, ps, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    n = 20
    ids = [pages - 1 - 2 * j for j in range(n)]
    k[0, pages - 40:] = torch.randn((40, kv, ps, hd), device="cuda").half()
    v[0, pages - 40:] = torch.randn((40, kv, ps, hd), device="cuda").half()
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    c = PagedCache(32, k, v, i32([ids]), i32([n * ps - 5]), refs)
    for ty, new in (("f32", 50), ("f16", 130), ("f32", 2)):
        q = randq(new, 32, hd, dt(ty))
        out = torch.zeros_like(q)
        start = run_prompt(c, [new], q, out)
        check_prompt(c, [new], q, out, start)
    one = randq(1, 32, hd, dt("f32"))
    out = torch.zeros_like(one)
    ane.attention_shared(c, 0, one, out)
    check_rows(c, 0, 0, one, out, [n * ps - 5], hd ** -0.5)
    kk = randq(1, kv, hd, dt("f32"), 5)
    ane.paged_rope_append(c, 0, None, None, kk, kk, None, None)
    assert bool((k[0, ids[-1], :, (n * ps - 6) % ps] == kk[0].half()).all())
    ane.pages_copy(c, i32([ids[0]]), i32([pages - 2]))
    assert bool((k[0, pages - 2] == k[0, ids[0]]).all()) and bool((v[0, pages - 2] == v[0, ids[0]]).all())


# ------------------------------------------------------------------ batches
SHARED = [
    # type, hd, heads, kv, page, lengths, group bounds, prefixes
    ("f32", 128, 32, 8, 64, [4096], None, None),
    ("f32", 128, 8, 2, 16, [1, 2, 15, 16, 17, 300, 0, 1000], None, None),
    ("f16", 64, 12, 4, 48, [64, 777, 4000, 3], None, None),
    ("f32", 128, 8, 2, 16, [500, 300, 257, 256, 700], [0, 5], [256]),
    ("f32", 128, 8, 2, 16, [500, 300, 257, 256, 700], [0, 5], [251]),
    ("f16", 128, 16, 4, 64, [900 + 7 * i for i in range(20)], [0, 13, 20], [800, 333]),
    ("f32", 64, 6, 2, 48, [400, 100, 1300, 1200, 1250, 60], [1, 2, 5], [50, 1111]),
    ("f32", 128, 8, 1, 32, [3000 + i for i in range(40)], [0, 40], [2990]),
    ("f16", 64, 64, 1, 16, [200, 210], [0, 2], [100]),
]


def share(c, bounds, prefixes):
    """The members of each group take the first row's pages (whole ones) and its positions."""
    ps = c.page_size
    for a, b, p in zip(bounds, bounds[1:], prefixes):
        for s in range(a + 1, b):
            n = min(p, int(c.kv_len[s]))
            c.page_table[s, :n // ps] = c.page_table[a, :n // ps]
            if n % ps:
                j = n // ps
                for x in (c.k_pages, c.v_pages):
                    x[:, int(c.page_table[s, j]), :, :n % ps] = x[:, int(c.page_table[a, j]), :, :n % ps].clone()


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd,heads,kv,ps,lens,bounds,prefixes", SHARED)
def test_shared(ane, ty, hd, heads, kv, ps, lens, bounds, prefixes):
    import torch

    c = make_cache(lens, heads, kv, hd, ps, layers=2, seed=4)
    kw = {}
    if bounds:
        share(c, bounds, prefixes)
        kw = dict(group_start=i32(bounds), prefix_len=i32(prefixes))
    q = randq(len(lens), heads, hd, dt(ty))
    for more in (dict(max_len=max(lens), max_prefix=max(prefixes or [0])), dict(), dict(max_len=16, max_prefix=16)):
        out = torch.full_like(q, 5.0)
        ane.attention_shared(c, 1, q, out, **kw, **more)
        for s, n in enumerate(lens):
            check_rows(c, 1, s, q[s:s + 1], out[s:s + 1], [n], hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd,prefix,apart,n", [("f32", 128, 150, 0, 300), ("f16", 64, 77, 9, 300), ("f16", 128, 16, 299, 300),
                                                  ("f32", 64, 40, 0, 420), ("f16", 64, 200, 3, 420)])
def test_shared_by_a_large_group(ane, ty, hd, prefix, apart, n):
    """300 or 420 rows of 8 query heads a kv head: the prefix on 128 rows a workgroup.
    The first `apart` rows are in no group; two rows are shorter than the
    prefix."""
    import torch

    heads, kv = 128, 16
    lens = [prefix + 3 + i % 40 for i in range(n)]
    lens[40], lens[299] = prefix - 5, 1
    c = make_cache(lens, heads, kv, hd, 16, seed=6)
    share(c, [apart, n], [prefix])
    q = randq(n, heads, hd, dt(ty))
    out = torch.full_like(q, 5.0)
    ane.attention_shared(c, 0, q, out, group_start=i32([apart, n]), prefix_len=i32([prefix]), max_len=prefix + 50,
                         max_prefix=prefix)
    for s in (0, 1, 8, 9, 15, 16, 17, 40, 150, 255, 256, 298, 299):
        check_rows(c, 0, s, q[s:s + 1], out[s:s + 1], [lens[s]], hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd,heads,kv", [("f32", 128, 32, 8), ("f16", 128, 8, 8), ("f32", 64, 24, 8), ("f16", 64, 36, 9),
                                            ("f32", 128, 320, 8)])
@pytest.mark.parametrize("prefix", [0, 100])
def test_shared_many_short(ane, ty, hd, heads, kv, prefix):
    """1024 (token, kv head) pairs and more over few keys each, the last
    workgroup with some to spare, with a prefix for two groups, rows in none."""
    import torch

    n = 131
    lens = [(i * 37) % 300 + (prefix if 20 <= i < 110 else 0) for i in range(n)]
    lens[7], lens[8], lens[30], lens[130] = 0, 1, prefix - 3 if prefix else 5, 299
    c = make_cache(lens, heads, kv, hd, 16, seed=8)
    kw = {}
    if prefix:
        share(c, [20, 64, 110], [prefix, prefix])
        kw = dict(group_start=i32([20, 64, 110]), prefix_len=i32([prefix, prefix]), max_prefix=prefix)
    page = int(c.page_table[10, 1])  # seen values that are not finite stay in their rows
    c.v_pages[0, page, 0, 3, 5] = math.inf
    q = randq(n, heads, hd, dt(ty))
    out = torch.full_like(q, 5.0)
    ane.attention_shared(c, 0, q, out, max_len=400, **kw)
    for s in [s for s in range(n) if s % 6 == 0 or s in (7, 8, 20, 30, 63, 64, 109, 110, 129, 130)]:
        check_rows(c, 0, s, q[s:s + 1], out[s:s + 1], [lens[s]], hd ** -0.5)
    assert not torch.isfinite(out[10, :heads // kv, 5]).any() and bool(torch.isfinite(out[11]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd,heads,kv,groups,each", [
    ("f32", 128, 4, 2, 63, 3), ("f32", 64, 4, 1, 64, 2), ("f16", 128, 8, 2, 65, 3), ("f32", 128, 8, 8, 130, 3),
    ("f16", 64, 2, 1, 1000, 2), ("f32", 64, 1, 1, 4097, 1), ("f32", 128, 128, 1, 70, 60)])
def test_shared_by_many_groups(ane, ty, hd, heads, kv, groups, each):
    """More groups than a wave looks through in one step (63) and in two, empty ones
    and rows in none (before the first group and behind the last) among them."""
    import torch

    r = random.Random(groups)
    bounds = [2]
    for _ in range(groups):
        bounds.append(bounds[-1] + r.choice([0, 1, each, each + 1]))
    n = bounds[-1] + 3
    prefix = [r.randrange(60) for _ in range(groups)]
    lens = [r.randrange(40) for _ in range(n)]
    for a, b, p in zip(bounds, bounds[1:], prefix):
        for s in range(a, b):
            lens[s] += p if r.random() < 0.9 else 0
    c = make_cache(lens, heads, kv, hd, 16, seed=groups)
    table = c.page_table.cpu()
    for a, b, p in zip(bounds, bounds[1:], prefix):  # as share() does, and no further than the first row reaches
        for s in range(a + 1, b):
            m = min(p, lens[s], lens[a])
            table[s, :m // 16] = table[a, :m // 16]
            if m % 16:
                for x in (c.k_pages, c.v_pages):
                    x[:, int(table[s, m // 16]), :, :m % 16] = x[:, int(table[a, m // 16]), :, :m % 16].clone()
    c.page_table.copy_(table)
    q = randq(n, heads, hd, dt(ty), seed=groups)
    out = torch.full_like(q, 5.0)
    ane.attention_shared(c, 0, q, out, group_start=i32(bounds), prefix_len=i32(prefix), max_prefix=60, max_len=100)
    assert not (out == 5.0).all(2).any()
    few = {0, 1, 2, 3, n - 4, n - 3, n - 2, n - 1} | {bounds[g] + d for g in (1, 31, 32, 61, 62, 63, 64, groups // 2, groups - 1)
                                                      if g < groups for d in (-1, 0, 1)} | set(range(0, n, 1 + n // 60))
    for s in sorted(few & set(range(n))):
        check_rows(c, 0, s, q[s:s + 1], out[s:s + 1], [lens[s]], hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd,heads,kv", [("f32", 128, 32, 8), ("f16", 64, 24, 8), ("f32", 64, 16, 8)])
@pytest.mark.parametrize("given", [True, False])
def test_shared_short_rows_and_a_few_long(ane, ty, hd, heads, kv, given):
    """As above, behind bounds that leave a row's own keys open: rows of 512 own
    keys, one more, and many, in groups and in none."""
    import torch

    n, prefix = 140, [600, 40]
    lens = [7 + (i * 37) % 300 + (prefix[0] if 10 <= i < 60 else prefix[1] if 60 <= i < 110 else 0) for i in range(n)]
    lens[3], lens[4], lens[5], lens[139], lens[138] = 512, 513, 1500, 2200, 0
    lens[11], lens[12], lens[59], lens[60], lens[61] = 600 + 512, 600 + 513, 590, 40 + 1300, 39
    c = make_cache(lens, heads, kv, hd, 16, seed=21)
    share(c, [10, 60, 110], prefix)
    q = randq(n, heads, hd, dt(ty))
    out = torch.full_like(q, 5.0)
    kw = dict(max_prefix=1200, max_len=1500) if given else dict(max_len=2200)  # (a wave a row, or four)
    ane.attention_shared(c, 0, q, out, group_start=i32([10, 60, 110]), prefix_len=i32(prefix), **kw)
    for s in sorted({3, 4, 5, 10, 11, 12, 13, 58, 59, 60, 61, 62, 109, 110, 137, 138, 139} | set(range(0, n, 9))):
        check_rows(c, 0, s, q[s:s + 1], out[s:s + 1], [lens[s]], hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("ty,hd", [("f32", 128), ("f16", 64)])
def test_shared_by_a_large_group_and_a_few_long(ane, ty, hd):
    """The same beside a prefix on 128 rows a workgroup."""
    import torch

    heads, kv, n, prefix = 128, 16, 420, 150
    lens = [prefix + 3 + i % 40 for i in range(n)]
    lens[0], lens[1], lens[50], lens[51], lens[52], lens[419] = 900, 512, prefix + 513, prefix + 512, 1600, 1
    c = make_cache(lens, heads, kv, hd, 16, seed=22)
    share(c, [2, n], [prefix])
    q = randq(n, heads, hd, dt(ty))
    out = torch.full_like(q, 5.0)
    ane.attention_shared(c, 0, q, out, group_start=i32([2, n]), prefix_len=i32([prefix]), max_len=1500, max_prefix=1200)
    for s in (0, 1, 2, 3, 49, 50, 51, 52, 53, 200, 418, 419):
        check_rows(c, 0, s, q[s:s + 1], out[s:s + 1], [lens[s]], hd ** -0.5)


@pytest.mark.gpu
def test_shared_odd_groups(ane):
    """Prefixes longer than a row or than the first row, groups of none and of
    one, an unknown sequence, sequences by number, strided rows."""
    import torch

    lens = [100, 300, 40, 0, 260, 77]
    c = make_cache(lens, 8, 2, 128, 16, seed=8)
    q = randq(7, 11, 128, dt("f32"))[:, 1:9]
    out = torch.full((7, 10, 128), 5.0, device="cuda")[:, 2:]
    seqs = [4, 1, 2, 3, 99, 5, 0]
    for a, b in ((4, 1), (4, 2), (4, 3)):  # one prefix of 250 for rows 0..3, each as far as it reaches
        n = min(250, lens[b])
        c.page_table[b, :n // 16] = c.page_table[a, :n // 16]
        if n % 16:
            for x in (c.k_pages, c.v_pages):
                x[:, int(c.page_table[b, n // 16]), :, :n % 16] = x[:, int(c.page_table[a, n // 16]), :, :n % 16].clone()
    ane.attention_shared(c, 0, q, out, group_start=i32([0, 4, 4, 6, 7]), prefix_len=i32([250, 9, 30, 5000]),
                         seqs=i32(seqs), max_prefix=250, max_len=300)
    for i, s in enumerate(seqs):
        if s == 99:  # the first row of its group: nothing to share, and nothing of its own
            assert not out[i].any()
        else:
            check_rows(c, 0, s, q[i:i + 1], out[i:i + 1], [lens[s]], 128 ** -0.5)


@pytest.mark.gpu
def test_shared_lengths_hide_what_is_behind(ane):
    """Rows of the last page past the length hold NaN (make_cache), and a
    non-finite own value stays in its own sequence."""
    import torch

    c = make_cache([100, 130, 99], 4, 1, 64, 16, seed=1)
    share(c, [0, 3], [90])
    page = int(c.page_table[1, 129 // 16])
    c.v_pages[0, page, 0, 129 % 16, 7] = math.inf
    q = randq(3, 4, 64, dt("f32"))
    out = torch.zeros_like(q)
    ane.attention_shared(c, 0, q, out, group_start=i32([0, 3]), prefix_len=i32([90]))
    check_rows(c, 0, 0, q[:1], out[:1], [100], 0.125)
    check_rows(c, 0, 2, q[2:], out[2:], [99], 0.125)
    assert bool(torch.isinf(out[1, :, 7]).all()) and bool(torch.isfinite(out[1, :, :7]).all())


# ------------------------------------------------------------------ pages
class Model:
    """The page calls in plain Python."""

    def __init__(self, c):
        self.c, self.ps, self.cap = c, c.page_size, c.page_size * c.max_pages
        self.table, self.lens, self.refs = c.page_table.tolist(), c.kv_len.tolist(), c.page_refs.tolist()
        self.k, self.v = c.k_pages.clone(), c.v_pages.clone()

    def pages(self, n):
        return -(-n // self.ps)

    def take(self, need):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        return free[:need]

    def serve(self, wants):
        """wants: [(valid, pages, do)]; True for each served."""
        free = [p for p, r in enumerate(self.refs) if r == 0]
        got, used, stop = [], 0, False
        for ok, need, do in wants:
            if ok and not stop and used + need <= len(free):
                do(free[used:used + need])
                used += need
                got.append(1)
            else:
                stop |= ok
                got.append(0)
        return got

    def reserve(self, seqs, new):
        seen, wants = set(), []
        for s, n in zip(seqs, new):
            ok = 0 <= s < len(self.lens) and n <= self.cap and s not in seen
            if not ok:
                wants.append((False, 0, None))
                continue
            seen.add(s)
            at = self.pages(self.lens[s])

            def do(ids, s=s, n=n, at=at):
                for j, p in enumerate(ids):
                    self.table[s][at + j] = p
                    self.refs[p] = 1
                self.lens[s] = max(self.lens[s], n)

            wants.append((True, max(0, self.pages(n) - at), do))
        return self.serve(wants)

    def fork(self, src, dst):
        seen, wants, lens = set(), [], list(self.lens)
        for a, b in zip(src, dst):
            ok = 0 <= a < len(lens) and 0 <= b < len(lens) and a != b and lens[b] == 0 and b not in seen
            if not ok:
                wants.append((False, 0, None))
                continue
            seen.add(b)
            n = lens[a]

            def do(ids, a=a, b=b, n=n):
                for j in range(n // self.ps):
                    self.table[b][j] = self.table[a][j]
                    self.refs[self.table[a][j]] += 1
                if n % self.ps:
                    j, r = n // self.ps, n % self.ps
                    self.table[b][j] = ids[0]
                    self.refs[ids[0]] = 1
                    for x in (self.k, self.v):
                        x[:, ids[0], :, :r] = x[:, self.table[a][j], :, :r]
                self.lens[b] = n

            wants.append((True, int(n % self.ps > 0), do))
        return self.serve(wants)

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.lens):
                for j in range(self.pages(self.lens[s])):
                    self.refs[self.table[s][j]] -= 1
                    self.table[s][j] = NO_PAGE
                self.lens[s] = 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        to = {}
        for p in range(n, len(self.refs)):
            if self.refs[p]:
                q = self.refs.index(0)
                to[p] = q
                self.refs[q], self.refs[p] = self.refs[p], 0
                for x in (self.k, self.v):
                    x[:, q] = x[:, p]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return n

    def check(self):
        c = self.c
        assert c.kv_len.tolist() == self.lens
        assert c.page_refs.tolist() == self.refs
        assert c.page_table.tolist() == self.table
        assert bool((c.k_pages == self.k).all()) and bool((c.v_pages == self.v).all())


def filled_cache(**kw):
    import torch

    c = PagedCache.empty(**kw)
    c.k_pages.normal_()
    c.v_pages.normal_()
    torch.cuda.synchronize()
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("seed,ps,pages,wide", [(0, 16, 40, 8), (1, 48, 200, 20), (2, 16, 20000, 600), (3, 64, 17, 4)])
def test_page_calls_follow_the_model(ane, seed, ps, pages, wide):
    """A long mix of calls, requests that name unknown sequences, one twice or
    themselves among them, pools that run out included."""
    r = random.Random(seed)
    S = 24
    c = filled_cache(n_layers=2, n_heads=2, n_kv_heads=2, head_dim=64, page_size=ps, n_pages=pages, n_seqs=S,
                     max_pages=wide)
    m, ws = Model(c), ane.pages_workspace(c)
    for step in range(24):
        n = r.choice([1, 3, 9, 30])
        pick = [r.choice([r.randrange(S), r.randrange(S), r.randrange(-1, S + 2)]) for _ in range(n)]
        what = r.choice(["reserve", "reserve", "fork", "fork", "free", "compact", "copy"])
        got = i32([9] * n)
        if what == "reserve":
            new = [r.choice([0, 1, ps, r.randrange(wide * ps + 1), wide * ps, wide * ps + 1]) for _ in range(n)]
            want = m.reserve(pick, new)
            ane.pages_reserve(c, i32(pick), i32(new), got, workspace=ws)
            assert got.tolist() == want
        elif what == "fork":
            dst = [r.randrange(-1, S + 1) for _ in range(n)]
            want = m.fork(pick, dst)
            ane.pages_fork(c, i32(pick), i32(dst), got, workspace=ws)
            assert got.tolist() == want
        elif what == "free":
            pick = pick[:4]
            m.free(pick)
            ane.pages_free(c, i32(pick))
        elif what == "copy":
            ids = r.sample(range(pages), 8)
            for a, b in zip(ids[:4], ids[4:]):
                for x in (m.k, m.v):
                    x[:, b] = x[:, a]
            ane.pages_copy(c, i32(ids[:4] + [pages, 0]), i32(ids[4:] + [1, -1]))
        else:
            live = i32([0])
            want = m.compact()
            ane.pages_compact(c, n_live=live, workspace=ws)
            assert int(live) == want
        m.check()


@pytest.mark.gpu
def test_compact_into_arrays_of_its_own(ane):
    c = filled_cache(n_layers=1, n_heads=1, n_kv_heads=1, head_dim=64, page_size=16, n_pages=50, n_seqs=6, max_pages=9)
    m = Model(c)
    for s in range(6):
        ane.pages_reserve(c, i32([s]), i32([130]))
        m.reserve([s], [130])
    for s in (0, 2, 3):
        ane.pages_free(c, i32([s]))
        m.free([s])
    table, refs, live = c.page_table.clone(), c.page_refs.clone(), i32([0])
    t2, r2 = i32([[3] * 9] * 6), i32([4] * 50)
    for _ in range(2):  # the cache's own arrays are as before, so the same again
        ane.pages_compact(c, table_out=t2, refs_out=r2, n_live=live)
        assert bool((c.page_table == table).all()) and bool((c.page_refs == refs).all())
    m.compact()  # 50 pages hold five sequences of nine, of which 1 and 4 are left
    assert t2.tolist() == m.table and r2.tolist() == m.refs and int(live) == 18
    assert bool((c.k_pages == m.k).all()) and bool((c.v_pages == m.v).all())


@pytest.mark.gpu
def test_many_requests(ane):
    """More requests than the planning workgroup has threads."""
    S = 3000
    c = filled_cache(n_layers=1, n_heads=1, n_kv_heads=1, head_dim=64, page_size=16, n_pages=5000, n_seqs=S, max_pages=3)
    m, r = Model(c), random.Random(5)
    new = [r.randrange(49) for _ in range(S // 2)]
    got = i32([0] * (S // 2))
    ane.pages_reserve(c, i32(list(range(S // 2))), i32(new), got)
    assert got.tolist() == m.reserve(range(S // 2), new)
    src, dst = [r.randrange(S // 2) for _ in range(2500)], [r.randrange(S // 2, S) for _ in range(2500)]
    got = i32([0] * 2500)
    ane.pages_fork(c, i32(src), i32(dst), got)
    assert got.tolist() == m.fork(src, dst)
    m.check()
    gone = [r.randrange(S) for _ in range(2000)]
    ane.pages_free(c, i32(gone))
    m.free(gone)
    m.check()


@pytest.mark.gpu
@pytest.mark.parametrize("need", [[8192], [5000, 1, 17, 0, 300, 16, 2], [70] * 40 + [400], [18] * 64 + [65, 257, 1]])
def test_reserve_long_rows(ane, need):
    """Requests for many pages, among short ones: the pages of the pool in order."""
    import torch

    total, n, wide = sum(need), len(need), max(need)
    c = PagedCache.empty(1, 1, 1, 64, 16, total + 40, n + 2, wide)
    taken = random.Random(n).sample(range(total + 40), 40)
    c.page_refs[i32(taken).long()] = 1
    order = random.Random(n + 1).sample(range(n + 2), n)
    served = i32([7] * n)
    ane.pages_reserve(c, i32(order), i32([16 * m - (m > 0) for m in need]), served)
    free = [p for p in range(total + 40) if p not in set(taken)]
    want = np.full((n + 2, wide), NO_PAGE, np.int32)
    for s, m in zip(order, need):
        want[s, :m], free = free[:m], free[m:]
    assert served.tolist() == [1] * n and not free
    assert np.array_equal(c.page_table.cpu().numpy(), want)
    assert bool((c.page_refs == 1).all())
    assert [int(x) for x in c.kv_len.cpu()[order]] == [16 * m - (m > 0) for m in need]


@pytest.mark.gpu
def test_reserve_more_pages_than_32_bits_count(ane):
    """Requests for 2^26 pages each, 40 of them behind two small ones."""
    import torch

    k = torch.zeros(1, 100, 1, 16, 64, dtype=torch.float16, device="cuda")
    table = torch.empty(44, 1 << 26, dtype=torch.int32, device="cuda")
    table[:, :8] = NO_PAGE
    c = PagedCache(1, k, k.clone(), table, i32([0] * 44), i32([0] * 100))
    served = i32([7] * 43)
    ane.pages_reserve(c, i32(range(43)), i32([33, 5] + [1 << 30] * 40 + [1]), served)
    assert served.tolist() == [1, 1] + [0] * 41
    assert table[:2, :4].tolist() == [[0, 1, 2, -1], [3, -1, -1, -1]] and bool((table[2:, :8] == -1).all())
    assert c.kv_len.tolist() == [33, 5] + [0] * 42 and int(c.page_refs.sum()) == 4


@pytest.mark.gpu
def test_pools_past_one_look(ane):
    """More pages than the planning workgroup looks at at a time (65536)."""
    P = 140001
    c = filled_cache(n_layers=1, n_heads=1, n_kv_heads=1, head_dim=64, page_size=16, n_pages=P, n_seqs=9, max_pages=60000)
    m, ws = Model(c), ane.pages_workspace(c)
    n = [16 * 60000 - 7, 16 * 50000, 16 * 29990 + 1, 3]
    got = i32([0] * 4)
    ane.pages_reserve(c, i32([3, 0, 8, 5]), i32(n), got, workspace=ws)
    assert got.tolist() == m.reserve([3, 0, 8, 5], n) == [1, 1, 1, 1]
    ane.pages_free(c, i32([3]))
    m.free([3])
    got = i32([0] * 3)
    ane.pages_fork(c, i32([8, 5, 0]), i32([1, 2, 4]), got, workspace=ws)
    assert got.tolist() == m.fork([8, 5, 0], [1, 2, 4]) == [1, 1, 1]
    m.check()
    live = i32([0])
    ane.pages_compact(c, n_live=live, workspace=ws)
    assert int(live) == sum(r > 0 for r in m.refs)
    moves = [p for p in range(int(live), P) if m.refs[p]]
    holes = [p for p in range(int(live)) if not m.refs[p]]
    to = dict(zip(moves, holes))
    for a, b in to.items():
        m.refs[b], m.refs[a] = m.refs[a], 0
    m.k[:, holes], m.v[:, holes] = m.k[:, moves], m.v[:, moves]
    m.table = [[to.get(p, p) for p in row] for row in m.table]
    m.check()


# ------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "f16"])
def test_serving_run(ane, ty):
    """A prompt appended and attended in two chunks, forked, the samples decoded
    behind their common prefix, some freed, the pool compacted, decoding goes
    on: every step against the formula over the tokens each sequence was given."""
    import torch

    heads, kv, hd, ps, S = 8, 2, 128, 16, 6
    c = PagedCache.empty(1, heads, kv, hd, ps, 60, S, 12)
    c.k_pages.fill_(math.nan)
    c.v_pages.fill_(math.nan)
    table = torch.from_numpy(ane.rope_table(200, hd)).cuda()
    ws = ane.pages_workspace(c)
    history = {s: ([], []) for s in range(S)}  # fp16 rows [kv][hd] of each sequence

    def step(seqs, new, seed, group=None):
        lens = [len(history[s][0]) for s in seqs]
        ok = i32([0] * len(seqs))
        ane.pages_reserve(c, i32(seqs), i32([a + b for a, b in zip(lens, new)]), ok, workspace=ws)
        assert ok.tolist() == [1] * len(seqs)
        T = sum(new)
        qkv = randq(T, heads + 2 * kv, hd, dt("f32"), seed)
        q = torch.empty((T, heads, hd), dtype=dt(ty), device="cuda")
        out = torch.zeros_like(q)
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        ane.paged_rope_append(c, 0, i32(start), qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], table, q,
                              seqs=i32(seqs))
        if group:
            ane.attention_shared(c, 0, q, out, group_start=i32([0, len(seqs)]), prefix_len=i32([group]), seqs=i32(seqs))
        else:
            ane.attention_prompt(c, 0, i32(start), q, out, seqs=i32(seqs))
        host = qkv.cpu().numpy()
        cs = table.cpu().numpy()
        for i, s in enumerate(seqs):
            for t in range(new[i]):
                r = start[i] + t
                history[s][0].append(np_turn(host[r, heads:heads + kv], cs[lens[i] + t][None]).astype(np.float16))
                history[s][1].append(host[r, heads + kv:].astype(np.float16))
            n = lens[i] + new[i]
            k, v = seq_kv(c, 0, s, n)
            for got, want in ((k, history[s][0]), (v, history[s][1])):
                same = np.array_equal(got.cpu().numpy(), np.stack(want, 1).astype(np.float64))
                assert same, (s, n)
            check_rows(c, 0, s, q[start[i]:start[i + 1]], out[start[i]:start[i + 1]],
                       [lens[i] + t + 1 for t in range(new[i])], hd ** -0.5)

    step([2], [70], 1)
    step([2, 0], [23, 40], 2)
    ane.pages_fork(c, i32([2, 2, 2]), i32([3, 4, 5]), workspace=ws)
    for s in (3, 4, 5):
        history[s] = (list(history[2][0]), list(history[2][1]))
    for i in range(20):
        step([2, 3, 4, 5], [1] * 4, 10 + i, group=93)
    ane.pages_free(c, i32([0, 3]))
    history[0], history[3] = ([], []), ([], [])
    ane.pages_compact(c, workspace=ws)
    refs = c.page_refs.tolist()
    live = sum(r > 0 for r in refs)
    assert all(refs[:live]) and not any(refs[live:])
    for i in range(3):
        step([4, 2, 5], [1] * 3, 50 + i, group=93)
    step([3, 0], [18, 1], 70)


@pytest.mark.gpu
def test_a_page_of_ctx_positions_is_the_decode_cache(ane):
    """max_pages 1, page_size ctx: the layout of ane_hip_attention_decode."""
    import torch

    ctx, heads, kv = 1024, 32, 8
    cfg = ane.DecodeConfig(1, 4096, 14336, heads, kv, 128, ctx, 1e-5)
    k, v = (torch.randn((1, 1, kv, ctx, 128), device="cuda").half() for _ in range(2))
    c = PagedCache(heads, k, v, i32([[0]]), i32([900]))
    q = randq(1, heads, 128, dt("f32"))
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    ane.attention_decode(cfg, q, k, v, 900, a)
    ane.attention_shared(c, 0, q, b)
    _, tol = formula(c, 0, 0, q, [900], 128 ** -0.5)
    assert bool(((a - b).abs() <= 2 * tol).all())


@pytest.mark.gpu
def test_captured_calls_follow_lengths_and_tables(ane):
    """One graph of a decode step, replayed while the lengths grow, with eager
    work between the replays; each replay against the eager calls."""
    import torch

    heads, kv, hd, ps, S = 8, 2, 128, 16, 3
    c = PagedCache.empty(1, heads, kv, hd, ps, 80, S, 24)
    table = torch.from_numpy(ane.rope_table(400, hd)).cuda()
    qkv = randq(S, heads + 2 * kv, hd, dt("f32"))
    q, out = (torch.zeros((S, heads, hd), device="cuda") for _ in range(2))
    want, new, seqs = i32([0] * S), i32([200, 30, 111]), i32([0, 1, 2])
    gs, pl = i32([0, 3]), i32([0])
    ws, aw = ane.pages_workspace(c), ane.attention_shared_workspace(c, S, 1, 384, 384)

    def step():
        ane.pages_reserve(c, seqs, new, want, workspace=ws)
        ane.paged_rope_append(c, 0, None, qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], table, q)
        ane.attention_shared(c, 0, q, out, group_start=gs, prefix_len=pl, max_prefix=384, max_len=384, workspace=aw)

    c.k_pages.normal_()
    c.v_pages.normal_()
    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step()
    for i in range(5):
        new += i32([1, 40, 7])
        qkv.normal_()
        g.replay()
        got = out.clone()
        assert want.tolist() == [1] * S and c.kv_len.tolist() == new.tolist()
        for s in range(S):
            check_rows(c, 0, s, q[s:s + 1], got[s:s + 1], [int(new[s])], hd ** -0.5)
        out.fill_(3.0)
        ane.attention_shared(c, 0, q, out, group_start=gs, prefix_len=pl, max_prefix=384, max_len=384)
        assert bool((out == got).all())


@pytest.mark.gpu
def test_wrappers_refuse_tensors_of_another_device(ane):
    """A tensor in host memory among those of a cache on the GPU."""
    import torch

    c = make_cache([40, 20], 4, 2, 64, 16, fill_rest=0.0)
    q, n2 = randq(3, 4, 64, dt("f32")), i32([0, 1])
    qs, ws = i32([0, 2, 3]), torch.zeros(1 << 20, dtype=torch.uint8)
    table = torch.zeros(64, 32, 2)
    for call in (lambda: ane.attention_prompt(c, 0, qs.cpu(), q, q), lambda: ane.attention_prompt(c, 0, qs, q.cpu(), q),
                 lambda: ane.attention_prompt(c, 0, qs, q, q.cpu()), lambda: ane.attention_prompt(c, 0, qs, q, q, workspace=ws),
                 lambda: ane.attention_prompt(c, 0, qs, q, q, seqs=n2.cpu()),
                 lambda: ane.attention_shared(c, 0, q, q, seqs=qs.cpu()),
                 lambda: ane.attention_shared(c, 0, q, q, group_start=n2, prefix_len=n2.cpu()),
                 lambda: ane.paged_rope_append(c, 0, qs, q, q[:, :2], q[:, 2:], table, q),
                 lambda: ane.paged_rope_append(c, 0, qs, None, q[:, :2].cpu(), q[:, 2:].cpu(), None, None),
                 lambda: ane.pages_reserve(c, n2, n2.cpu()), lambda: ane.pages_fork(c, n2, n2, n2.cpu()),
                 lambda: ane.pages_free(c, n2.cpu()), lambda: ane.pages_copy(c, n2, n2.cpu()),
                 lambda: ane.pages_compact(c, n_live=n2.cpu()), lambda: ane.pages_compact(c, workspace=ws)):
        with pytest.raises(ValueError, match="device"):
            call()
    with pytest.raises(ValueError):
        PagedCache(4, c.k_pages, c.v_pages, c.page_table.cpu(), c.kv_len)


@pytest.mark.gpu
def test_two_streams(ane):
    """Calls at once on two streams, each with its own workspace."""
    import torch

    c = make_cache([3000, 2500, 40, 1200], 8, 2, 128, 16, seed=6)
    q1, q2 = randq(4, 8, 128, dt("f32"), 1), randq(130, 8, 128, dt("f16"), 2)
    a, b = torch.zeros_like(q1), torch.zeros_like(q2)
    ane.attention_shared(c, 0, q1, a)
    ane.attention_prompt(c, 0, i32([0, 10, 130]), q2, b, seqs=i32([1, 0]))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    start, sq = i32([0, 10, 130]), i32([1, 0])
    torch.cuda.synchronize()
    for _ in range(10):
        x, y = torch.zeros_like(q1), torch.zeros_like(q2)
        torch.cuda.synchronize()
        ane.attention_shared(c, 0, q1, x, stream=s1)
        ane.attention_prompt(c, 0, start, q2, y, seqs=sq, stream=s2)
        torch.cuda.synchronize()
        assert bool((x == a).all()) and bool((y == b).all())
