"""The int8 linear layer of a batch (include/ane_decode.h; ane_amd/csrc/linear_i8.hip):
tokens quantized with a scale each, the product with the scales of token and
channel.

Everything is defined step by step in 32 bits around an exact integer sum, so
the results are compared bit for bit with the same steps in numpy (the sum of
squares of the norm is the one place with a free order: 64-bit sums whose
rounding to 32 bits the order does not reach for these inputs).
"""
import itertools

import numpy as np
import pytest

import ane_amd
from ane_amd import AneError

P = 0x10000  # an address no refused call touches


# ------------------------------------------------------------------ the steps in numpy
def quantized(x, norm_w=None, eps=1e-5):
    y = x.astype(np.float32)
    with np.errstate(all="ignore"):
        if norm_w is not None:
            ms = ((y.astype(np.float64) ** 2).sum(axis=1) / x.shape[1]).astype(np.float32)
            inv = np.float32(1) / np.sqrt(ms + np.float32(eps))
            y = (y * inv[:, None]) * norm_w
        top = np.abs(y).max(axis=1)  # (NaN where there is one)
        up = np.where(top < np.float32(2.0 ** -96), np.float32(2.0 ** 96), np.float32(1))
        scale = np.where(top == 0, np.float32(1), top * up / np.float32(127) / up)
        per = np.where(top == 0, np.float32(127), np.float32(1) / (top * up) * np.float32(127))
        t = (y * up[:, None]) * per[:, None]
        q = np.rint(np.clip(np.where(np.isnan(t), 0, t), -127, 127)).astype(np.int8)
    return q, scale.astype(np.float32)


def product(q, qs, w, ws, bias=None, residual=None, half=False):
    acc = q.astype(np.float64) @ w.astype(np.float64).T  # exact: below 2^53
    with np.errstate(all="ignore"):
        y = acc.astype(np.float32) * qs[:, None] * ws
        y = y + (np.float32(0) if bias is None else bias)
        if residual is not None:
            y = y + residual.astype(np.float32)
        return y.astype(np.float16) if half else y


def same(got, want):
    assert got.shape == want.shape and got.dtype == want.dtype
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))[:5]


def inputs(T, N, K, seed=0, half_in=False, half_out=False):
    r = np.random.default_rng(seed * 1000003 + T * 7919 + N * 31 + K)
    x = (r.standard_normal((T, K)) * np.exp(r.uniform(-4, 4, (T, 1)))).astype(np.float16 if half_in else np.float32)
    w = r.integers(-128, 128, (N, K)).astype(np.int8)
    ws = (r.uniform(0.1, 1.1, N) * 1e-3).astype(np.float32)
    norm = (1 + 0.1 * r.standard_normal(K)).astype(np.float32)
    bias = r.standard_normal(N).astype(np.float32)
    res = r.standard_normal((T, N)).astype(np.float16 if half_out else np.float32)
    return x, w, ws, norm, bias, res


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rows16(a, fill=99):
    """int8 rows on the device, each starting on 16 bytes, `fill` behind the last value."""
    import torch

    n, k = a.shape
    t = torch.full((n, (k + 15) // 16 * 16), fill, dtype=torch.int8, device="cuda")
    t[:, :k] = dev(a)
    return t[:, :k]


# ------------------------------------------------------------------ CPU: refusals
def c_quant(T=4, K=64, ty=0, x=P, xs=64, nw=None, eps=1e-5, q=P, qs=64, sc=P):
    return ane_amd.lib().ane_hip_quantize_tokens(T, K, ty, x, xs, nw, eps, q, qs, sc, None)


def c_dense(T=4, N=8, K=64, q=P, qs=64, sc=P, w=P, wst=64, ws=P, bias=None, res=None, rst=0, ty=0, out=P, os_=8):
    return ane_amd.lib().ane_hip_dense_i8_scaled(T, N, K, q, qs, sc, w, wst, ws, bias, res, rst, ty, out, os_, None)


def c_linear(T=4, N=8, K=64, ty=0, x=P, xs=64, nw=None, eps=1e-5, w=P, wst=64, ws=P, bias=None, res=None, rst=0, to=0, out=P,
             os_=8, work=P, wb=1 << 40):
    return ane_amd.lib().ane_hip_linear_i8(T, N, K, ty, x, xs, nw, eps, w, wst, ws, bias, res, rst, to, out, os_, work, wb, None)


INVALID, POINTER, WORKSPACE = 1, 2, 8


@pytest.mark.parametrize("kw,st", [
    (dict(K=0), INVALID), (dict(K=1 << 17), INVALID), (dict(ty=2), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(x=None), POINTER), (dict(q=None), POINTER), (dict(sc=None), POINTER),
    (dict(x=P + 2), INVALID), (dict(ty=1, x=P + 1), INVALID), (dict(xs=63), INVALID), (dict(q=P + 8), INVALID),
    (dict(qs=72), INVALID), (dict(qs=48), INVALID), (dict(sc=P + 1), INVALID), (dict(nw=P + 2), INVALID),
    (dict(T=65535 * 128 + 1), INVALID), (dict(T=0), 0), (dict(T=0, x=None, q=None), 0)])
def test_quantize_refusals(kw, st):
    assert c_quant(**kw) == st


@pytest.mark.parametrize("kw,st", [
    (dict(K=0), INVALID), (dict(K=1 << 17), INVALID), (dict(ty=2), INVALID), (dict(q=None), POINTER), (dict(sc=None), POINTER),
    (dict(w=None), POINTER), (dict(ws=None), POINTER), (dict(out=None), POINTER), (dict(q=P + 4), INVALID),
    (dict(w=P + 8), INVALID), (dict(qs=56), INVALID), (dict(qs=1 << 31), INVALID), (dict(wst=48), INVALID),
    (dict(wst=72), INVALID), (dict(wst=1 << 31), INVALID), (dict(os_=7), INVALID), (dict(res=P, rst=7), INVALID),
    (dict(out=P + 2), INVALID), (dict(ty=1, out=P + 1), INVALID), (dict(res=P + 2, rst=8), INVALID), (dict(bias=P + 2), INVALID),
    (dict(ws=P + 2), INVALID), (dict(T=65535 * 128 + 1), INVALID), (dict(N=65535 * 128 + 1, os_=1 << 30), INVALID),
    (dict(T=1 << 19, N=1 << 19, os_=1 << 19), INVALID), (dict(T=0), 0), (dict(N=0), 0)])
def test_dense_refusals(kw, st):
    assert c_dense(**kw) == st


@pytest.mark.parametrize("kw,st", [
    (dict(K=0), INVALID), (dict(ty=3), INVALID), (dict(to=2), INVALID), (dict(x=None), POINTER), (dict(w=None), POINTER),
    (dict(work=None), WORKSPACE), (dict(work=P + 128), WORKSPACE), (dict(wb=0), WORKSPACE), (dict(wst=56), INVALID),
    (dict(T=0), 0), (dict(N=0), 0)])
def test_linear_refusals(kw, st):
    assert c_linear(**kw) == st


def test_workspace_size():
    f = ane_amd.lib().ane_hip_linear_i8_workspace_size
    assert f(0, 5, 5) == f(5, 0, 5) == f(5, 5, 0) == f(5, 5, 1 << 17) == 0
    assert f(7, 5, 100) >= 7 * 112 + 7 * 4
    need = f(3, 8, 64)
    assert c_linear(T=3, wb=need - 1) == WORKSPACE


def test_python_refusals():
    import torch

    x, w, out = torch.zeros(2, 64), torch.zeros(8, 64, dtype=torch.int8), torch.zeros(2, 8)
    ws, q, qs = torch.ones(8), torch.zeros(2, 64, dtype=torch.int8), torch.ones(2)
    with pytest.raises(ValueError, match="GPU"):
        ane_amd.linear_i8(x, w, ws, out)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(w=w.float()), dict(w=w[:, :63]), dict(w=w.t().contiguous().t()),
                dict(w_scales=ws.double()), dict(w_scales=ws[:7]), dict(out=out[:, :7]), dict(out=out[:1]),
                dict(out=out.double()), dict(norm_w=torch.ones(63)), dict(bias=torch.ones(9)), dict(residual=out.half()),
                dict(residual=out[:, :7]), dict(x=x[:1].expand(2, 64)), dict(out=out[:1].expand(2, 8))):
        with pytest.raises(ValueError):
            ane_amd.linear_i8(**{**dict(x=x, w=w, w_scales=ws, out=out), **bad})
    for bad in (dict(q=q.float()), dict(q=torch.zeros(2, 60, dtype=torch.int8)), dict(scales=qs[:1]), dict(x=x[:1])):
        with pytest.raises(ValueError):
            ane_amd.quantize_tokens(**{**dict(x=x, q=q, scales=qs), **bad})
    # the last row's own bytes end before the next 16
    flat = torch.zeros(64 + 60, dtype=torch.int8)
    with pytest.raises(ValueError, match="last row"):
        ane_amd.dense_i8_scaled(torch.as_strided(flat, (2, 60), (64, 1)), qs, w[:, :60], ws, out)


# ------------------------------------------------------------------ GPU
def run_quant(x, norm=None, eps=1e-5):
    import torch

    T, K = x.shape
    buf = torch.full((T, (K + 15) // 16 * 16 + 16), 77, dtype=torch.int8, device="cuda")
    sc = torch.empty(T, device="cuda")
    ane_amd.quantize_tokens(dev(x), buf[:, :K], sc, norm_w=None if norm is None else dev(norm), eps=eps)
    torch.cuda.synchronize()
    b = buf.cpu().numpy()
    kp = (K + 15) // 16 * 16
    assert (b[:, K:kp] == 0).all() and (b[:, kp:] == 77).all()
    return b[:, :K], sc.cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("K", [1, 7, 8, 9, 100, 511, 512, 513, 2047, 2048, 2049, 4096, 5000, 8192, 14336, 16384, 16385, 50001,
                               131071])
def test_quantize(ane, K, norm, half):
    T = 5 if K > 512 else 9
    x, _, _, nw, _, _ = inputs(T, 1, K, seed=1, half_in=half)
    if T > 3:
        x[2] = 0
    q, s = run_quant(x, nw if norm else None)
    wq, wsc = quantized(x, nw if norm else None)
    same(s, wsc)
    same(q, wq)


@pytest.mark.gpu
def test_quantize_special_values(ane):
    K = 700
    x = np.random.default_rng(5).standard_normal((9, K)).astype(np.float32)
    x[0] *= 1e-42  # denormal
    x[1] *= np.float32(1e-38)
    x[2] *= np.float32(3e37)
    x[3, 5] = np.inf
    x[4, 699] = np.nan
    x[5] = 0
    x[5, 0] = np.float32(1e-45)
    x[6] = np.float32(-0.0)
    x[7] = np.float32(2.5)  # all at the maximum
    x[8] = np.arange(K, dtype=np.float32) * np.float32(127.0 / 254) % np.float32(127)  # halves: ties to even
    x[8, 0] = 127
    q, s = run_quant(x)
    wq, wsc = quantized(x)
    same(s, wsc)
    same(q, wq)
    # (2^-149 / 127 is below half of the smallest fp32, 2^-150: it rounds to 0, and so does all of that token)
    assert np.isinf(s[3]) and np.isnan(s[4]) and s[5] == 0 and s[6] == 1
    # a row that is not finite gives rows of NaN and touches no other
    w, ws = np.ones((3, K), np.int8), np.ones(3, np.float32)
    import torch

    out = torch.zeros((9, 3), device="cuda")
    ane.linear_i8(dev(x), rows16(w), dev(ws), out)
    o = out.cpu().numpy()
    assert np.isnan(o[3:5]).all() and not np.isnan(np.delete(o, [3, 4], axis=0)).any()
    same(o, product(wq, wsc, w, ws))


SHAPES = [(1, 1, 1), (1, 6144, 4096), (1, 17, 31), (2, 100, 777), (3, 16, 16), (5, 33, 100), (15, 2003, 64), (16, 4096, 513),
          (17, 48, 1000), (32, 4096, 14336), (33, 500, 200), (64, 1000, 4096), (65, 129, 96), (100, 4096, 4096), (128, 640, 1777),
          (129, 300, 130), (200, 8192, 256), (256, 256, 64), (301, 2003, 1777), (512, 4096, 1040), (600, 5000, 1000),
          (1000, 1536, 1000), (1024, 1024, 4096), (2048, 4096, 512), (4096, 4096, 144), (5000, 3000, 48), (9000, 130, 80), (76, 39, 7203), (300, 5, 400), (40, 20, 9000), (100, 61, 3000),
          (300, 28672, 192)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", SHAPES)
def test_linear(ane, T, N, K):
    import torch

    i = SHAPES.index((T, N, K))
    for k, (half_in, half_out) in enumerate(itertools.product([False, True], [False, True])):
        x, w, ws, norm, bias, res = inputs(T, N, K, seed=2, half_in=half_in, half_out=half_out)
        use = [(i + k) & 1, (i + k) & 2, (i ^ k) & 4]
        norm, bias, res = (v if u else None for v, u in zip((norm, bias, res), use))
        q, qs = quantized(x, norm)
        want = product(q, qs, w, ws, bias, res, half_out)
        d = [None if v is None else dev(v) for v in (norm, bias, res)]
        out = torch.full((T, N), float("nan"), dtype=torch.float16 if half_out else torch.float32, device="cuda")
        W = rows16(w)
        ane.linear_i8(dev(x), W, dev(ws), out, norm_w=d[0], bias=d[1], residual=d[2])
        same(out.cpu().numpy(), want)
        out.fill_(float("nan"))
        ane.dense_i8_scaled(rows16(q, fill=0), dev(qs), W, dev(ws), out, bias=d[1], residual=d[2])
        same(out.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(1, 130, 200), (20, 100, 300), (130, 260, 256), (700, 4099, 320), (5000, 3333, 64)])
@pytest.mark.parametrize("half", [False, True])
def test_strides_and_in_place(ane, T, N, K, half):
    """Rows inside wider ones at odd offsets; the residual is the output."""
    import torch

    ty = torch.float16 if half else torch.float32
    x, w, ws, norm, bias, res = inputs(T, N, K, seed=3, half_in=half, half_out=half)
    wide_x = torch.zeros((T, K + 5), dtype=ty, device="cuda")
    wide_x[:, 3:3 + K] = dev(x)
    wide_w = torch.full((N, 16 + (K + 15) // 16 * 16), 55, dtype=torch.int8, device="cuda")
    wide_w[:, 16:16 + K] = dev(w)
    for lead in (1, 4):  # out's rows off and on vector alignment
        wide = torch.full((T, N + lead + 3), 7.0, dtype=ty, device="cuda")
        o = wide[:, lead:lead + N]
        o.copy_(dev(res))
        ane.linear_i8(wide_x[:, 3:3 + K], wide_w[:, 16:16 + K], dev(ws), o, norm_w=dev(norm), bias=dev(bias), residual=o)
        q, qs = quantized(x, norm)
        same(o.cpu().numpy(), product(q, qs, w, ws, bias, res, half))
        assert (wide[:, :lead] == 7).all() and (wide[:, lead + N:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(5, 2100), (300, 2100)])
def test_weights_past_32_bit_offsets(ane, T, N):
    import torch

    K, stride = 96, 1 << 20
    x, w, ws, _, bias, _ = inputs(T, N, K, seed=4)
    big = torch.zeros((N, stride), dtype=torch.int8, device="cuda")  # 2.2 GB
    big[:, :K] = dev(w)
    out = torch.zeros((T, N), device="cuda")
    ane.linear_i8(dev(x), big[:, :K], dev(ws), out, bias=dev(bias))
    q, qs = quantized(x)
    same(out.cpu().numpy(), product(q, qs, w, ws, bias))


@pytest.mark.gpu
def test_largest_sums(ane):
    """K at its limit with every product at its largest: the sums come within 2^15 of 2^31."""
    import torch

    K = (1 << 17) - 1
    for T in (1, 40, 300):
        q = torch.full((T, K + 1), -128, dtype=torch.int8, device="cuda")
        q[:, K:] = 0
        w = torch.full((256, K + 1), -128, dtype=torch.int8, device="cuda")
        w[1::2] = 127
        out = torch.zeros((T, 256), device="cuda")
        ane.dense_i8_scaled(q[:, :K], torch.ones(T, device="cuda"), w[:, :K], torch.ones(256, device="cuda"), out)
        o = out.cpu().numpy()
        assert (o[:, ::2] == np.float32(K * 16384)).all() and (o[:, 1::2] == np.float32(-K * 128 * 127)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(1, 6144, 4096), (32, 4096, 14336), (100, 4096, 4096), (600, 5000, 1000)])
def test_other_stream_and_graph(ane, T, N, K):
    """Called on a stream of its own, then captured; replays follow new inputs, with eager calls between them."""
    import torch

    x, w, ws, norm, _, res = inputs(T, N, K, seed=5)
    X, W, S, R, nw = dev(x), rows16(w), dev(ws), dev(res), dev(norm)
    out, work = torch.zeros((T, N), device="cuda"), ane.linear_i8_workspace(T, N, K)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    ane.linear_i8(X, W, S, out, norm_w=nw, residual=R, workspace=work, stream=st)
    st.synchronize()
    want = product(*quantized(x, norm), w, ws, None, res)
    same(out.cpu().numpy(), want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ane.linear_i8(X, W, S, out, norm_w=nw, residual=R, workspace=work)
    for i in range(3):
        x2 = inputs(T, N, K, seed=6 + i)[0]
        X.copy_(dev(x2))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        same(out.cpu().numpy(), product(*quantized(x2, norm), w, ws, None, res))
        eager = torch.zeros_like(out)
        ane.linear_i8(X, W, S, eager, norm_w=nw, residual=R)  # a workspace of its own
        assert torch.equal(eager, out)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 8, 40, 300])
@pytest.mark.parametrize("half", [False, True])
def test_output_in_place_of_the_input(ane, T, half):
    """x = residual = out, as in a layer whose input nobody needs afterwards, with many workgroups that read a token."""
    N = K = 8192
    x, w, ws, norm, bias, _ = inputs(T, N, K, seed=9, half_in=half, half_out=half)
    X, W, S, nw, b = dev(x), rows16(w), dev(ws), dev(norm), dev(bias)
    for i in range(3):
        want = product(*quantized(x, norm), w, ws, bias, x, half)
        ane.linear_i8(X, W, S, X, norm_w=nw, bias=b, residual=X)
        x = X.cpu().numpy()
        same(x, want)
    y = dev(inputs(T, N, K, seed=10, half_in=half)[0])
    want = product(*quantized(y.cpu().numpy(), None), w[:-96], ws[:-96], None, None, half)
    ane.linear_i8(y, W[:-96], S[:-96], y[:, 96:])  # behind its start
    same(y[:, 96:].cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(3, 300), (100, 600)])
def test_tokens_past_32_bit_offsets(ane, T, N):
    import torch

    K, stride = 80, (1 << 31) // (T - 1) // 16 * 16 + 16
    x, w, ws, _, bias, _ = inputs(T, N, K, seed=11)
    q, qs = quantized(x)
    far = torch.zeros((T, stride), dtype=torch.int8, device="cuda")  # up to 3.2 GB
    far[:, :K] = dev(q)
    out = torch.zeros((T, N), device="cuda")
    ane.dense_i8_scaled(far[:, :K], dev(qs), rows16(w), dev(ws), out, bias=dev(bias))
    same(out.cpu().numpy(), product(q, qs, w, ws, bias))


@pytest.mark.gpu
def test_two_streams_at_once(ane):
    """K in parts on two streams, each with its workspace, many calls in flight."""
    import torch

    T, N, K = 32, 4096, 14336
    jobs = []
    for seed in (12, 13):
        x, w, ws, norm, _, _ = inputs(T, N, K, seed=seed)
        jobs.append((torch.cuda.Stream(), dev(x), rows16(w), dev(ws), dev(norm), [torch.zeros((T, N), device="cuda") for _ in range(6)],
                     ane.linear_i8_workspace(T, N, K), product(*quantized(x, norm), w, ws, None, None)))
    torch.cuda.synchronize()
    for i in range(6):
        for st, X, W, S, nw, outs, work, _ in jobs:
            ane.linear_i8(X, W, S, outs[i], norm_w=nw, workspace=work, stream=st)
    torch.cuda.synchronize()
    for *_, outs, _, want in jobs:
        for o in outs:
            same(o.cpu().numpy(), want)


@pytest.mark.gpu
def test_zero_sizes_leave_outputs(ane):
    import torch

    out = torch.full((0, 8), 3.0, device="cuda")
    w, ws = torch.zeros((8, 64), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    ane.linear_i8(torch.zeros((0, 64), device="cuda"), w, ws, out)
    with pytest.raises((AneError, ValueError)):
        ane.linear_i8(torch.zeros((2, 0), device="cuda"), torch.zeros((8, 0), dtype=torch.int8, device="cuda"), ws,
                      torch.zeros((2, 8), device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("K", [100, 777, 1777, 4096, 5000, 14336, 20000])
@pytest.mark.parametrize("half", [False, True])
def test_a_token_does_not_depend_on_its_batch(ane, K, half):
    """The integers, the scale and the row of the product have the same bits alone and in batches of every size, whichever
    kernels they go through; the norm is ane_hip_rms_norm's."""
    import torch

    N, T = 200, 1100
    x, w, ws, norm, bias, _ = inputs(T, N, K, seed=9, half_in=half)
    X, W, S, nw, B = dev(x), rows16(w), dev(ws), dev(norm), dev(bias)
    q0 = torch.zeros((T, (K + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :K]
    s0, out0 = torch.zeros(T, device="cuda"), torch.zeros((T, N), device="cuda")
    ane.quantize_tokens(X, q0, s0, norm_w=nw)
    ane.linear_i8(X, W, S, out0, norm_w=nw, bias=B)
    for n in (1, 2, 3, 8, 16, 40, 64, 100, 257, 600):
        q, s, out = rows16(np.zeros((n, K), np.int8), fill=0), torch.zeros(n, device="cuda"), torch.zeros((n, N), device="cuda")
        ane.quantize_tokens(X[:n], q, s, norm_w=nw)
        ane.linear_i8(X[:n], W, S, out, norm_w=nw, bias=B)
        assert torch.equal(q, q0[:n]) and torch.equal(s, s0[:n]) and torch.equal(out, out0[:n])
        ane.dense_i8_scaled(q, s, W, S, out.zero_(), bias=B)
        assert torch.equal(out, out0[:n])
    if K % 32 == 0 and not half:
        y, one = torch.zeros(K, device="cuda"), torch.zeros(1, device="cuda")
        ane.rms_norm(K, X[3].contiguous(), nw, 1e-5, y)
        qy = torch.zeros((1, K), dtype=torch.int8, device="cuda")
        ane.quantize_tokens(y[None], qy, one)
        assert torch.equal(qy[0], q0[3]) and torch.equal(one[0], s0[3])


@pytest.mark.gpu
def test_one_token_over_very_many_rows(ane):
    """More rows than 64 a wave on two workgroups a CU."""
    import torch

    N, K = 300_001, 48
    x, w, ws, _, bias, _ = inputs(1, N, K, seed=10)
    out = torch.zeros((1, N), device="cuda")
    ane.linear_i8(dev(x), rows16(w), dev(ws), out, bias=dev(bias))
    same(out.cpu().numpy(), product(*quantized(x), w, ws, bias))


def test_plans():
    """Which kernel takes a product (ane::scaled_plan, gemm_i8.hip; 256 CUs), and the room for its parts of K."""
    import ctypes

    class Plan(ctypes.Structure):
        _fields_ = [("kernel", ctypes.c_int), ("split", ctypes.c_uint32)]

    f = ane_amd.lib()._FuncPtr(("_ZN3ane11scaled_planEjjjb", ane_amd.lib()))
    f.restype, f.argtypes = Plan, [ctypes.c_uint32] * 3 + [ctypes.c_bool]
    rows, few, t64, t128d, t128, t256 = range(6)
    for T, N, K, may, want in ((4, 4096, 14336, True, (rows, 1)), (8, 4096, 14336, True, (t64, 4)), (5, 4096, 8192, False, (rows, 1)),
                               (1, 99, 70000, False, (few, 1)), (16, 4096, 4096, True, (few, 1)), (16, 6144, 4096, True, (t64, 2)), (32, 512, 14336, True, (t64, 8)),
                               (32, 2003, 1777, True, (few, 1)), (100, 39, 7203, True, (t64, 7)), (1400, 6784, 896, True, (t256, 1)), (1879, 19392, 384, True, (t128, 1)), (32, 4096, 4096, True, (t64, 4)), (32, 4096, 14336, True, (t64, 4)),
                               (32, 4096, 14336, False, (few, 1)), (64, 28672, 4096, True, (t64, 1)),
                               (192, 4096, 14336, True, (t128d, 4)), (512, 4096, 14336, True, (t128d, 2)),
                               (512, 4096, 14336, False, (t64, 1)), (16, 65536, 4096, True, (t64, 1)),
                               (128, 65536, 4096, True, (t128, 1)), (512, 6144, 4096, True, (t128d, 1)),
                               (768, 6144, 4096, True, (t128, 1)), (4096, 28672, 4096, True, (t256, 1))):
        p = f(T, N, K, may)
        assert (p.kernel, p.split) == want, (T, N, K)
    for T, N, K in ((32, 4096, 14336), (192, 4095, 14336), (64, 4001, 4096)):
        split = f(T, N, K, True).split
        need = T * (-(-K // 128) * 128) + 4 * T + 1024 + split * T * (-(-N // 4) * 4) * 4
        assert split > 1 and need <= ane_amd.lib().ane_hip_linear_i8_workspace_size(T, N, K) <= need + 1024


def test_a_workspace_covers_fewer_tokens():
    """The size for T tokens is enough for every call of fewer, also where only those split K."""
    import ctypes

    class Plan(ctypes.Structure):
        _fields_ = [("kernel", ctypes.c_int), ("split", ctypes.c_uint32)]

    plan = ane_amd.lib()._FuncPtr(("_ZN3ane11scaled_planEjjjb", ane_amd.lib()))
    plan.restype, plan.argtypes = Plan, [ctypes.c_uint32] * 3 + [ctypes.c_bool]
    size = ane_amd.lib().ane_hip_linear_i8_workspace_size

    def up(x, m):
        return -(-x // m) * m

    for N, K in ((6144, 4096), (4096, 4096), (4096, 14336), (28672, 4096), (64, 14336), (39, 7203), (700, 2048), (1, 131071),
                 (2100, 96)):
        most = 0
        for T in [*range(1, 1200), *range(1200, 17000, 61), 100_000]:
            split = plan(T, N, K, True).split
            need = up(T * up(K, 128), 256) + up(4 * T, 256) + (1024 + split * T * up(N, 4) * 4 if split > 1 else 0)
            most = max(most, need)
            assert size(T, N, K) >= most, (T, N, K)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,most", [(6144, 4096, 65), (4096, 4096, 129), (512, 14336, 700)])
def test_one_workspace_for_batches_of_every_size(ane, N, K, most):
    """A workspace of the largest batch's size through smaller ones, which split K, and back."""
    import torch

    work = ane.linear_i8_workspace(most, N, K)
    x, w, ws, norm, _, res = inputs(most, N, K, seed=14)
    X, W, S, nw, R = dev(x), rows16(w), dev(ws), dev(norm), dev(res)
    want = product(*quantized(x, norm), w, ws, None, res)
    for T in (most, 64, 32, 16, 9, 8, 1, 33, most):
        out = torch.full((T, N), float("nan"), device="cuda")
        ane.linear_i8(X[:T], W, S, out, norm_w=nw, residual=R[:T], workspace=work)
        same(out.cpu().numpy(), want[:T])


@pytest.mark.parametrize("T", [1 << 22, 65535 * 128])
def test_launches_past_32_bits_are_refused(T):
    """Above 16384 values a token takes 1024 threads, and a launch holds fewer than 2^32."""
    assert c_quant(T=T, K=16385, xs=16385, qs=16400) == INVALID
    assert c_linear(T=T, K=16385, xs=16385, wst=16400) == INVALID


@pytest.mark.gpu
def test_denormal_scales_are_rounded_once(ane):
    """max / 127 just below the middle of two denormals, whose quotient in 24 bits is that middle."""
    k = np.array([(1 << 17) + 1, (1 << 17) + 77, 200001, 150003, (1 << 18) - 1, 99, 5], np.float64)
    top = ((127 * k + 63) * 2.0 ** -149).astype(np.float32)
    assert (top.astype(np.float64) == (127 * k + 63) * 2.0 ** -149).all()
    x = np.random.default_rng(6).uniform(-1, 1, (len(k), 300)).astype(np.float32) * top[:, None]
    x[:, 7] = top
    q, s = run_quant(x)
    same(s, (k * 2.0 ** -149).astype(np.float32))
    same(q, quantized(x)[0])
