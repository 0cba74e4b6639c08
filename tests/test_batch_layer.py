"""One layer of a batched step through the operators as they are used together:
int8 linear layers, head norms with rotation and append, attention under a rule,
for two prompts, then single tokens, then a second chunk; against the same layer
in 64 bits on whole sequences.

The two differ in the int8 rounding of activations that differ by rounding noise:
a value next to a border goes to either integer, so tolerances are those of such
steps.  A product's input off by e (relative to its token's largest value) moves
at most a share e * 127 * 2 of its integers by one step; with the fp16 cache (2^-11
each in k and v) e is below 2^-9, so at most half of the values of a row move by one
of 127 steps: sqrt(K / 2) steps of about max|x| / 127, against sqrt(K) values of
about max|x| / 4: 0.7 * 4 / 127 = 2.3 % of the result's size, twice over for two
products behind the cache; and for a single value a row's spread of five standard
deviations.
"""
import math

import pytest

import ane_amd
from tests.test_paged import dt, i32


class Layer:
    def __init__(self, hidden, heads, kv, hd, seed):
        import torch

        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(n, k):
            w = torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k)
            s = w.abs().amax(1) / 127
            wide = torch.zeros((n, -(-k // 16) * 16), dtype=torch.int8, device="cuda")  # rows that start on 16 bytes
            wide[:, :k] = torch.round(w / s[:, None])
            return wide[:, :k], s

        self.heads, self.kv, self.hd = heads, kv, hd
        self.qkv, self.o = weights((heads + 2 * kv) * hd, hidden), weights(hidden, heads * hd)
        self.norm = torch.rand(hidden, generator=g, device="cuda") + 0.5
        self.qn, self.kn = (torch.rand(hd, generator=g, device="cuda") + 0.5 for _ in range(2))
        self.freqs = torch.from_numpy(ane_amd.rope_freqs(hd // 2, 10000.0, 4.0, "turns", context=64)[0]).cuda()
        self.slopes = torch.tensor([2.0 ** -(i + 1) for i in range(heads)], device="cuda")
        self.cap, self.window = 15.0, 90

    def step(self, cache, start, x, max_len, seqs=None):
        """x [tokens][hidden] (the residual stream) through the layer, in place."""
        import torch

        T, h = x.shape[0], self.heads
        qkv = torch.empty((T, h + 2 * self.kv, self.hd), device="cuda")
        ane_amd.linear_i8(x, *self.qkv, qkv.view(T, -1), norm_w=self.norm)
        q = torch.empty((T, h, self.hd), device="cuda")
        ane_amd.paged_norm_rope_append(cache, 0, start, qkv[:, :h], qkv[:, h:h + self.kv], qkv[:, h + self.kv:],
                                       ane_amd.Rope(self.freqs, half=True), q, q_norm=self.qn, k_norm=self.kn, seqs=seqs)
        out = torch.empty_like(q)
        ane_amd.attention_prompt(cache, 0, start, q, out, max_len=max_len, seqs=seqs,
                                 rule=ane_amd.AttentionRule(self.cap, self.slopes, self.window))
        ane_amd.linear_i8(out.view(T, -1), *self.o, x, residual=x)

    def whole(self, x):
        """The same for all positions [n][hidden] of one sequence, in 64 bits around the int8 steps."""
        import torch

        def linear(x, w):
            s = x.abs().amax(1, keepdim=True) / 127
            return torch.round(x / s) @ w[0].double().t().contiguous() * s * w[1].double()

        def rms(x, w, eps):
            return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()

        x = x.double()
        n, h, kv, hd = x.shape[0], self.heads, self.kv, self.hd
        qkv = linear(rms(x, self.norm, 1e-5), self.qkv).view(n, h + 2 * kv, hd)
        z = torch.polar(torch.ones(n, 1, hd // 4, dtype=torch.float64, device="cuda"),
                        (torch.arange(n, device="cuda").double()[:, None] * self.freqs)[:, None])

        def turn(y):
            a, b = y[..., :hd // 4], y[..., hd // 4:hd // 2]
            c = torch.complex(a.contiguous(), b.contiguous()) * z
            return torch.cat([c.real, c.imag, y[..., hd // 2:]], -1)

        q, k, v = turn(rms(qkv[:, :h], self.qn, 1e-6)), turn(rms(qkv[:, h:h + kv], self.kn, 1e-6)), qkv[:, h + kv:]
        p = torch.arange(n, device="cuda")
        d = p[:, None] - p[None]
        o = torch.empty_like(q)
        for i in range(h):
            g = i // (h // kv)
            s = torch.tanh(q[:, i] @ k[:, g].t().contiguous() / math.sqrt(hd) / self.cap) * self.cap - float(self.slopes[i]) * d.abs()
            o[:, i] = torch.softmax(s.masked_fill((d < 0) | (d >= self.window), -math.inf), -1) @ v[:, g].contiguous()
        return x + linear(o.reshape(n, -1), self.o)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,heads,kv,hd", [(512, 8, 2, 64), (1000, 4, 4, 128)])
def test_prompts_then_tokens_then_a_chunk(ane, hidden, heads, kv, hd):
    import torch

    layer = Layer(hidden, heads, kv, hd, seed=hidden)
    cache = ane.PagedCache.empty(1, heads, kv, hd, 16, 64, 4, 32)
    served = torch.zeros(4, dtype=torch.int32, device="cuda")
    lens = [0, 0, 0]
    xs = [torch.randn((330, hidden), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda") for i in range(3)]
    outs = [[] for _ in xs]
    # two prompts; a token of each; the third's prompt beside a chunk of the first; single tokens of all, out of order
    for seqs, new in (([0, 1], [200, 37]), ([0, 1], [1, 1]), ([2, 0], [90, 60]), ([2, 0, 1], [1, 1, 1]), ([1, 2, 0], [1, 1, 1])):
        for s, n in zip(seqs, new):
            lens[s] += n
        ane.pages_reserve(cache, i32(seqs), i32([lens[s] for s in seqs]), served)
        x = torch.cat([xs[s][lens[s] - n:lens[s]] for s, n in zip(seqs, new)])
        single = max(new) == 1
        start = [sum(new[:i]) for i in range(len(new) + 1)]
        layer.step(cache, None if single else i32(start), x, max(lens), seqs=i32(seqs))
        for i, s in enumerate(seqs):
            outs[s].append(x[start[i]:start[i + 1]])
        assert bool((served[:len(seqs)] == 1).all())
    for s, n in enumerate(lens):
        got, want = torch.cat(outs[s]).double(), layer.whole(xs[s][:n])
        moved = want - xs[s][:n].double()  # what the layer adds
        err = got - want
        assert float(err.norm() / moved.norm()) < 2 * 0.023
        assert float((err.norm(dim=1) / moved.norm(dim=1)).max()) < 2 * 0.023 * 5
