"""Attention over a paged cache (m27q_attn_paged) against its definition in 64 bits.

Tolerance of an output value, with p the exact weights and A = sum p |v|: the scores are fp32 sums of D exact products
(e_s = (D + 8) 2^-24 scale sum |q k|, the largest of the row's keys, taken twice: in a weight and in the sum of
weights; 2^-22 for exp2 and its argument's rounding relative to the largest score), the weights are rounded (2^-11 F16,
2^-8 BF16; with an F32 output 2^-22 or 2^-23), fp32 sums over n keys ((n + 8) 2^-24), weights below the type's normal range
(2^-30 of the largest value each, F16), and the output's own rounding."""
import numpy as np
import pytest

from gpu_util import say

OUT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
WEIGHT = {("f16", "f16"): 2.0 ** -11, ("bf16", "bf16"): 2.0 ** -8, ("f16", "f32"): 2.0 ** -22, ("bf16", "f32"): 2.0 ** -23}


def dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Problem:
    """Sequences of (new rows, cached tokens) with pages in no order; slots of no token hold NaN."""

    def __init__(self, m27q, dev, lens, H, Hk, D, page, t="f16", seed=0, q_pad=0, spread=1.5):
        import torch
        g = torch.Generator().manual_seed(seed + 7 * D + page)
        self.lens, self.H, self.Hk, self.D, self.page, self.t = lens, H, Hk, D, page, t
        n, T = len(lens), sum(a for a, _ in lens)
        per = max(1, max(-(-m // page) for _, m in lens))
        pages = n * per + 2
        self.table = torch.randperm(pages, generator=g)[: n * per].view(n, per).to(torch.int32)
        self.kc = torch.full((pages, Hk, page, D), float("nan"), dtype=dtype(t))
        self.vc = self.kc.clone()
        self.k, self.v = [], []
        for s, (_, m) in enumerate(lens):
            k, v = (torch.randn(m, Hk, D, generator=g).to(dtype(t)) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            self.put(s)
        buf = torch.randn(T, H, D + q_pad, generator=g)
        self.q = (spread * buf).to(dtype(t))
        self.start = torch.tensor(np.concatenate([[0], np.cumsum([a for a, _ in lens])]), dtype=torch.int32)
        self.kv = torch.tensor([m for _, m in lens], dtype=torch.int32)
        self.T, self.m, self.dev = T, m27q, dev
        self.max_q, self.max_kv = max(1, max(a for a, _ in lens)), max(1, int(self.kv.max()))

    def put(self, s):
        import torch
        j = torch.arange(self.k[s].shape[0])
        p, o = self.table[s, j // self.page].long(), j % self.page
        self.kc[p, :, o], self.vc[p, :, o] = self.k[s], self.v[s]

    def run(self, out_t, scale, window=0, stream=None, fill=0.0, max_q=None, max_kv=None):
        import torch
        d = self.dev
        cache = self.m.KVCache(self.kc.to(d), self.vc.to(d))
        seqs = self.m.Seqs(self.start.to(d), self.kv.to(d), self.table.to(d), self.T, max_q or self.max_q, max_kv or self.max_kv)
        scratch = torch.full((self.m.attn_scratch_bytes(seqs, self.H, cache),), 255, dtype=torch.uint8, device=d)
        out = torch.full((self.T, self.H, self.D), fill, dtype=dtype(out_t), device=d)
        q = self.q.to(d)[..., : self.D]
        torch.cuda.synchronize()
        self.m.attn_paged(seqs, cache, q, out, scratch, scale, window, stream=stream)
        torch.cuda.synchronize()
        return out.double().cpu().numpy()

    def want(self, scale, window=0, gone=()):
        """The definition, and each value's tolerance without the output's rounding as (A-factor, A, n max|v|)."""
        out = np.zeros((self.T, self.H, self.D))
        A, es, small = np.zeros_like(out), np.zeros((self.T, self.H, 1)), np.zeros((self.T, self.H, 1))
        G, t = self.H // self.Hk, 0
        q = self.q.double().numpy()[..., : self.D]
        for s, (a, m) in enumerate(self.lens):
            k, v = self.k[s].double().numpy(), self.v[s].double().numpy()
            j = np.arange(m)
            there = ~np.isin(j // self.page, [p for ss, p in gone if ss == s])
            for i in range(a):
                at = m - a + i
                see = there & (j <= at)
                if window:
                    see &= j > at - window
                if see.any():
                    for h in range(self.H):
                        kk, vv = k[see, h // G], v[see, h // G]
                        x = scale * (kk @ q[t, h])
                        p = np.exp(x - x.max())
                        p /= p.sum()
                        out[t, h] = p @ vv
                        A[t, h] = p @ np.abs(vv)
                        es[t, h] = (2 * (self.D + 8) * 2.0 ** -24 * abs(scale) * (np.abs(kk) @ np.abs(q[t, h])).max()
                                    + 2.0 ** -22 * (1 + np.ptp(x)) + (see.sum() + 8) * 2.0 ** -24)
                        small[t, h] = see.sum() * 2.0 ** -30 * np.abs(vv).max()
                t += 1
        return out, A, es, small

    def check(self, out_t, scale, window=0, gone=(), **how):
        got = self.run(out_t, scale, window, **how)
        want, A, es, small = self.want(scale, window, gone)
        tol = (WEIGHT[self.t, out_t] + es) * A + small + OUT[out_t] * np.abs(want) + 2.0 ** -25 * (out_t == "f16")
        assert np.isfinite(got).all()
        assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


CASES = [
    # lens, H, Hk, D, page, type, output
    ([(1, 1)], 1, 1, 64, 16, "f16", "f16"),
    ([(1, 1021)], 24, 4, 256, 64, "f16", "f32"),
    ([(1, 5), (1, 300), (1, 64), (1, 33)], 8, 2, 128, 16, "bf16", "f32"),
    ([(5, 700), (3, 90)], 6, 1, 256, 32, "bf16", "bf16"),
    ([(16, 16)], 4, 4, 64, 16, "f16", "f32"),
    ([(33, 33), (0, 40), (70, 129), (1, 0)], 6, 2, 128, 16, "f16", "f16"),
    ([(130, 200)], 3, 1, 64, 64, "bf16", "f32"),
    ([(200, 450)], 8, 1, 128, 128, "f16", "f32"),
    ([(65, 321), (129, 129)], 12, 2, 256, 16, "bf16", "bf16"),
    ([(2, 2500)], 32, 1, 64, 256, "f16", "f16"),
    ([(1, 4096)], 64, 1, 128, 64, "bf16", "f32"),
    ([(9, 6)], 2, 1, 64, 16, "f16", "f32"),   # the first rows have no place yet
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,Hk,D,page,t,out", CASES)
def test_attention_against_definition(m27q, dev, lens, H, Hk, D, page, t, out):
    say("attn", lens, H, Hk, D, page, t, out)
    Problem(m27q, dev, lens, H, Hk, D, page, t).check(out, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 5000])
@pytest.mark.parametrize("lens,H,Hk,D,t", [([(1, 700), (1, 20)], 4, 2, 64, "f16"), ([(150, 260)], 2, 1, 128, "bf16"),
                                           ([(40, 300), (7, 9)], 6, 1, 256, "f16")])
def test_window(m27q, dev, window, lens, H, Hk, D, t):
    say("attn window", window, lens)
    Problem(m27q, dev, lens, H, Hk, D, 16, t, seed=window).check("f32", D ** -0.5, window)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0, 30.0])
def test_scale(m27q, dev, scale):
    """No scale, a negative one, one that leaves a single key."""
    say("attn scale", scale)
    Problem(m27q, dev, [(3, 100), (40, 170)], 4, 2, 64, 16, "f16", spread=0.5).check("f32", scale)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 333), (2, 70)], [(90, 333), (20, 70)]])
def test_pages_that_are_none(m27q, dev, lens):
    """Keys on pages outside the pool are left out; a row that has no others gives zeros."""
    say("attn bad pages", lens)
    p = Problem(m27q, dev, lens, 4, 2, 128, 16)
    gone = [(0, 0), (0, 7), (0, 20)] + [(1, i) for i in range(5)]
    for i, (s, b) in enumerate(gone):
        p.table[s, b] = (-1, 10 ** 6, -2 ** 31, p.kc.shape[0])[i % 4]
    p.check("f32", 0.1, gone=gone)
    assert not p.run("f32", 0.1)[lens[0][0]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("lens", [[(4, 200)], [(60, 200)]])
def test_hidden_values_have_no_effect(m27q, dev, t, what, lens):
    """A key or value that is not finite shows in the rows that see it and in no other."""
    say("attn odd values", t, what, lens)
    a, m = lens[0]
    p = Problem(m27q, dev, lens, 2, 1, 64, 16, t)
    clean = p.run("f32", 0.125)
    row = a - 2  # seen by the last two rows alone
    p.v[0][m - 2, 0, 5] = what
    p.put(0)
    got = p.run("f32", 0.125)
    assert np.array_equal(got[:row], clean[:row])
    cols = np.arange(64) != 5
    assert np.array_equal(got[row:][..., cols], clean[row:][..., cols])
    assert np.isnan(got[row:][..., 5]).all() if np.isnan(what) else np.array_equal(got[row:][..., 5], np.full((2, 2), what))
    p.v[0][m - 2, 0, 5] = 0
    p.k[0][m - 2, 0, 5] = float("nan")
    p.put(0)
    got = p.run("f32", 0.125)
    p.k[0][m - 2, 0, 5] = 0
    assert np.array_equal(got[:row], clean[:row])
    assert np.isnan(got[row:]).all()


@pytest.mark.gpu
def test_strided_rows_and_untouched_rows(m27q, dev):
    """Queries out of a wider projection; rows of no sequence and rows past max_q keep what they hold."""
    import torch
    say("attn strides")
    p = Problem(m27q, dev, [(5, 80), (7, 90)], 4, 2, 64, 16, q_pad=64)
    p.check("f16", 0.125)
    p.T += 3
    p.q = torch.cat([p.q, p.q[:3]])
    full = p.run("f32", 0.125, fill=9.0)
    assert (full[12:] == 9).all()
    part = p.run("f32", 0.125, fill=9.0, max_q=6)
    assert (part[11:] == 9).all()
    assert np.allclose(part[:11], full[:11], rtol=0, atol=1e-5)


@pytest.mark.gpu
def test_same_result_every_time_on_any_stream(m27q, dev):
    import torch
    say("attn streams")
    p = Problem(m27q, dev, [(2, 3000), (1, 900)], 12, 2, 128, 32)
    a = p.run("f32", 0.1)
    s = torch.cuda.Stream()
    for _ in range(3):
        assert np.array_equal(p.run("f32", 0.1, stream=s), a)


@pytest.mark.gpu
def test_pages_past_32_bits(m27q, dev):
    """Pages 2^31 values apart."""
    import torch
    say("attn far pages")
    D, page = 64, 16
    pool = torch.empty((3 << 31) + 2 * page * D, dtype=torch.float16, device=dev)
    kc = pool.as_strided((3, 1, page, D), (1 << 31, page * D, D, 1))
    vc = pool[page * D:].as_strided((3, 1, page, D), (1 << 31, page * D, D, 1))
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, 1, page, D, generator=g).half().to(dev) for _ in range(2))
    kc.copy_(k)
    vc.copy_(v)
    q = torch.randn(1, 1, D, generator=g).half().to(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    seqs = m27q.Seqs(i32(0, 1), i32(40), i32(2, 0, 1).view(1, 3), 1, 1, 48)
    outs = []
    for kk, vv in ((kc, vc), (k, v)):
        cache = m27q.KVCache(kk, vv)
        out = torch.empty(1, 1, D, device=dev)
        m27q.attn_paged(seqs, cache, q, out, torch.empty(m27q.attn_scratch_bytes(seqs, 1, cache), dtype=torch.uint8, device=dev), 0.1)
        outs.append(out.cpu())
    assert torch.equal(outs[0], outs[1]) and bool(outs[0].abs().sum() > 0)


@pytest.mark.gpu
def test_graph_replays_with_new_lengths(m27q, dev):
    """Append and attention captured once; each replay finds new lengths, pages and rows in the same buffers."""
    import torch
    say("attn graph")
    H, Hk, D, page, n = 6, 1, 128, 16, 3
    g = torch.Generator(device=dev).manual_seed(4)
    table = torch.randperm(60, generator=g, device=dev).to(torch.int32).view(n, 20)
    kc = torch.zeros(60, Hk, page, D, dtype=torch.float16, device=dev)
    cache = m27q.KVCache(kc, torch.zeros_like(kc))
    start, kv = torch.arange(n + 1, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)
    pos = torch.zeros(n, dtype=torch.int32, device=dev)
    seqs = m27q.Seqs(start, kv, table, n, 1, 320)
    r = m27q.Rope.make(64, 1e6, device=dev)
    q, k, v = torch.empty(n, H, D, device=dev), torch.empty(n, Hk, D, device=dev), torch.empty(n, Hk, D, device=dev)
    qr, out = torch.empty(n, H, D, dtype=torch.float16, device=dev), torch.empty(n, H, D, device=dev)
    scratch = torch.empty(m27q.attn_scratch_bytes(seqs, H, cache), dtype=torch.uint8, device=dev)

    def step():
        m27q.rope_append(r, pos, seqs, cache, q, qr, k, v)
        m27q.attn_paged(seqs, cache, qr, out, scratch, 0.1)

    def inputs(i):
        for x in (q, k, v):
            x.normal_(generator=g)
        kv.copy_(torch.tensor([1 + i, 100 + 40 * i, 300 + i], dtype=torch.int32))
        pos.copy_(kv - 1)
    inputs(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(5):
        inputs(i)
        graph.replay()
        torch.cuda.synchronize()
        got, kept = out.clone(), kc.clone()
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(kc, kept)
