"""Attention behind shared prefixes (m27q_attn_shared) against the definition of m27q_attn_paged in 64 bits.

The tolerance is that of the paged attention's tests: a part's weights are rounded relative to themselves, and a factor
that joins parts adds an exponential and a product (2^-22 of the largest score, 2^-24), which those count for each key."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_attn import OUT, WEIGHT, Problem, dtype


class Shared(Problem):
    """`groups`: (first sequence, sequences, shared places) in order; shared places hold one set of keys, values and pages."""

    def __init__(self, m27q, dev, lens, groups, H, Hk, D, page, t="f16", **how):
        super().__init__(m27q, dev, lens, H, Hk, D, page, t, **how)
        self.groups = groups
        for first, count, n in groups:
            most = max([m for _, m in lens[first: first + count]] + [0])
            lead = max(range(first, first + count), key=lambda s: lens[s][1])  # holds all that is shared
            for s in range(first, first + count):
                m = min(n, lens[s][1])
                pages = -(-min(n, most) // page) if n % page else n // page
                whole = min(n // page, pages)
                self.table[s, :whole] = self.table[lead, :whole]
                self.k[s][:m], self.v[s][:m] = self.k[lead][:m], self.v[lead][:m]
        for s in range(len(lens)):
            self.put(s)

    def run(self, out_t, scale, stream=None, fill=0.0, max_q=None, max_kv=None, max_rows=None, max_len=None, first=None, length=None,
            times=None):
        """With every head `times` over, so that the prefix is worth a pass of its own (None: as many as that takes, or
        once where that is more than there can be); all copies give the same."""
        import torch
        d, m = self.dev, self.m
        if times is None:
            times = next((f for f in (1, 4, 16, 64, 256) if self.Hk * f <= 512 and self.H * f <= 1024 and self.pair(
                f, max_q, max_kv, max_rows, max_len, first, length)[3]), 1)
        seqs, x, cache, self.apart = self.pair(times, max_q, max_kv, max_rows, max_len, first, length)
        H = self.H * times
        scratch = torch.full((m.attn_shared_scratch_bytes(seqs, x, H, cache),), 255, dtype=torch.uint8, device=d)
        out = torch.full((self.T, H, self.D), fill, dtype=dtype(out_t), device=d)
        q = self.q.to(d).repeat(1, times, 1)[..., : self.D]
        torch.cuda.synchronize()
        m.attn_shared(seqs, x, cache, q, out, scratch, scale, stream=stream)
        torch.cuda.synchronize()
        out = out.view(self.T, times, self.H, self.D)
        assert times == 1 or torch.equal(out.view(torch.uint8), out[:, :1].expand_as(out).contiguous().view(torch.uint8))
        return out[:, 0].double().cpu().numpy()

    def pair(self, times, max_q, max_kv, max_rows, max_len, first, length):
        """The call's records, and whether its prefix is taken by itself (its scratch tells)."""
        import torch
        d, m = self.dev, self.m
        cache = m.KVCache(self.kc.to(d).repeat(1, times, 1, 1), self.vc.to(d).repeat(1, times, 1, 1))
        seqs = m.Seqs(self.start.to(d), self.kv.to(d), self.table.to(d), self.T, max_q or self.max_q, max_kv or self.max_kv)
        edge = first or [g[0] for g in self.groups] + [self.groups[-1][0] + self.groups[-1][1]]
        length = length or [g[2] for g in self.groups]
        start = self.start.tolist()
        rows = max_rows or max(1, max(start[min(max(b, 0), len(start) - 1)] - start[min(max(a, 0), len(start) - 1)]
                                          for a, b in zip(edge, edge[1:])))
        x = m.Prefixes(torch.tensor(edge, dtype=torch.int32, device=d), torch.tensor(length, dtype=torch.int32, device=d), rows,
                       max_len or max(1, max(length)))
        H = self.H * times
        return seqs, x, cache, m.attn_shared_scratch_bytes(seqs, x, H, cache) != m.attn_scratch_bytes(seqs, H, cache)

    def check(self, out_t, scale, gone=(), **how):
        want, A, es, small = self.want(scale, 0, gone)
        tol = (WEIGHT[self.t, out_t] + es) * A + small + OUT[out_t] * np.abs(want) + 2.0 ** -25 * (out_t == "f16")
        for times in (1, None):
            got = self.run(out_t, scale, times=times, **how)
            assert np.isfinite(got).all()
            assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


CASES = [
    # lens (new, cached), groups (first, sequences, shared), H, Hk, D, page, type, output
    ([(1, 40), (1, 45)], [(0, 2, 32)], 1, 1, 64, 16, "f16", "f32"),
    ([(1, 300), (1, 290), (1, 257), (1, 400)], [(0, 4, 256)], 24, 4, 256, 64, "f16", "f32"),
    ([(1, 300), (0, 290), (1, 257), (1, 400), (1, 5), (1, 120)], [(0, 4, 256), (4, 2, 0)], 12, 2, 128, 32, "bf16", "bf16"),
    ([(5, 700), (3, 650), (8, 648)], [(0, 3, 640)], 6, 1, 256, 16, "bf16", "f32"),              # 96 rows: the kernel of many
    ([(1, 600 + 7 * i) for i in range(40)], [(0, 40, 544)], 8, 2, 64, 16, "f16", "f16"),
    ([(1, 200)] * 3 + [(2, 90)] * 3 + [(1, 33)], [(0, 3, 160), (3, 3, 64)], 4, 2, 64, 32, "bf16", "f32"),  # the last shares nothing
    ([(1, 50), (1, 300), (1, 310)], [(1, 2, 256)], 4, 2, 64, 16, "f16", "f32"),                 # nor does the first here
    ([(70, 470), (33, 433), (130, 530)], [(0, 3, 400)], 6, 2, 128, 16, "f16", "f16"),           # prompts; 16 shared places left over
    ([(150, 450), (1, 310)], [(0, 2, 300)], 2, 1, 64, 128, "bf16", "f32"),                      # 300 is no whole page
    ([(20, 20), (9, 6), (1, 0), (1, 600)], [(0, 4, 512)], 4, 1, 64, 16, "f16", "f32"),          # a prefix past a sequence's own tokens
    ([(40, 100), (50, 90), (3, 200)], [(0, 3, 96)], 2, 2, 128, 16, "bf16", "bf16"),             # rows inside the prefix
    ([(1, 2100), (1, 2050)], [(0, 2, 2048)], 64, 1, 128, 256, "bf16", "f32"),
    ([(1, 64)] * 5, [(0, 5, 64)], 3, 1, 64, 16, "f16", "f32"),                                  # nothing but the prefix
    ([(1, 31), (1, 20)], [(0, 2, 16)], 2, 1, 64, 16, "f16", "f32"),                             # below a tile
    ([(1, 300), (1, 290), (40, 100), (9, 700)], [(0, 2, 256)], 6, 2, 128, 16, "bf16", "f32"),   # few rows share, more do not
    ([(1, 300), (1, 290), (12, 700)], [(0, 2, 256)], 4, 2, 256, 64, "f16", "f16"),              # 16 rows share, 32 do not
    ([(2, 90), (9, 100), (5, 77)], [(0, 3, 64)], 2, 1, 64, 16, "f16", "f32"),                   # 32 rows
    ([(2, 90), (9, 100), (6, 77)], [(0, 3, 64)], 2, 1, 256, 16, "f16", "f32"),                  # 34
    ([(1, 3300)] * 16, [(0, 16, 3200)], 8, 1, 64, 128, "f16", "f32"),                           # 128: one workgroup's
    ([(1, 3300)] * 16 + [(2, 3250)], [(0, 17, 3200)], 8, 1, 64, 128, "bf16", "bf16"),           # 144
    ([(1, 40 + i) for i in range(150)], [(2 * i, 2, 32) for i in range(75)], 2, 1, 64, 16, "f16", "f32"),  # groups past 64
    ([(1, 9000)] * 3, [(0, 3, 64)], 4, 2, 128, 64, "f16", "f32"),                               # mostly their own
    ([(1, 12100), (3, 12050)], [(0, 2, 12032)], 2, 2, 64, 64, "bf16", "f32"),                   # mostly shared
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,groups,H,Hk,D,page,t,out", CASES)
def test_shared_attention_against_definition(m27q, dev, lens, groups, H, Hk, D, page, t, out):
    say("shared", lens[:4], groups, H, Hk, D, page, t, out)
    Shared(m27q, dev, lens, groups, H, Hk, D, page, t).check(out, D ** -0.5)


@pytest.mark.gpu
def test_which_prefixes_are_taken_by_themselves(m27q, dev):
    """Most of the cases above, some of them with their heads as they are: both ways are tested."""
    import torch
    apart = []
    for lens, groups, H, Hk, D, page, t, _ in CASES:
        p = Shared(m27q, dev, lens, groups, H, Hk, D, page, t)
        p.run("f32", 0.1)
        apart.append(p.apart)
    assert sum(apart) >= len(CASES) // 2, apart
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    one = lambda n, places, heads: (m27q.Seqs(i32(*range(n + 1)), i32(*[places + 300] * n), torch.zeros(  # noqa: E731
        n, 1024, dtype=torch.int32, device=dev), n, 1, places + 300), m27q.Prefixes(i32(0, n), i32(places), n, places), heads)
    pages = torch.zeros(1, 4, 64, 256, dtype=torch.float16, device=dev)
    cache = m27q.KVCache(pages, pages)
    for (seqs, x, heads), apart in ((one(4, 2048, 24), False), (one(4, 32768, 24), True), (one(64, 512, 24), False), (one(64, 32768, 24), True),
                                    (one(1, 32768, 24), False)):
        assert (m27q.attn_shared_scratch_bytes(seqs, x, heads, cache) != m27q.attn_scratch_bytes(seqs, heads, cache)) == apart


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.1, 30.0])
def test_scale(m27q, dev, scale):
    say("shared scale", scale)
    Shared(m27q, dev, [(3, 100), (40, 170)], [(0, 2, 64)], 4, 2, 64, 16, "f16", spread=0.5).check("f32", scale)


@pytest.mark.gpu
def test_bounds(m27q, dev):
    """max_len below a len: the rest is each sequence's own; a len of nothing, or below 0; groups over the batch's end."""
    say("shared bounds")
    p = Shared(m27q, dev, [(1, 700), (1, 650), (2, 800)], [(0, 3, 640)], 4, 2, 64, 16)
    for how in (dict(max_len=100), dict(max_len=31), dict(length=[0]), dict(length=[-5]), dict(length=[2 ** 31 - 1]),
                dict(first=[0, 9]), dict(first=[-3, 3]), dict(first=[3, 3]), dict(first=[0, 1, 3], length=[640, 64])):
        if how.get("length") == [2 ** 31 - 1]:
            how["max_len"] = 640
        p.check("f32", 0.125, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,n,H,Hk,D,page", [
    ([(0, 2100), (1, 40)] + [(1, 2100 + 9 * i) for i in range(11)], 2048, 2, 2, 128, 64),  # few rows
    ([(0, 1040), (1, 0), (5, 20)] + [(5, 1030 + i) for i in range(9)], 1024, 2, 2, 128, 32),
    ([(0, 450), (60, 65), (90, 430), (20, 400)], 256, 6, 2, 64, 16)])
def test_tables_that_end_within_the_prefix(m27q, dev, lens, n, H, Hk, D, page):
    """A group's first sequence has left the batch, the next one's tokens end within the prefix: their tables name no page
    that is not theirs."""
    say("shared short tables", lens[:4])
    p = Shared(m27q, dev, lens, [(0, len(lens), n)], H, Hk, D, page)
    for s, (a, m) in enumerate(lens):
        p.table[s, -(-m // page) if a else 0:] = -1
    p.check("f32", 0.125)
    assert p.apart


LOOSE = [
    # lens, groups (first, sequences, shared), H, Hk, D, page, type, output; max_len as large as max_kv
    ([(1, 300), (1, 290), (1, 6000)], [(0, 2, 256)], 6, 2, 256, 64, "f16", "f32"),              # a long one of no group: few rows
    ([(1, 300), (1, 290), (1, 6000)], [(0, 2, 256), (2, 1, 5952)], 6, 2, 256, 64, "f16", "f32"),  # it is a group by itself
    ([(1, 5000), (1, 4990), (1, 20), (1, 33)], [(0, 2, 64), (2, 2, 0)], 4, 1, 128, 16, "bf16", "bf16"),  # long behind little
    ([(5, 400 + i) for i in range(9)] + [(5, 5000)], [(0, 9, 352)], 6, 1, 64, 16, "f16", "f32"),  # many rows
    ([(1, 40)] * 50 + [(1, 3000)], [(0, 50, 32)], 4, 1, 128, 16, "bf16", "f32"),
    ([(70, 470), (33, 433), (130, 4030)], [(0, 2, 384)], 2, 1, 64, 16, "f16", "f16"),           # prompts
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,groups,H,Hk,D,page,t,out", LOOSE)
def test_sequences_longer_than_the_bounds_let_expect(m27q, dev, lens, groups, H, Hk, D, page, t, out):
    """max_len as large as max_kv, as a step that is captured with the largest bounds has it."""
    say("shared loose", lens[-2:], groups, H, Hk, D, page, t, out)
    p = Shared(m27q, dev, lens, groups, H, Hk, D, page, t)
    p.check(out, D ** -0.5, max_len=p.max_kv)
    p.check(out, D ** -0.5, max_len=max(1, p.max_kv - 40), length=[0] * len(groups))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 333), (2, 370)], [(90, 433), (20, 370)]])
def test_pages_that_are_none(m27q, dev, lens):
    """Pages outside the pool, of the prefix and behind it, are left out."""
    say("shared bad pages", lens)
    p = Shared(m27q, dev, lens, [(0, 2, 256)], 4, 2, 128, 16)
    gone = [(s, b) for s in (0, 1) for b in (0, 7)] + [(0, 20), (1, 17)]
    for i, (s, b) in enumerate(gone):
        p.table[s, b] = (-1, 10 ** 6, -2 ** 31, p.kc.shape[0])[i % 4]
    p.check("f32", 0.1, gone=gone)
    p.table[:] = -1
    assert not p.run("f32", 0.1).any()


@pytest.mark.gpu
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("lens", [[(1, 200), (1, 210), (1, 170)], [(60, 200), (1, 230), (30, 190)]])
def test_values_that_are_not_finite(m27q, dev, what, lens):
    """A value of the prefix shows in every row that sees it, one behind it in its own sequence's rows alone."""
    say("shared odd values", what, lens)
    p = Shared(m27q, dev, lens, [(0, 3, 128)], 2, 1, 64, 16)
    clean = p.run("f32", 0.125)
    cols = np.arange(64) != 5
    for s, place, rows in ((0, 100, slice(0, p.T)), (1, lens[1][1] - 1, slice(int(p.start[2]) - 1, int(p.start[2])))):
        kept = [(p.kc.clone(), p.vc.clone())]
        page, slot = p.table[s, place // 16].long(), place % 16
        p.vc[page, 0, slot, 5] = what
        got = p.run("f32", 0.125)
        bad = np.zeros(p.T, bool)
        bad[rows] = True
        if s == 0:  # rows of the first sequence's prompt that stand before the place do not see it
            at = np.concatenate([np.arange(m - a, m) for a, m in lens])
            bad &= at >= place
        assert np.array_equal(got[~bad], clean[~bad])
        assert np.array_equal(got[bad][..., cols], clean[bad][..., cols])
        assert np.isnan(got[bad][..., 5]).all() if np.isnan(what) else (got[bad][..., 5] == what).all()
        p.kc, p.vc = kept[0]


@pytest.mark.gpu
def test_untouched_rows_and_same_results(m27q, dev):
    """Rows of no sequence, past max_q or past max_rows keep what they hold; a run is the same on any stream, and that of the
    paged attention to the order of sums."""
    import torch
    say("shared rows")
    p = Shared(m27q, dev, [(5, 280), (7, 290), (4, 300)], [(0, 2, 256)], 4, 2, 64, 16, q_pad=64)
    p.T += 3
    p.q = torch.cat([p.q, p.q[:3]])
    full = p.run("f32", 0.125, fill=9.0)
    assert (full[16:] == 9).all() and (full[:16] != 9).all()
    assert np.array_equal(full, p.run("f32", 0.125, fill=9.0, stream=torch.cuda.Stream()))
    part = p.run("f32", 0.125, fill=9.0, max_q=6)
    assert (part[11] == 9).all() and np.allclose(np.delete(part, 11, 0), np.delete(full, 11, 0), rtol=0, atol=1e-5)
    part = p.run("f32", 0.125, fill=9.0, max_rows=8)
    assert not p.apart or (part[8:12] == 9).all()
    assert np.allclose(part[:8], full[:8], rtol=0, atol=1e-5)
    assert np.allclose(part[12:], full[12:], rtol=0, atol=1e-5)
    assert np.allclose(Problem.run(p, "f32", 0.125, fill=9.0), full, rtol=0, atol=1e-5)


@pytest.mark.gpu
def test_graph_replays_with_new_groups(m27q, dev):
    """Captured once; each replay finds new lengths, groups, shared places and rows in the same buffers."""
    import torch
    say("shared graph")
    H, Hk, D, page, n = 336, 56, 128, 16, 5
    g = torch.Generator(device=dev).manual_seed(4)
    kc, vc = (torch.randn(200, Hk, page, D, generator=g, device=dev).half() for _ in range(2))
    cache = m27q.KVCache(kc, vc)
    start, kv = torch.arange(n + 1, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)
    table = torch.zeros(n, 40, dtype=torch.int32, device=dev)
    first, length = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    seqs, x = m27q.Seqs(start, kv, table, n, 1, 640), m27q.Prefixes(first, length, n, 512)
    q, out, plain = torch.empty(n, H, D, dtype=torch.float16, device=dev), torch.empty(n, H, D, device=dev), torch.empty(n, H, D, device=dev)
    scratch = torch.empty(m27q.attn_shared_scratch_bytes(seqs, x, H, cache), dtype=torch.uint8, device=dev)
    other = torch.empty(m27q.attn_scratch_bytes(seqs, H, cache), dtype=torch.uint8, device=dev)

    def inputs(i):
        q.normal_(generator=g)
        table.copy_(torch.randperm(200, generator=g, device=dev)[:n * 40].view(n, 40))
        a, b = (0, 2, 5), (1, 1, 4)
        edge = (a, b, (0, 5, 5), (0, 0, 5))[i % 4]
        shared = (160 + 32 * i, 64 * i)
        for j in range(2):
            table[edge[j]:edge[j + 1], :shared[j] // page] = table[edge[j], :shared[j] // page].clone() if edge[j] < n else 0
        first.copy_(torch.tensor(edge, dtype=torch.int32))
        length.copy_(torch.tensor(shared, dtype=torch.int32))
        kv.copy_(torch.tensor([300 + 20 * i, 330, 340 + i, 420, 301], dtype=torch.int32))
    step = lambda: m27q.attn_shared(seqs, x, cache, q, out, scratch, 0.1)  # noqa: E731
    inputs(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):
        inputs(i)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        step()
        m27q.attn_paged(seqs, cache, q, plain, other, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(out, got)
        assert torch.allclose(plain, got, rtol=0, atol=1e-5)


@pytest.mark.gpu
def test_pages_past_32_bits(m27q, dev):
    """Pages 2^31 values apart."""
    import torch
    say("shared far pages")
    D, page, H = 256, 1024, 40
    size = H * page * D
    pool = torch.empty((2 << 31) + 2 * size, dtype=torch.float16, device=dev)
    kc = pool.as_strided((3, H, page, D), (1 << 31, page * D, D, 1))
    vc = pool[size:].as_strided((3, H, page, D), (1 << 31, page * D, D, 1))
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, H, page, D, generator=g).half().to(dev) for _ in range(2))
    kc.copy_(k)
    vc.copy_(v)
    q = torch.randn(2, H, D, generator=g).half().to(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    seqs, x = m27q.Seqs(i32(0, 1, 2), i32(1084, 1064), i32(2, 0, 2, 1).view(2, 2), 2, 1, 1100), m27q.Prefixes(i32(0, 2), i32(1024), 2, 1024)
    outs = []
    for kk, vv in ((kc, vc), (k, v)):
        cache = m27q.KVCache(kk, vv)
        out = torch.empty(2, H, D, device=dev)
        scratch = torch.empty(m27q.attn_shared_scratch_bytes(seqs, x, H, cache), dtype=torch.uint8, device=dev)
        assert scratch.numel() != m27q.attn_scratch_bytes(seqs, H, cache)  # the prefix by itself
        m27q.attn_shared(seqs, x, cache, q, out, scratch, 0.1)
        outs.append(out.cpu())
    assert torch.equal(outs[0], outs[1]) and bool(outs[0].abs().sum() > 0)
