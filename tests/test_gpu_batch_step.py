"""A served batch's step as it is used: residual and norm into codes, products, rotary positions with the paged write,
attention behind a shared prefix, norm, head, a token for each sequence.  Beside the same step without these
operators, and captured and replayed.

Tolerances.  The two steps differ by summation orders, which move an activation across a rounding to its int8 code (1 / 254
of its group's largest): a relative difference (in norm) of 1 / 254 would take all of them.  Tokens are compared where
the logits of both steps give the same one."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_sample_rows import SLACK, allowed

D, ROT, PAGE, HIDDEN, VOCAB = 64, 32, 16, 256, 1000


def q8_0(rng, rows, cols):
    w = rng.standard_normal((rows, cols // 32, 32)) / np.sqrt(cols)
    d = (np.abs(w).max(-1, keepdims=True) / 127).astype(np.float16)
    codes = np.round(w / d.astype(np.float64)).clip(-127, 127).astype(np.int8)
    return np.concatenate([d.view(np.uint8), codes.view(np.uint8)], axis=-1).reshape(-1)


class Step:
    def __init__(self, m, dev, n, prefix, H=6, HK=1, seed=0):
        import torch
        self.H, self.HK = H, HK
        self.m, self.n, self.dev, self.prefix = m, n, dev, prefix
        rng = np.random.default_rng(seed)
        weight = lambda rows, cols=HIDDEN: m.Weight.upload(q8_0(rng, rows, cols), m.Q8_0, cols // 32, rows, device=dev)  # noqa: E731
        self.qkv, self.o, self.head = [weight(H * D), weight(HK * D), weight(HK * D)], weight(HIDDEN, H * D), weight(VOCAB)
        g = torch.Generator(device=dev).manual_seed(seed)
        self.g = g
        rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
        self.norms = [1 + 0.1 * rand(HIDDEN) for _ in range(2)]
        pages = prefix // PAGE + 4 * n
        self.cache = m.KVCache(rand(pages, HK, PAGE, D).bfloat16(), rand(pages, HK, PAGE, D).bfloat16())
        own = torch.arange(4 * n, device=dev).view(n, 4) + prefix // PAGE
        self.table = torch.cat([torch.arange(prefix // PAGE, device=dev).expand(n, -1), own], 1).to(torch.int32).contiguous()
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        self.start, self.kv, self.pos = ints(range(n + 1)), ints([prefix + 1] * n), ints([prefix] * n)
        self.seqs = m.Seqs(self.start, self.kv, self.table, n, 1, prefix + 4 * PAGE)
        self.prefixes = m.Prefixes(ints([0, n]), ints([prefix]), n, prefix)
        self.rope = m.Rope.make(ROT, 1e4, device=dev)
        self.x, self.res = rand(n, HIDDEN), rand(n, HIDDEN)
        self.u, self.T = torch.zeros(n, device=dev), torch.linspace(0.0, 1.5, n, device=dev)
        self.top_k = ints([5 * (i % 5) for i in range(n)])
        e = lambda *s, **k: torch.empty(*s, device=dev, **k)  # noqa: E731
        self.h, self.h2, self.y, self.act, self.act2 = e(n, HIDDEN), e(n, HIDDEN), e(n, HIDDEN), m.Act(n, HIDDEN, dev), m.Act(n, H * D, dev)
        self.q, self.k, self.v, self.turned = e(n, H, D), e(n, HK, D), e(n, HK, D), e(n, H, D, dtype=torch.bfloat16)
        self.out, self.logits = e(n, H, D), e(n, VOCAB)
        self.token, self.prob = torch.zeros(n, dtype=torch.int32, device=dev), e(n)
        self.scratch = e(m.attn_shared_scratch_bytes(self.seqs, self.prefixes, H, self.cache), dtype=torch.uint8)
        self.apart = self.scratch.numel() != m.attn_scratch_bytes(self.seqs, H, self.cache)  # the prefix in a pass of its own
        self.plain = e(m.attn_scratch_bytes(self.seqs, H, self.cache), dtype=torch.uint8)
        self.pick = e(m.sample_rows_scratch_bytes(n, VOCAB), dtype=torch.uint8)

    def inputs(self, i):
        self.x.normal_(generator=self.g)
        self.res.normal_(generator=self.g)
        self.u.uniform_(generator=self.g)
        self.kv.fill_(self.prefix + 1 + i)
        self.pos.fill_(self.prefix + i)

    def products(self, act, weights, outs):
        self.m.matmul_q8_multi(weights, act, [o.view(self.n, -1) for o in outs])

    def run(self):
        m = self.m
        m.rms_norm(self.x, self.norms[0], 1e-6, add=self.res, sum=self.h, act=self.act)
        self.products(self.act, self.qkv, [self.q, self.k, self.v])
        m.rope_append(self.rope, self.pos, self.seqs, self.cache, self.q, self.turned, self.k, self.v)
        m.attn_shared(self.seqs, self.prefixes, self.cache, self.turned, self.out, self.scratch, D ** -0.5)
        m.quant_act(self.out, self.act2)
        m.matmul_q8(self.o, self.act2, self.y)
        m.rms_norm(self.y, self.norms[1], 1e-6, add=self.h, sum=self.h2, act=self.act)
        self.products(self.act, [self.head], [self.logits])
        m.sample_rows(self.logits, self.u, self.token, self.pick, self.T, self.top_k, prob=self.prob)

    def without(self):
        """The same step by torch's norm, the paged attention, and candidates one row at a time: logits and tokens."""
        import torch
        m, n, H = self.m, self.n, self.H
        norm = lambda x, w: x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
        h = self.x + self.res
        act, act2 = m.Act(n, HIDDEN, self.dev), m.Act(n, H * D, self.dev)
        q, k, v, turned, out, y, logits = (torch.empty_like(t) for t in (self.q, self.k, self.v, self.turned, self.out, self.y, self.logits))
        m.quant_act(norm(h, self.norms[0]), act)
        self.products(act, self.qkv, [q, k, v])
        m.rope_append(self.rope, self.pos, self.seqs, self.cache, q, turned, k, v)
        m.attn_paged(self.seqs, self.cache, turned, out, self.plain, D ** -0.5)
        m.quant_act(out, act2)
        m.matmul_q8(self.o, act2, y)
        m.quant_act(norm(h + y, self.norms[1]), act)
        self.products(act, [self.head], [logits])
        return logits


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(9, 160), (40, 4096, 32, 8)])
def test_step_beside_the_one_without(m27q, dev, size):
    import torch
    say("batch step")
    s = Step(m27q, dev, *size)
    for i in range(4):
        s.inputs(i)
        s.run()
        logits = s.without()
        torch.cuda.synchronize()
        assert float((s.logits - logits).norm() / logits.norm()) < 1 / 254
        # the tokens of those logits, row by row from the candidates
        scratch = torch.empty(m27q.topk_scratch_bytes(VOCAB, 64), dtype=torch.uint8, device=dev)
        idx, val = torch.empty(64, dtype=torch.int32, device=dev), torch.empty(64, device=dev)
        tok = torch.empty(1, dtype=torch.int32, device=dev)
        for r in range(s.n):
            k = int(s.top_k[r]) or 64
            m27q.topk(s.logits[r], k, idx, val, scratch)
            if float(s.T[r]) <= 0:
                assert int(s.token[r]) == int(idx[0]) and float(s.prob[r]) == 1
            elif int(s.top_k[r]):
                near = []
                for e in (-1e-4, 0, 1e-4):
                    m27q.sample(idx, val, k, float(s.T[r]), 0.0, 1.0, (s.u[r:r + 1] + e).clamp(0, 1), tok)
                    near.append(int(tok[0]))
                assert int(s.token[r]) in near
            else:
                assert 0 <= int(s.token[r]) < VOCAB and 0 < float(s.prob[r]) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(9, 160), (40, 4096, 32, 8)])
def test_tokens_of_a_step_against_the_definition(m27q, dev, size):
    """Every row's token and share, those without a number of candidates too, from the step's own logits."""
    import torch
    say("batch step tokens", size)
    s = Step(m27q, dev, *size, seed=1)
    for i in range(3):
        s.inputs(i)
        s.run()
        torch.cuda.synchronize()
        logits, T, u = s.logits.cpu().numpy(), s.T.cpu().numpy(), s.u.cpu().numpy()
        for r in range(s.n):
            ok = allowed(logits[r], T[r], int(s.top_k[r]), np.float32(1), np.float32(0), u[r])
            token, prob = int(s.token[r]), float(s.prob[r])
            assert token in ok, (r, token, list(ok)[:4])
            assert any(abs(prob - p) <= (8 * SLACK + 2.0 ** -24) * p + 2.0 ** -126 for p in ok[token]), (r, prob, ok[token])


@pytest.mark.gpu
@pytest.mark.parametrize("size,apart", [((9, 160), False), ((40, 4096, 32, 8), True), ((5, 3200, 24, 12), True)])
def test_step_captured_and_replayed(m27q, dev, size, apart):
    import torch
    say("batch step graph")
    s = Step(m27q, dev, *size, seed=3)
    assert s.apart == apart
    s.inputs(0)
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for i in range(5):
        s.inputs(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (s.logits, s.token, s.prob, s.cache.k, s.h2)]
        s.token.zero_()
        s.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (s.logits, s.token, s.prob, s.cache.k, s.h2)))
        assert torch.isfinite(s.logits).all()


@pytest.mark.gpu
def test_two_calls_on_two_streams(m27q, dev):
    """Two batches at once, each with scratch of its own."""
    import torch
    say("batch step streams")
    steps = [Step(m27q, dev, 40, 4096, 32, 8, seed=i) for i in (5, 6)]
    assert all(s.apart for s in steps)
    for i, s in enumerate(steps):
        s.inputs(i)
    want = []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        want.append((s.logits.clone(), s.token.clone()))
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.run()
    torch.cuda.synchronize()
    for s, (logits, token) in zip(steps, want):
        assert torch.equal(s.logits, logits) and torch.equal(s.token, token)
