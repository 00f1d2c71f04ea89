"""m27q_sample_rows against its definition in 64 bits.

A weight is rounded by at most 2^-36 of its size (or of the largest's times 2^-36 where weights are summed to one place), so
a running sum is off by less than 2^-35 of the sum of all weights: a token whose border lies that near its target may be
either neighbour, and every other one is the definition's.  prob: that again, and its rounding to 32 bits."""
import numpy as np
import pytest

from gpu_util import say

SLACK = 2.0 ** -35


def allowed(x, T, k, top_p, min_p, u):
    """{token: probs} of the tokens that a row may give, and their shares of what may be kept."""
    x = x.astype(np.float64)
    nan = np.isnan(x)
    idx = np.lexsort((np.arange(x.size), -np.where(nan, -np.inf, x), nan))
    best = x[idx[0]]
    if not T > 0 or not np.isfinite(best):
        return {int(idx[0]): [1.0]}
    n = x.size
    k = n if k < 1 or k > n else k
    there = np.isfinite(x[idx])  # a banned token has no weight, at an infinite temperature either
    w = np.zeros(x.size)
    w[there] = np.exp((x[idx][there] - best) / np.float64(T))
    run = np.cumsum(w)
    slack = SLACK * run[-1]
    count = [min(k, max(1, int((w[:k] >= min_p).sum()))) if min_p > 0 else k]
    if top_p < 1:
        goal = max(0.0, float(top_p)) * run[k - 1]
        ends = {int(np.searchsorted(run[:k], goal + e)) + 1 for e in (-slack, 0, slack)}
        count = [min(c, max(1, e)) for c in count for e in sorted(ends)]
    u = 0.0 if not u > 0 else min(1.0, float(u))
    out = {}
    for c in set(count):
        total = run[c - 1]
        lo, hi = (min(c - 1, int(np.searchsorted(run[:c], u * total + e))) for e in (-slack, slack))
        for i in range(lo, hi + 1):
            out.setdefault(int(idx[i]), []).append(w[i] / total)
    return out


def logits(rng, rows, n, kind):
    x = (2.2 * rng.standard_normal((rows, n))).astype(np.float32)
    if kind == "peaks":
        for r in range(rows):
            at = rng.choice(n, min(n, 30), replace=False)
            x[r, at] = 6 + 3 * rng.standard_normal(at.size)
    if kind == "flat":
        x *= 1e-3
    if kind == "ties":
        x = np.round(x)
    if kind == "same":
        x[:] = -3.25
    if kind == "far":
        x *= 40
    return x


def run(m, dev, x, T, k, top_p, min_p, u, stream=None, stride=0, t="f32", missing=()):
    import torch
    rows, n = x.shape
    d = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]
    buf = torch.full((rows, n + stride), 99.0, dtype=d, device=dev)
    buf[:, :n] = torch.from_numpy(x).to(dev).to(d)
    arr = lambda v, dt: torch.as_tensor(np.broadcast_to(np.asarray(v, dt), (rows,)).copy(), device=dev)  # noqa: E731
    args = {"temperature": arr(T, np.float32), "top_k": arr(k, np.int32), "top_p": arr(top_p, np.float32), "min_p": arr(min_p, np.float32)}
    for name in missing:
        args[name] = None
    token = torch.full((rows,), -7, dtype=torch.int32, device=dev)
    prob = torch.full((rows,), -7.0, device=dev)
    scratch = torch.full((m.sample_rows_scratch_bytes(rows, n),), 255, dtype=torch.uint8, device=dev)
    uu = arr(u, np.float32)
    torch.cuda.synchronize()
    m.sample_rows(buf[:, :n], uu, token, scratch, prob=prob, stream=stream, **args)
    torch.cuda.synchronize()
    return token.cpu().numpy(), prob.cpu().numpy(), buf[:, :n].float().cpu().numpy()


def check(m, dev, x, T, k, top_p, min_p, u, **how):
    token, prob, seen = run(m, dev, x, T, k, top_p, min_p, u, **how)
    rows = x.shape[0]
    each = lambda v, t: np.broadcast_to(np.asarray(v, t), (rows,))  # noqa: E731
    T, k, top_p, min_p, u = each(T, np.float32), each(k, np.int64), each(top_p, np.float32), each(min_p, np.float32), each(u, np.float32)
    for r in range(rows):
        ok = allowed(seen[r], T[r], int(k[r]), top_p[r], min_p[r], u[r])
        assert int(token[r]) in ok, (r, int(token[r]), list(ok.items())[:4])
        probs = np.array(ok[int(token[r])])
        assert np.any(np.abs(prob[r] - probs) <= (8 * SLACK + 2.0 ** -24) * probs + 2.0 ** -126), (r, prob[r], probs)


RULES = [  # T, top_k, top_p, min_p
    (1.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.05), (1.0, 0, 0.9, 0.0), (1.5, 0, 1.0, 0.02), (1.3, 500, 0.98, 0.0), (0.0, 5, 0.5, 0.1),
    (0.05, 0, 0.99, 0.0), (5.0, 0, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 2, 0.3, 0.9), (30.0, 999, 1.0, 0.0), (0.9, 0, 1e-6, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 63, 1000, 4097, 32003, 248320])
@pytest.mark.parametrize("kind", ["bulk", "peaks", "flat", "ties", "far"])
def test_rows_of_every_rule(m27q, dev, n, kind):
    """A row of each rule in one batch, at several u."""
    say("sample rows", n, kind)
    rng = np.random.default_rng(n)
    x = logits(rng, len(RULES), n, kind)
    T, k, top_p, min_p = (np.array(v) for v in zip(*RULES))
    for u in (0.0, 1e-7, float(rng.random()), float(rng.random()), 1 - 2.0 ** -24):
        check(m27q, dev, x, T, k, top_p, min_p, u)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [8191, 8192, 8193, 32 * 8192, 32 * 8192 + 1, 64 * 8192 + 1, 1000003, 1 << 24])
def test_lengths_around_parts(m27q, dev, n):
    """Parts of 8192 tokens, 32 or 64 of them at a time, up to the longest row."""
    say("sample parts", n)
    rng = np.random.default_rng(n)
    x = logits(rng, 2, n, "peaks")
    x[1, -1] = x[1].max()  # a tie with the last token
    for T, k, top_p, min_p in ((1.0, 0, 0.97, 0.0), (0.8, 40, 1.0, 0.02))[: 1 if n > 1 << 20 else 2]:
        check(m27q, dev, x, T, k, top_p, min_p, (0.3, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 2000, 50000, 248320])
def test_all_the_same(m27q, dev, n):
    """Equal logits: ties go by index, and every cut falls inside them."""
    say("sample same", n)
    x = np.full((len(RULES), n), -3.25, np.float32)
    T, k, top_p, min_p = (np.array(v) for v in zip(*RULES))
    for u in (0.0, 0.37, 0.999):
        check(m27q, dev, x, T, k, top_p, min_p, u)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("n,stride", [(1001, 0), (32003, 5), (151936, 64)])
def test_types_and_strides(m27q, dev, t, n, stride):
    say("sample types", t, n, stride)
    rng = np.random.default_rng(n)
    T, k, top_p, min_p = (np.array(v) for v in zip(*RULES))
    check(m27q, dev, logits(rng, len(RULES), n, "peaks"), T, k, top_p, min_p, rng.random(len(RULES)), t=t, stride=stride)
    check(m27q, dev, logits(rng, 3, n, "bulk"), 0.8, 50, 0.9, 0.0, rng.random(3), stride=stride + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["bulk", "flat", "far", "ties"])
def test_many_equal_logits(m27q, dev, t, kind):
    """16 bits: hundreds of tokens share a value, and several values, or one, a bin."""
    say("sample equal", t, kind)
    rng = np.random.default_rng(len(kind))
    x = logits(rng, 8, 120000, kind)
    if kind == "flat":
        x += np.float32(3)
    for T in (1.0, 0.2, 4.0, 1e-3, float("inf")):
        T = np.full(8, T, np.float32)
        check(m27q, dev, x, T, [0, 0, 0, 700, 30000, 50, 0, 0], [0.9, 0.5, 0.999, 1.0, 1.0, 0.9, 1.0, 1.0],
              [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.1, 0.0], rng.random(8), t=t)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 17, 130, 300])
def test_batches(m27q, dev, rows):
    """A row gives in a batch what it gives alone."""
    say("sample batches", rows)
    rng = np.random.default_rng(rows)
    x = logits(rng, rows, 20011, "peaks")
    rules = [RULES[i % len(RULES)] for i in range(rows)]
    T, k, top_p, min_p = (np.array(v) for v in zip(*rules))
    u = rng.random(rows)
    check(m27q, dev, x, T, k, top_p, min_p, u)
    token, prob, _ = run(m27q, dev, x, T, k, top_p, min_p, u)
    for r in {0, rows // 2, rows - 1}:
        a, b, _ = run(m27q, dev, x[r:r + 1], T[r], k[r], top_p[r], min_p[r], u[r])
        assert a[0] == token[r] and b[0] == prob[r]


@pytest.mark.gpu
def test_missing_arrays(m27q, dev):
    say("sample missing")
    rng = np.random.default_rng(3)
    x = logits(rng, 4, 9000, "peaks")
    u = rng.random(4)
    check(m27q, dev, x, 1.0, 0, 1.0, 0.0, u, missing=("temperature", "top_k", "top_p", "min_p"))
    check(m27q, dev, x, 0.6, 0, 0.9, 0.0, u, missing=("top_k", "min_p"))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [100, 30000])
def test_values_at_the_ends(m27q, dev, n):
    """Banned tokens, rows of nothing else, infinities, NaN, signed zeros, and parameters out of range."""
    say("sample ends", n)
    rng = np.random.default_rng(8)
    nan, inf = float("nan"), float("inf")
    x = logits(rng, 10, n, "peaks")
    x[0, ::2] = -inf
    x[1] = -inf
    x[2, 17] = x[2, 40] = inf
    x[3, ::3] = nan
    x[4] = nan
    x[5] = -inf
    x[5, 9] = -5.0
    x[6] = np.where(np.arange(n) % 2, -0.0, 0.0)
    x[7] = 3.0e38 * np.sign(x[7])
    x[8] *= 1e-40
    x[9, 1:] = nan
    for T, k, top_p, min_p in RULES + [(nan, 0, 1.0, 0.0), (inf, 0, 0.5, 0.0), (1e-30, 0, 0.9, 0.0), (1.0, -4, 1.0, 0.0),
                                       (1.0, 2 ** 31 - 1, 2.0, -1.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1.0, 3.0), (1.0, 0, 0.0, 0.0)]:
        for u in (0.0, 0.6):
            check(m27q, dev, x, T, k, top_p, min_p, u)
    y = logits(rng, 5, n, "peaks")
    for u in ([-1.0, 2.0, nan, 1.0, inf],):
        check(m27q, dev, y, 1.0, 0, 0.9, 0.0, u)
    token, _, _ = run(m27q, dev, y, 1.0, 7, nan, nan, 0.5)
    want, _, _ = run(m27q, dev, y, 1.0, 7, 1.0, 0.0, 0.5)
    assert np.array_equal(token, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 100, 900, 5000, 8193, 20000])
def test_what_lies_behind_a_row_is_not_its(m27q, dev, n):
    """Rows of the lowest number (all tokens masked with it), whose border's logits reach down to -infinity, and temperatures
    that take every number: the values behind a row, as large or larger, are none of its tokens."""
    import torch
    say("sample behind rows", n)
    low, inf = torch.finfo(torch.float32).min, float("inf")
    buf = torch.full((4, n + 9000), low, device=dev)
    buf[2, n:] = 5.0
    buf[3] = 1.0
    buf[3, 0] = -2.0
    x = buf[:, :n]
    seen = x.cpu().numpy()
    token, prob = torch.empty(4, dtype=torch.int32, device=dev), torch.empty(4, device=dev)
    scratch = torch.empty(m27q.sample_rows_scratch_bytes(4, n), dtype=torch.uint8, device=dev)
    f32 = lambda v: torch.full((4,), v, device=dev)  # noqa: E731
    for T in (1.0, 0.01, 3e31, inf):
        for k, top_p, min_p in ((0, 1.0, 0.0), (n // 2 + 1, 1.0, 0.0), (0, 0.6, 0.0), (0, 1.0, 0.3)):
            for u in (0.0, 0.45, 1.0):
                m27q.sample_rows(x, f32(u), token, scratch, f32(T), torch.full((4,), k, dtype=torch.int32, device=dev), f32(top_p),
                                 f32(min_p), prob)
                for r, (t, p) in enumerate(zip(token.tolist(), prob.tolist())):
                    ok = allowed(seen[r], np.float32(T), k, np.float32(top_p), np.float32(min_p), np.float32(u))
                    assert t in ok, (T, k, top_p, min_p, u, r, t, list(ok)[:4])
                    assert any(abs(p - q) <= (8 * SLACK + 2.0 ** -24) * q for q in ok[t]), (T, k, top_p, min_p, u, r, p, ok[t])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2000, 9001, 40000])
@pytest.mark.parametrize("T", [float("inf"), 1e35, 3e31])
def test_largest_numbers_at_the_highest_temperatures(m27q, dev, n, T):
    """Logits at the largest number of 32 bits, a few, half of them or all, where the temperature leaves every token its weight:
    the borders' bin then holds all numbers, up to infinity."""
    say("sample largest", n, T)
    rng = np.random.default_rng(n)
    top = np.float32(np.finfo(np.float32).max)
    x = logits(rng, 6, n, "bulk")
    x[0] = top
    x[1, [3, n // 2, n - 1]] = top
    x[2] = np.where(rng.random(n) < 0.5, top, -top)
    x[3, ::2], x[3, 1::3] = top, -np.inf
    x[4] = np.nextafter(top, np.float32(0)) * (1 - 2.0 ** -22 * rng.integers(0, 2, n))
    x[4, 7] = top
    x[5] = -top
    for k, top_p, min_p in ((0, 1.0, 0.0), (n // 3, 1.0, 0.0), (0, 0.7, 0.0), (0, 1.0, 0.5), (2, 1.0, 0.0), (n // 2, 0.5, 0.1)):
        for u in (0.0, 1e-4, 0.6, 1.0):
            check(m27q, dev, x, T, k, top_p, min_p, u)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1e-3, 1e-5, 8e-6, 3e-6, 1e-6, 1e-9, 1e-11, 1e-13])
def test_temperatures_near_0(m27q, dev, T):
    """Steps between logits from a few octaves to more than numbers of 32 and of 52 bits hold: several sizes of logits, rows with
    two parts of a row far apart, and equal largest ones."""
    say("sample cold", T)
    rng = np.random.default_rng(6)
    x = logits(rng, 6, 20000, "ties") + np.float32(7)
    x[1] *= 1000
    x[2, 8192:] -= 200
    x[3] = np.nextafter(np.float32(10), np.float32(20) * (rng.integers(0, 2, 20000) * 2 - 1)).astype(np.float32)
    x[4, :8192] += 3e6
    x[5] = -x[5] * 1e4
    for top_k, top_p, min_p in ((0, 1.0, 0.0), (50, 0.9, 0.0), (0, 0.6, 0.3)):
        for u in (0.0, 0.4, 0.99):
            check(m27q, dev, x, T, top_k, top_p, min_p, u)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 1, 2, 5])
@pytest.mark.parametrize("T", [1, 2, 3, 40])
def test_smallest_logits_and_temperatures(m27q, dev, T, top):
    """Logits and temperatures of a few times the smallest number of 32 bits: most of a row's tokens stand around the end of
    its bins, where a step of the logits is more than an octave."""
    say("sample smallest", T, top)
    rng = np.random.default_rng(T)
    tiny = np.float32(2.0 ** -149)
    x = np.empty((4, 20000), np.float32)
    x[0] = (-rng.integers(100, 108, 20000) * T) * tiny
    x[1] = (-rng.integers(0, 120, 20000) * T) * tiny
    x[2] = (top - 105 * T) * tiny
    x[3] = top * tiny
    x[:, 9000] = top * tiny
    for k, top_p, min_p in ((0, 1.0, 0.0), (0, 0.9, 0.0), (50, 1.0, 0.0), (0, 1.0, 0.1)):
        for u in (0.0, 0.5, 0.999):
            check(m27q, dev, x, T * tiny, k, top_p, min_p, u)


@pytest.mark.gpu
def test_agrees_with_sampling_of_candidates(m27q, ora, dev):
    """m27q_topk and m27q_sample give the same tokens where u is not beside a border (they sum in 32 bits)."""
    import torch
    say("sample against candidates")
    rng = np.random.default_rng(11)
    x = logits(rng, 1, 248320, "peaks")
    us = np.linspace(0.001, 0.999, 64).astype(np.float32)
    idx, val, tok = (torch.empty(40, dtype=d, device=dev) for d in (torch.int32, torch.float32, torch.int32))
    scratch = torch.empty(m27q.topk_scratch_bytes(248320, 40), dtype=torch.uint8, device=dev)
    m27q.topk(torch.from_numpy(x[0]).to(dev), 40, idx, val, scratch)
    token, _, _ = run(m27q, dev, np.repeat(x, 64, 0), 0.8, 40, 0.95, 0.01, us)
    for u, t in zip(us, token):
        near = [set(allowed(x[0], np.float32(0.8), 40, np.float32(0.95), np.float32(0.01), u + e)) for e in (-1e-5, 1e-5)]
        m27q.sample(idx, val, 40, 0.8, 0.01, 0.95, torch.tensor([u], device=dev), tok)
        assert int(tok[0]) == int(t) or near[0] != near[1], float(u)


@pytest.mark.gpu
def test_shares_of_tokens(m27q, dev):
    """Over a grid of u every token comes up as often as its share says."""
    say("sample shares")
    rng = np.random.default_rng(5)
    row = logits(rng, 1, 700, "peaks")
    n = 4000
    us = (np.arange(n) + 0.5) / n
    token, prob, _ = run(m27q, dev, np.repeat(row, n, 0), 1.2, 0, 0.9, 0.001, us)
    for t in np.unique(token):
        assert abs((token == t).sum() / n - prob[token == t][0]) <= 1.0 / n + 1e-6
    kept = allowed(row[0], np.float32(1.2), 0, np.float32(0.9), np.float32(0.001), 1.0)  # the last of the kept ones
    assert list(kept) == [int(token[-1])]
    assert abs(sum(prob[token == t][0] for t in np.unique(token)) - 1) <= 1e-5  # all of them came up


@pytest.mark.gpu
def test_graph_replays_with_new_rules(m27q, dev):
    import torch
    say("sample graph")
    rng = np.random.default_rng(2)
    n, rows = 70001, 12
    x = torch.zeros(rows, n, device=dev)
    T, top_p, min_p, u = (torch.zeros(rows, device=dev) for _ in range(4))
    k, token, prob = torch.zeros(rows, dtype=torch.int32, device=dev), torch.zeros(rows, dtype=torch.int32, device=dev), torch.zeros(rows, device=dev)
    scratch = torch.empty(m27q.sample_rows_scratch_bytes(rows, n), dtype=torch.uint8, device=dev)
    step = lambda s=None: m27q.sample_rows(x, u, token, scratch, T, k, top_p, min_p, prob, stream=s)  # noqa: E731

    def inputs(i):
        x.copy_(torch.from_numpy(logits(rng, rows, n, ("peaks", "bulk", "flat", "ties")[i % 4])))
        rules = [RULES[(r + i) % len(RULES)] for r in range(rows)]
        for t, v in zip((T, k, top_p, min_p), zip(*rules)):
            t.copy_(torch.tensor(v))
        u.copy_(torch.from_numpy(rng.random(rows)))
    inputs(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(5):
        inputs(i)
        scratch.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        got = token.clone(), prob.clone()
        token.zero_()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        step(side)
        torch.cuda.synchronize()
        assert torch.equal(token, got[0]) and torch.equal(prob, got[1])


@pytest.mark.gpu
def test_rows_past_32_bits(m27q, dev):
    """Rows 2^31 values apart."""
    import torch
    say("sample far rows")
    n = 5000
    pool = torch.empty((2 << 31) + n, dtype=torch.float16, device=dev)
    x = pool.as_strided((3, n), (1 << 31, 1))
    v = torch.from_numpy(logits(np.random.default_rng(1), 3, n, "peaks")).half().to(dev)
    x.copy_(v)
    out = []
    for z in (x, v):
        token = torch.empty(3, dtype=torch.int32, device=dev)
        scratch = torch.empty(m27q.sample_rows_scratch_bytes(3, n), dtype=torch.uint8, device=dev)
        m27q.sample_rows(z, torch.tensor([0.2, 0.5, 0.9], device=dev), token, scratch)
        out.append(token.tolist())
    assert out[0] == out[1]
