"""The gated delta rule (m27q_delta_rule) against its definition in 64 bits, row by row.

Tolerance: with |k| = 1 and 0 <= beta <= 1 a step's own rounding errors do not grow in later steps (|1 - beta k k^T| <= 1,
e^g <= 1).  A step makes about dk + 64 roundings of 2^-24 of the row's size M (the largest of a state row's norm and its
v over the sequence), with random signs; 8 standard deviations of their sum over L steps are
8 sqrt(L (dk + 64)) 2^-24 M; an output takes |q| = 1 times that and its type's rounding."""
import numpy as np
import pytest

from gpu_util import say

OUT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Problem:
    def __init__(self, m27q, dev, lens, Hk, H, dk, dv, t="f32", seed=0, rate=1.0, slots=None, n_slots=None):
        import torch
        g = torch.Generator().manual_seed(seed + dk + dv + sum(lens))
        self.m, self.dev, self.lens, self.t = m27q, dev, lens, t
        T = sum(lens)
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
        self.q, self.k = (unit(torch.randn(T, Hk, dk, generator=g)).to(dtype(t)) for _ in range(2))
        self.v = torch.randn(T, H, dv, generator=g).to(dtype(t))
        self.g = -rate * torch.nn.functional.softplus(torch.randn(T, H, generator=g) - 3)
        self.beta = torch.sigmoid(torch.randn(T, H, generator=g))
        self.slots, self.n_slots = slots, n_slots or len(lens)
        self.state = torch.randn(self.n_slots, H, dv, dk, generator=g) * 0.3
        self.start = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32)

    def run(self, head_map=0, state=True, state_out="new", stream=None, max_len=None):
        import torch
        d, (T, H, dv), dk = self.dev, self.v.shape, self.k.shape[2]
        st = self.state.to(d) if state else None
        so = {"new": torch.full_like(self.state, 5.0).to(d), "same": st, None: None}[state_out]
        out = torch.full((T, H, dv), 3.0, dtype=dtype(self.t), device=d)
        most = max_len or max(1, max(self.lens))
        scratch = torch.full((self.m.delta_scratch_bytes(len(self.lens), T, most, H, dk, dv),), 255, dtype=torch.uint8, device=d)
        args = [x.to(d) for x in (self.start, self.q, self.k, self.v, self.g, self.beta)]
        slots = None if self.slots is None else torch.tensor(self.slots, dtype=torch.int32, device=d)
        torch.cuda.synchronize()
        self.m.delta_rule(*args, st, so, out, scratch, dk ** -0.5, most, slots=slots, head_map=head_map, stream=stream)
        torch.cuda.synchronize()
        return out.double().cpu().numpy(), None if so is None else so.double().cpu().numpy()

    def want(self, head_map=0, state=True):
        """Outputs, final states, and each row's size M ([T, H, dv] and [n, H, dv])."""
        q, k, v, g, b = (x.double().numpy() for x in (self.q, self.k, self.v, self.g, self.beta))
        T, H, dv = v.shape
        Hk, dk = k.shape[1:]
        heads = np.arange(H) % Hk if head_map else np.arange(H) // (H // Hk)
        out, size, ends, sizes, t = np.zeros((T, H, dv)), np.zeros((T, H, dv)), [], [], 0
        for s, n in enumerate(self.lens):
            slot = s if self.slots is None else self.slots[s]
            S = np.zeros((H, dv, dk))
            if state and 0 <= slot < self.n_slots:
                S = self.state[slot].double().numpy().copy()
            M = np.linalg.norm(S, axis=-1)
            for _ in range(n):
                kk, qq = k[t, heads], q[t, heads]
                S = S * np.exp(g[t])[:, None, None]
                u = b[t][:, None] * (v[t] - np.einsum("hvk,hk->hv", S, kk))
                S = S + u[..., None] * kk[:, None]
                out[t] = dk ** -0.5 * np.einsum("hvk,hk->hv", S, qq)
                M = np.maximum(np.maximum(M, np.linalg.norm(S, axis=-1)), np.abs(v[t]))
                size[t] = M
                t += 1
            ends.append(S)
            sizes.append(M)
        return out, ends, size, sizes

    def check(self, **how):
        got, state = self.run(**how)
        want, ends, size, sizes = self.want(how.get("head_map", 0), how.get("state", True))
        dk = self.k.shape[2]
        step = lambda n: 8 * np.sqrt(max(n, 1) * (dk + 64)) * 2.0 ** -24  # noqa: E731
        t = 0
        for s, n in enumerate(self.lens):
            tol = step(n) * size[t: t + n] * dk ** -0.5 * 1.01 + OUT[self.t] * np.abs(want[t: t + n]) + 2.0 ** -25 * (self.t == "f16")
            assert np.all(np.abs(got[t: t + n] - want[t: t + n]) <= tol), (s, np.max(np.abs(got[t: t + n] - want[t: t + n]) / tol))
            slot = s if self.slots is None else self.slots[s]
            if state is not None and 0 <= slot < self.n_slots:
                d = np.abs(state[slot] - ends[s])
                assert np.all(d <= step(n) * sizes[s][..., None]), (s, np.max(d / (step(n) * sizes[s][..., None])))
            t += n
        return state


CASES = [
    # lens, k heads, heads, dk, dv, type
    ([1], 1, 1, 64, 16, "f32"), ([1], 16, 48, 128, 128, "f32"), ([5, 1, 0, 16], 2, 6, 128, 64, "f32"),
    ([1] * 9, 4, 4, 64, 64, "bf16"), ([7, 3], 1, 3, 128, 256, "f16"), ([63], 2, 4, 128, 128, "f32"),
    ([64], 2, 2, 64, 32, "f32"), ([65, 1, 0, 130], 2, 4, 128, 48, "f32"), ([300, 17], 1, 2, 128, 128, "bf16"),
    ([129, 64], 2, 2, 64, 80, "f16"), ([513], 1, 3, 128, 96, "f32"), ([1000], 1, 1, 64, 64, "f32"),
    ([40, 33, 100], 3, 3, 64, 256, "f32"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Hk,H,dk,dv,t", CASES)
def test_delta_against_definition(m27q, dev, lens, Hk, H, dk, dv, t):
    say("delta", lens, Hk, H, dk, dv, t)
    Problem(m27q, dev, lens, Hk, H, dk, dv, t).check()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[3, 2], [150, 70]])
@pytest.mark.parametrize("rate", [0.0, 20.0, 1000.0])
def test_decays(m27q, dev, lens, rate):
    """No decay at all, decays to e^-20 a row, and to zero."""
    say("delta decays", lens, rate)
    Problem(m27q, dev, lens, 2, 4, 128, 64, rate=rate).check()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[6], [200]])
def test_cleared_states(m27q, dev, lens):
    """g = -inf forgets what was before; the row's own part stays."""
    say("delta cleared", lens)
    p = Problem(m27q, dev, lens, 1, 2, 128, 32)
    for t in (0, lens[0] // 2, lens[0] - 1):
        p.g[t, 0] = -float("inf")
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[4, 9], [90, 140]])
def test_alike_keys(m27q, dev, lens):
    """Every key the same: the triangular system at its worst (all off-diagonal products 1)."""
    say("delta alike keys", lens)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32, rate=0.1)
    p.k[:] = p.k[0]
    p.beta[:] = 1.0
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[2, 3, 1], [70, 64, 129]])
def test_head_order_slots_and_state_buffers(m27q, dev, lens):
    say("delta slots", lens)
    p = Problem(m27q, dev, lens, 2, 6, 64, 32)
    p.check(head_map=1)
    p = Problem(m27q, dev, lens, 2, 4, 64, 32, slots=[4, -1, 0], n_slots=5)
    before = p.state.double().numpy()
    state = p.check()
    assert (state[1:4] == 5).all()  # slots of nobody are not written
    state = p.check(state_out="same")
    assert np.array_equal(state[1:4], before[1:4])
    p.check(state=False)
    p.check(state_out=None)
    p.slots = [7, 2 ** 31 - 1, 3]
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[3, 0], [100, 0]])
def test_empty_sequences_keep_their_state(m27q, dev, lens, t):
    say("delta empty", lens, t)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32, t)
    state = p.check()
    assert np.array_equal(state[1], p.state[1].double().numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[5, 6], [100, 130]])
def test_strided_rows_and_odd_values(m27q, dev, lens):
    """q, k and v as parts of one projection, outputs heads first; a NaN stays in its sequence and head."""
    import torch
    say("delta strides", lens)
    p = Problem(m27q, dev, lens, 2, 2, 64, 32)
    a, sa = p.run()
    T = sum(lens)
    wide = torch.cat([p.q.view(T, -1), p.k.view(T, -1), p.v.view(T, -1)], 1).to(dev)
    q, k, v = wide[:, :128].view(T, 2, 64), wide[:, 128:256].view(T, 2, 64), wide[:, 256:].view(T, 2, 32)
    out, so = torch.empty(2, T, 32, device=dev).transpose(0, 1), torch.empty_like(p.state).to(dev)
    scratch = torch.empty(m27q.delta_scratch_bytes(2, T, max(lens), 2, 64, 32), dtype=torch.uint8, device=dev)
    m27q.delta_rule(p.start.to(dev), q, k, v, p.g.to(dev), p.beta.to(dev), p.state.to(dev), so, out, scratch, 64 ** -0.5, max(lens))
    assert np.array_equal(out.double().cpu().numpy(), a) and np.array_equal(so.double().cpu().numpy(), sa)
    p.v[2, 1, 7] = float("nan")
    b, sb = p.run()
    assert np.array_equal(b[:, 0], a[:, 0]) and np.array_equal(b[lens[0]:], a[lens[0]:]) and np.isnan(b[2: lens[0], 1, 7]).all()
    assert np.array_equal(sb[1], sa[1]) and np.array_equal(sb[0, 0], sa[0, 0])


@pytest.mark.gpu
def test_rows_one_by_one_give_the_whole(m27q, dev):
    """A prompt in one call and then token by token, states in place, against all of it at once."""
    import torch
    say("delta stepwise")
    L, n = 150, 12
    p = Problem(m27q, dev, [L], 2, 4, 128, 64)
    whole, end = p.run()
    d = [x.to(dev) for x in (p.q, p.k, p.v, p.g, p.beta)]
    st = p.state.to(dev)
    outs = []
    for a, b in [(0, L - n)] + [(i, i + 1) for i in range(L - n, L)]:
        out = torch.empty(b - a, 4, 64, device=dev)
        start = torch.tensor([0, b - a], dtype=torch.int32, device=dev)
        scratch = torch.empty(m27q.delta_scratch_bytes(1, b - a, b - a, 4, 128, 64), dtype=torch.uint8, device=dev)
        m27q.delta_rule(start, *[x[a:b].contiguous() for x in d], st, st, out, scratch, 128 ** -0.5, b - a)
        outs.append(out.cpu())
    tol = 16 * np.sqrt(L * 192) * 2.0 ** -24 * 5
    assert np.abs(torch.cat(outs).double().numpy() - whole).max() <= tol * 128 ** -0.5
    assert np.abs(st.double().cpu().numpy() - end).max() <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1, 1, 1], [200, 60, 90]])
def test_same_result_every_time_on_any_stream_and_in_a_graph(m27q, dev, lens):
    import torch
    say("delta streams", lens)
    p = Problem(m27q, dev, lens, 2, 4, 128, 64)
    a, sa = p.run()
    s = torch.cuda.Stream()
    for _ in range(3):
        b, sb = p.run(stream=s)
        assert np.array_equal(a, b) and np.array_equal(sa, sb)
    T = sum(lens)
    args = [x.to(dev) for x in (p.start, p.q, p.k, p.v, p.g, p.beta)]
    st, so, out = p.state.to(dev), torch.empty_like(p.state).to(dev), torch.empty(T, 4, 64, device=dev)
    scratch = torch.empty(m27q.delta_scratch_bytes(3, T, max(lens), 4, 128, 64), dtype=torch.uint8, device=dev)
    call = lambda: m27q.delta_rule(*args, st, so, out, scratch, 128 ** -0.5, max(lens))  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        args[3].mul_(0.9)
        st.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        b, sb = out.clone(), so.clone()
        out.zero_()
        so.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(b, out) and torch.equal(sb, so)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("lens,row", [([9], 4), ([150], 0), ([150], 70), ([70, 200], 133), ([64], 63)])
@pytest.mark.parametrize("where", ["v", "k", "q", "g", "beta", "state"])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_values_that_are_not_finite(m27q, dev, lens, row, where, what, t):
    """They show in the rows, heads and values that the definition carries them to, and nowhere before."""
    say("delta odd values", lens, row, where, what, t)
    p = Problem(m27q, dev, lens, 1, 2, 64, 48, t)
    x = getattr(p, where)
    if where == "state":
        x[-1, 1, 17, 3] = what
    elif where in ("g", "beta"):
        x[row, 1] = what
    else:
        x[row, x.shape[1] - 1, 5] = what
    got, state = p.run()
    with np.errstate(all="ignore"):
        want, ends, size, sizes = p.want()
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    ok, at = np.isfinite(want), 0
    for s, n in enumerate(lens):
        rows = slice(at, at + n)
        tol = 8 * np.sqrt(max(n, 1) * 128) * 2.0 ** -24 * 64 ** -0.5 * 1.01 * np.where(np.isfinite(size[rows]), size[rows], 0) \
            + OUT[t] * np.abs(np.where(ok[rows], want[rows], 0))
        assert np.all(np.abs(got[rows] - want[rows])[ok[rows]] <= tol[ok[rows]])
        fine = np.isfinite(ends[s])
        assert np.array_equal(np.isfinite(state[s]), fine)
        tol = 8 * np.sqrt(max(n, 1) * 128) * 2.0 ** -24 * np.where(np.isfinite(sizes[s]), sizes[s], np.inf)[..., None]
        assert np.all((np.abs(state[s] - ends[s]) <= tol)[fine])
        at += n


SIXTEENS = [
    # lens, k heads, heads, dk, dv, type: 8 to 64 rows, and more of them where there are many sequences
    ([8], 1, 1, 64, 16, "f32"), ([16], 16, 48, 128, 128, "bf16"), ([17, 1, 0, 31], 2, 6, 128, 80, "f32"),
    ([33, 48], 1, 3, 64, 256, "f16"), ([64, 50, 63], 4, 4, 128, 128, "f32"), ([32], 2, 2, 64, 48, "bf16"),
    ([20] * 7 + [130, 0, 75], 4, 8, 128, 256, "f32"), ([100] * 9, 8, 24, 64, 128, "f16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Hk,H,dk,dv,t", SIXTEENS)
def test_sixteen_rows_at_a_time(m27q, dev, lens, Hk, H, dk, dv, t):
    say("delta sixteens", lens, Hk, H, dk, dv, t)
    Problem(m27q, dev, lens, Hk, H, dk, dv, t).check()


@pytest.mark.gpu
@pytest.mark.parametrize("rate", [0.0, 20.0, 1000.0])
@pytest.mark.parametrize("head_map", [0, 1])
def test_sixteens_decays_slots_and_head_order(m27q, dev, rate, head_map):
    say("delta sixteens", rate, head_map)
    p = Problem(m27q, dev, [20, 9, 35], 2, 6, 128, 64, rate=rate, slots=[3, 0, -1], n_slots=5)
    p.check(head_map=head_map)
    p.check(head_map=head_map, state_out="same")
    p.check(head_map=head_map, state=False)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[14, 49], [64]])
def test_sixteens_alike_keys_and_cleared_states(m27q, dev, lens):
    say("delta sixteens alike", lens)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32, rate=0.1)
    p.k[:] = p.k[0]
    p.beta[:] = 1.0
    p.check()
    for t in (0, 5, sum(lens) - 1):
        p.g[t, 0] = -float("inf")
    p.check()


@pytest.mark.gpu
def test_sixteens_past_what_the_products_hold(m27q, dev):
    """Values near the largest fp32 one (whose 16-bit parts overflow) and growth that overflows on the way."""
    say("delta sixteens, large")
    p = Problem(m27q, dev, [40], 1, 2, 64, 32)
    p.v[21, 1, 3] = 3.4e38
    p.g[30, 0] = 60.0
    p.g[33, 0] = 40.0
    got, _ = p.run()
    with np.errstate(all="ignore"):
        want, _, _, _ = p.want()
        want32 = np.abs(want) < 2.0 ** 127
    tol = 8 * np.sqrt(40 * 128) * 2.0 ** -24 * 64 ** -0.5
    for h, rows in ((0, slice(0, 30)), (1, slice(0, 21))):
        assert np.all(np.abs(got[rows, h] - want[rows, h]) <= tol * 5)  # states of norm 5 at most before
    assert np.all(np.isfinite(got[:33]) | ~want32[:33])
