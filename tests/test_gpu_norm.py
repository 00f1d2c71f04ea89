"""m27q_rms_norm against its definition in 64 bits.

Tolerances.  h: one fp32 addition (2^-24 of it) and the output's rounding.  y: h's 2^-24; of the squares' sum at most
dim / 64 + 24 roundings one after another (a thread's own, the lanes' and waves'), all terms positive, halved by the root;
mean, eps, root and quotient 2^-24 each, two products: (dim / 128 + 12 + 6) 2^-24 of |y|, and the output's rounding (2^-25
absolute more for float16's subnormal values).  Codes: half a step d, and y's error; d is the largest |y| of 32 over 127."""
import numpy as np
import pytest

from gpu_util import say

ROUND = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def make(dev, tokens, heads, dim, t, seed=0, pad=0, off=0, spread=3.0):
    """[tokens, heads, dim] values out of a wider buffer, `off` values into it."""
    import torch
    g = torch.Generator().manual_seed(seed + 31 * dim + tokens)
    buf = (spread * torch.randn(tokens * heads * (dim + pad) + off + 8, generator=g)).to(dtype(t)).to(dev)
    return buf[off:off + tokens * heads * (dim + pad)].view(tokens, heads, dim + pad)[..., :dim]


def want(x, add, weight, eps):
    x = x.double().cpu().numpy()
    h = x if add is None else x + add.double().cpu().numpy()
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return h, y if weight is None else y * weight.double().cpu().numpy()


def tol(y, dim):
    return (dim / 128 + 18) * 2.0 ** -24 * np.abs(y)


def check(m, dev, tokens, heads, dim, types, eps=1e-6, codes=False, weighted=True, seed=0, **how):
    import torch
    tx, ta, ts, to = types
    x = make(dev, tokens, heads, dim, tx, seed, **how)
    add = None if ta is None else make(dev, tokens, heads, dim, ta, seed + 1, **how)
    w = (1 + 0.3 * torch.randn(dim, generator=torch.Generator().manual_seed(seed))).to(dev) if weighted else None
    total = None if ts is None else make(dev, tokens, heads, dim, ts, **how)
    out = None if to is None else make(dev, tokens, heads, dim, to, **how)
    act = m.Act(tokens, heads * dim, dev) if codes else None
    m.rms_norm(x, w, eps, add=add, sum=total, out=out, act=act)
    torch.cuda.synchronize()
    h, y = want(x, add, w, eps)
    for got, v, t, extra in ((total, h, ts, 2.0 ** -24 * np.abs(h)), (out, y, to, tol(y, dim))):
        if got is not None:
            err = np.abs(got.double().cpu().numpy() - v)
            assert np.all(err <= extra + ROUND[t] * np.abs(v) * (1 + 2.0 ** -7) + TINY[t]), float((err / np.abs(v)).max())
    if codes:
        c, d, s = (a.cpu().numpy() for a in act.parts())
        c, y = c.reshape(-1, 32).astype(np.int64), y.reshape(-1, 32)
        d = d.reshape(-1, 1).astype(np.float64)
        top = np.abs(y).max(-1, keepdims=True)
        assert np.all(np.abs(d * 127 - top) <= tol(top, dim) + 2.0 ** -23 * top)
        assert np.all(np.abs(c * d - y) <= d * (0.5 + 2.0 ** -15) + tol(y, dim) + tol(top, dim))
        lo, hi = c[:, :16].sum(-1), c[:, 16:].sum(-1)
        assert np.array_equal(s.reshape(-1).view(np.uint32), ((lo & 0xffff) | ((hi & 0xffff) << 16)).astype(np.uint32))
        if out is not None and to == "f32":  # the quantizer's own codes of what came out
            other = m.Act(tokens, heads * dim, dev)
            m.quant_act(out.reshape(tokens, -1).contiguous(), other)
            for a, b in zip(act.parts(), other.parts()):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 3, 32, 64, 100, 128, 256, 320, 512, 544, 1000, 1024, 2048, 2080, 5120, 8192, 8224, 16384,
                                 17408, 33000, 65536, 131104])
def test_dims(m27q, dev, dim):
    say("norm dim", dim)
    for tokens in (1, 5):
        check(m27q, dev, tokens, 1, dim, ("f32", "f32", "f32", "f32"), codes=dim % 32 == 0, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [("f32", None, None, "f32"), ("f16", "f16", "f16", "f16"), ("bf16", "bf16", "bf16", "bf16"),
                                   ("f32", "bf16", "bf16", None), ("f16", "f32", None, "bf16"), ("bf16", None, "f32", "f16")])
@pytest.mark.parametrize("tokens,heads,dim", [(3, 1, 5120), (7, 24, 256), (65, 4, 64), (2, 3, 96), (9, 16, 128), (4, 2, 800), (2, 1, 1056), (2, 1, 8224), (3, 1, 16384)])
def test_types_and_heads(m27q, dev, types, tokens, heads, dim):
    say("norm types", types, tokens, heads, dim)
    check(m27q, dev, tokens, heads, dim, types, codes=True)
    check(m27q, dev, tokens, heads, dim, types, codes=False, weighted=False, eps=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,heads,dim", [(1500, 1, 1056), (1100, 1, 5120), (700, 3, 256), (1030, 1, 100)])
def test_rows_alone_and_in_a_batch(m27q, dev, t, tokens, heads, dim):
    import torch
    say("norm batch", t, tokens, heads, dim)
    x = torch.randn(tokens, heads, dim, device=dev, generator=torch.Generator(dev).manual_seed(dim)).to(torch.float32 if t == "f32" else torch.bfloat16)
    y, one = torch.empty_like(x), torch.empty_like(x[:1])
    m27q.rms_norm(x, out=y)
    for i in (0, tokens // 2, tokens - 1):
        m27q.rms_norm(x[i:i + 1], out=one)
        assert torch.equal(one[0], y[i])


@pytest.mark.gpu
@pytest.mark.parametrize("pad,off", [(0, 1), (8, 0), (3, 0), (64, 8), (1, 5)])
@pytest.mark.parametrize("dim", [64, 256, 640, 5120])
def test_strides_and_alignment(m27q, dev, pad, off, dim):
    say("norm strides", pad, off, dim)
    for t in ("f32", "bf16"):
        check(m27q, dev, 6, 2, dim, (t, t, t, "f32"), codes=True, pad=pad, off=off)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 250, 5120, 40000])
@pytest.mark.parametrize("where", ["sum is x", "sum is add", "out is x", "out is add, sum is x"])
def test_in_place(m27q, dev, dim, where):
    import torch
    say("norm in place", dim, where)
    x, add = make(dev, 4, 1, dim, "f32", 1).clone(), make(dev, 4, 1, dim, "f32", 2).clone()
    total, out = torch.empty_like(x), torch.empty_like(x)
    m27q.rms_norm(x, None, 1e-6, add=add, sum=total, out=out)
    a, b = x.clone(), add.clone()
    places = {"sum is x": (a, torch.empty_like(x)), "sum is add": (b, torch.empty_like(x)), "out is x": (torch.empty_like(x), a),
              "out is add, sum is x": (a, b)}[where]
    m27q.rms_norm(a, None, 1e-6, add=b, sum=places[0], out=places[1])
    assert torch.equal(places[0], total) and torch.equal(places[1], out)


@pytest.mark.gpu
def test_a_residual_for_all_tokens(m27q, dev):
    """A residual that is one row for every token (its tokens no distance apart)."""
    import torch
    say("norm broadcast")
    x, add = make(dev, 5, 1, 256, "f32", 1), make(dev, 1, 1, 256, "f32", 2)
    out = torch.empty(5, 1, 256, device=dev)
    m27q.rms_norm(x, None, 1e-6, add=add.expand(5, 1, 256), out=out)
    _, y = want(x, add.expand(5, 1, 256), None, 1e-6)
    assert np.all(np.abs(out.double().cpu().numpy() - y) <= tol(y, 256) + 2.0 ** -24 * np.abs(y))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 96, 5120, 40000])
def test_values_at_the_ends(m27q, dev, dim):
    """Rows of zeros, of tiny and of huge values, and rows that are not finite, beside ordinary ones."""
    import torch
    say("norm ends", dim)
    x = make(dev, 7, 1, dim, "f32", 5).clone().view(7, dim)
    plain = x.clone()
    x[1] = 0
    x[2] *= 1e-30
    x[3] *= 1e30
    x[4, dim // 2] = float("nan")
    x[5, 3] = float("inf")
    out, act = torch.empty_like(x), m27q.Act(7, dim, dev)
    m27q.rms_norm(x, None, 1e-6, out=out, act=act)
    ref = torch.empty_like(x)
    m27q.rms_norm(plain, None, 1e-6, out=ref)
    assert torch.equal(out[0], ref[0]) and torch.equal(out[6], ref[6])
    assert not out[1].any() and not out[3].any()          # zeros; squares past fp32
    assert bool((out[2] - x[2] * 1e3).abs().max() <= 2e-6 * x[2].abs().max() * 1e3)  # eps alone: 1 / sqrt(1e-6)
    assert torch.isnan(out[4]).all()
    assert torch.isnan(out[5, 3]) and not out[5, :3].any()  # inf / inf, finite / inf
    codes, d, _ = act.parts()
    assert not codes[1].any() and not d[1].any() and not d[4].any()


@pytest.mark.gpu
def test_graph_and_streams(m27q, dev):
    import torch
    say("norm graph")
    x, add = make(dev, 9, 1, 5120, "f32", 1).clone(), make(dev, 9, 1, 5120, "f32", 2).clone()
    total, out, act = torch.empty_like(x), torch.empty_like(x), m27q.Act(9, 5120, dev)
    step = lambda s=None: m27q.rms_norm(x, None, 1e-6, add=add, sum=total, out=out, act=act, stream=s)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(make(dev, 9, 1, 5120, "f32", 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [total.clone(), out.clone(), act.buf.clone()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        out.zero_()
        torch.cuda.synchronize()
        step(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, [total, out, act.buf]))


@pytest.mark.gpu
def test_rows_past_32_bits(m27q, dev):
    """Tokens 2^31 - 64 values apart."""
    import torch
    say("norm far rows")
    far = (1 << 31) - 64
    pool = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device=dev)
    x = pool.as_strided((3, 1, 128), (far, 128, 1))
    v = make(dev, 3, 1, 128, "bf16", 3)
    x.copy_(v)
    a, b = torch.empty(3, 1, 128, device=dev), torch.empty(3, 1, 128, device=dev)
    m27q.rms_norm(x, None, 1e-6, out=a)
    m27q.rms_norm(v, None, 1e-6, out=b)
    assert torch.equal(a, b) and bool(a.abs().sum() > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,dim", [((1 << 24) // 17 + 5, 17, 8), ((1 << 22) // 3 + 7, 3, 520)])
def test_more_rows_than_workgroups_of_the_largest_kind(m27q, dev, tokens, heads, dim):
    """Past 2^32 / 256 short rows or 2^32 / 1024 longer ones, of kernels with fewer threads a row."""
    import torch
    say("norm many rows", tokens, heads, dim)
    some = make(dev, 1000, heads, dim, "bf16", 3)
    x = some.repeat(-(-tokens // 1000), 1, 1)[:tokens]
    out, one = torch.empty_like(x), torch.empty_like(some)
    m27q.rms_norm(x, None, 1e-6, out=out)
    m27q.rms_norm(some, None, 1e-6, out=one)
    assert bool(one.abs().sum() > 0)
    for at in range(0, tokens, 1000):
        if at % 100000 == 0 or at + 1000 >= tokens:
            assert torch.equal(out[at: at + 1000], one[: tokens - at])
