"""Rotary positions (m27q_rope) and the append to the paged cache (m27q_rope_append) against the definition in
64 bits.

Tolerance of a rotated value, per pair (a, b): the angle's own error (64-bit turns, 32 of them kept: 2^-24 of pi/4
twice, 1e-7), the polynomials' cut and roundings (3 * 2^-24), the factor mscale, two products and a sum: at most
8 * 2^-24 of mscale (|a| + |b|), plus one rounding to the output's type."""
import numpy as np
import pytest

from gpu_util import say

ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def rotated(x, pos, rot, base, half, scaling=0, factor=1.0, trained=0.0):
    """x [T, H, D] in 64 bits, its rotation, and |a| + |b| of each value's pair (0 where it stays)."""
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    m = 1.0
    if scaling == 1:
        f = f / factor
    elif scaling == 2:
        f = (base * factor ** (rot / (rot - 2.0))) ** (-2.0 * np.arange(rot // 2) / rot)
    elif scaling == 3:
        def at(n):
            return rot * np.log(trained / (n * 2 * np.pi)) / (2 * np.log(base))
        low, high = max(0, np.floor(at(32))), min(rot - 1, np.ceil(at(1)))
        r = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0, 1)
        f, m = f / factor * r + f * (1 - r), 0.1 * np.log(factor) + 1
    ang = (pos.astype(np.float64)[:, None] * f)[:, None]
    c, s = m * np.cos(ang), m * np.sin(ang)
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    out, size = x.copy(), np.zeros_like(x)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = m * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return out, size


def check(got, want, size, t):
    got = got.double().cpu().numpy()
    tol = 8 * 2.0 ** -24 * size + ULP[t] * np.abs(want) + (2.0 ** -25 if t == "f16" else 0)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) - tol)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,D,rot,half,tin,tout,scaling", [
    (1, 1, 64, 64, True, "f32", "f32", 0), (1, 24, 256, 64, True, "f32", "f16", 0),
    (777, 16, 128, 128, False, "f32", "f32", 0), (33, 3, 128, 32, True, "bf16", "bf16", 1),
    (5, 8, 80, 20, True, "f16", "f32", 2), (7, 5, 33, 6, False, "f32", "bf16", 3), (9, 2, 96, 24, False, "f16", "f16", 3),
    (64, 4, 1024, 1024, True, "bf16", "f32", 0), (3, 1, 2, 2, True, "f32", "f32", 0)])
def test_rope_against_definition(m27q, dev, T, H, D, rot, half, tin, tout, scaling):
    import torch
    say("rope", T, H, D, rot, half, tin, tout, scaling)
    g = torch.Generator().manual_seed(T * 1000 + D)
    x = torch.randn(T, H, D, generator=g).to(dtype(tin))
    pos = torch.randint(0, 1 << 20, (T,), generator=g, dtype=torch.int32)
    pos[0] = 0 if T > 1 else 2 ** 31 - 1
    if T > 2:
        pos[1], pos[2] = -5, 262143
    r = m27q.Rope.make(rot, 1e7, m27q.ROPE_HALF if half else m27q.ROPE_PAIRS, scaling, 4.0, 8192.0, dev)
    out = torch.empty(T, H, D, dtype=dtype(tout), device=dev)
    xd = x.to(dev)
    m27q.rope(r, pos.to(dev), xd, out)
    want, size = rotated(x.double().numpy(), pos.numpy(), rot, 1e7, half, scaling, 4.0, 8192.0)
    check(out, want, size, tout)
    if tin == tout:  # in place gives the same bits
        m27q.rope(r, pos.to(dev), xd, xd)
        assert torch.equal(xd, out)


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 3])
def test_rope_strided_rows(m27q, dev, pad):
    """Query and gate side by side, heads first, and rows whose alignment only allows single values."""
    import torch
    say("rope strided", pad)
    T, H, D, rot = 13, 6, 128, 64
    g = torch.Generator().manual_seed(3)
    pos = torch.arange(100, 100 + T, dtype=torch.int32)
    r = m27q.Rope.make(rot, 1e6, m27q.ROPE_HALF, device=dev)
    buf = torch.randn(T, H, 2, D + pad, generator=g).to(dev)
    x = buf[:, :, 1, pad:]
    want, size = rotated(x.double().cpu().numpy(), pos.numpy(), rot, 1e6, True)
    out = torch.full((H, T, D + pad), 7.0, device=dev)
    m27q.rope(r, pos.to(dev), x, out[:, :, pad:].transpose(0, 1))
    check(out[:, :, pad:].transpose(0, 1), want, size, "f32")
    assert bool((out[:, :, :pad] == 7).all())
    keep = buf[:, :, 0].clone()
    m27q.rope(r, pos.to(dev), x, x)
    check(x, want, size, "f32")
    assert torch.equal(buf[:, :, 0], keep)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,page,D,H,Hk,rot,tin,tc", [
    ([(1, 1)], 16, 256, 24, 4, 64, "f32", "f16"), ([(3, 40), (0, 9), (17, 17), (1, 65)], 32, 64, 4, 2, 64, "f32", "bf16"),
    ([(70, 200), (5, 5)], 64, 128, 8, 8, 32, "bf16", "bf16"), ([(9, 30)], 16, 40, 3, 1, 10, "f16", "f16"),
    ([(1, 7 + i) for i in range(150)], 16, 64, 2, 1, 16, "f32", "f16")])
def test_append_writes_its_places_and_no_others(m27q, dev, lens, page, D, H, Hk, rot, tin, tc):
    import torch
    say("append", lens[:4], page, D, H, Hk)
    g = torch.Generator().manual_seed(page + D)
    n, T = len(lens), sum(a for a, _ in lens)
    per = max(-(-m // page) for _, m in lens)
    pages = n * per + 2
    table = torch.randperm(pages, generator=g)[: n * per].view(n, per).to(torch.int32)
    start = torch.tensor(np.concatenate([[0], np.cumsum([a for a, _ in lens])]), dtype=torch.int32)
    kv = torch.tensor([m for _, m in lens], dtype=torch.int32)
    pos = torch.cat([torch.arange(m - a, m) for a, m in lens]).to(torch.int32)
    buf = torch.randn(T, H, 2, D, generator=g).to(dtype(tin)).to(dev)
    q = buf[:, :, 0]
    k, v = (torch.randn(T, Hk, D, generator=g).to(dtype(tin)).to(dev) for _ in range(2))
    pool = torch.full((pages, 2, Hk, page, D), -3.0, dtype=dtype(tc), device=dev)  # K and V pages alternate
    cache = m27q.KVCache(pool[:, 0], pool[:, 1])
    seqs = m27q.Seqs(start.to(dev), kv.to(dev), table.to(dev), T, max(max(a for a, _ in lens), 1), int(kv.max()))
    r = m27q.Rope.make(rot, 1e7, m27q.ROPE_HALF, device=dev)
    q_out = torch.empty(T, H, D, dtype=dtype(tc), device=dev)
    m27q.rope_append(r, pos.to(dev), seqs, cache, q, q_out, k, v)
    want, size = rotated(q.double().cpu().numpy(), pos.numpy(), rot, 1e7, True)
    check(q_out, want, size, tc)
    want, size = rotated(k.double().cpu().numpy(), pos.numpy(), rot, 1e7, True)
    seen = torch.zeros(pages, page, dtype=torch.bool)
    t = 0
    for s, (a, m) in enumerate(lens):
        for j in range(m - a, m):
            p, o = int(table[s, j // page]), j % page
            seen[p, o] = True
            check(pool[p, 0, :, o], want[t], size[t], tc)
            assert torch.equal(pool[p, 1, :, o], v[t].to(dtype(tc)))
            t += 1
    assert bool((pool.cpu().permute(0, 3, 1, 2, 4)[~seen] == -3).all())


@pytest.mark.gpu
def test_append_leaves_out_what_has_no_place(m27q, dev):
    """Rows before place 0, on pages that are none, past the table, of no sequence: not written; the queries are."""
    import torch
    say("append without places")
    page, D, T = 16, 64, 10
    table = torch.tensor([[0, 9], [2, 1], [-1, 3]], dtype=torch.int32)   # 4 pages: 9 and -1 are none
    start = torch.tensor([0, 4, 6, 8], dtype=torch.int32)                # rows 8, 9 belong to nobody
    kv = torch.tensor([2, 34, 17], dtype=torch.int32)  # rows 0, 1: places -2, -1; rows 4, 5: 32, 33; 6: 15 (page -1)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(T, 1, D, generator=g).to(dev) for _ in range(3))
    pool = torch.zeros(2, 4, 1, page, D, dtype=torch.float16, device=dev)
    cache = m27q.KVCache(pool[0], pool[1])
    pos = torch.arange(T, dtype=torch.int32)
    q_out = torch.zeros(T, 1, D, device=dev)
    r = m27q.Rope.make(D, 1e4, device=dev)
    m27q.rope_append(r, pos.to(dev), m27q.Seqs(start.to(dev), kv.to(dev), table.to(dev), T, 4, 34), cache, q, q_out, k, v)
    want, size = rotated(q.double().cpu().numpy(), pos.numpy(), D, 1e4, True)
    check(q_out, want, size, "f32")
    got = pool[1].cpu()
    places = {(0, 0): 2, (0, 1): 3, (3, 0): 7}
    for p in range(4):
        for o in range(page):
            row = places.get((p, o))
            assert torch.equal(got[p, 0, o], torch.zeros(D, dtype=torch.float16) if row is None else v[row, 0].half().cpu())


def test_turns_are_the_definition(m27q):
    """f_j / 2 pi as 64-bit fractions, plain and scaled, and mscale."""
    for rot, base, sc, fac, tr in ((64, 1e7, 0, 1, 0), (128, 1e4, 1, 8.0, 0), (64, 1e6, 2, 4.0, 0), (128, 1e6, 3, 16.0, 4096.0),
                                   (2, 1.0, 0, 1, 0)):
        t, m = m27q.rope_turns(rot, base, sc, fac, tr)
        x = np.zeros((1, 1, rot))
        x[..., : rot // 2] = 1  # (1, 0) turned by one position: (cos f, sin f)
        want, _ = rotated(x, np.array([1]), rot, base, True, sc, fac, tr)
        ang = t.astype(np.float64) * (2 * np.pi / 2.0 ** 64)
        assert np.allclose(m * np.cos(ang), want[0, 0, : rot // 2], rtol=0, atol=2e-7 * m)  # m is a float
        # in units of 2^-64 of a turn: the cut to a whole number, and the roundings of the double formula
        f = np.arctan2(want[0, 0, rot // 2:], want[0, 0, : rot // 2]) / (2 * np.pi) * 2.0 ** 64
        assert np.all(np.abs(t.astype(np.float64) - f) <= 1 + f * 2.0 ** -48)
