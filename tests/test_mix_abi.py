"""What the token mixers refuse, on the host before any HIP call (no GPU needed: the addresses are never followed)."""
import ctypes as C

import numpy as np
import pytest

FAKE = 0x10000
NULL, SHAPE, TYPE, LAYOUT, SCRATCH, RANGE = 1, 2, 3, 4, 5, 6


def rows(m, heads=4, dim=64, t=None, ptr=FAKE, token=None, head=None):
    return m.Rows(ptr, m.F16 if t is None else t, heads, dim, 0, heads * dim if token is None else token,
                  dim if head is None else head)


def seqs(m, **k):
    a = dict(start=FAKE, kv_len=FAKE, table=FAKE, n=2, table_stride=8, tokens=6, max_q=3, max_kv=100, pad=0)
    a.update(k)
    return m.SeqsDesc(*a.values())


def cache(m, **k):
    a = dict(k=FAKE, v=FAKE, type=m.F16, pages=20, heads=2, page_size=16, dim=64, pad=0, page_stride=2 * 16 * 64)
    a.update(k)
    return m.CacheDesc(*a.values())


def plan(m, turns=FAKE, rot=32, layout=0):
    return m.RopePlan(turns, rot, layout, 1.0, 0)


def ref(x):
    return None if x is None else C.byref(x)


def test_rope_refuses(m27q):
    m = m27q
    def call(p=0, pos=FAKE, tokens=6, x=0, out=0):
        f = [rows(m) if v == 0 else v for v in (x, out)]
        return m.lib().m27q_rope(ref(plan(m) if p == 0 else p), pos, tokens, ref(f[0]), ref(f[1]), None)
    assert call(p=None) == call(pos=None) == call(x=None) == call(out=None) == NULL
    assert call(p=plan(m, turns=None)) == call(x=rows(m, ptr=None)) == call(out=rows(m, ptr=None)) == NULL
    assert call(tokens=0) == call(tokens=-1) == call(tokens=(1 << 24) + 1) == SHAPE
    for rot in (0, 1, 31, 66):
        assert call(p=plan(m, rot=rot)) == SHAPE
    assert call(out=rows(m, heads=2)) == call(out=rows(m, dim=32)) == call(x=rows(m, heads=0)) == SHAPE
    assert call(x=rows(m, dim=1026), out=rows(m, dim=1026)) == call(x=rows(m, token=-1)) == SHAPE
    assert call(out=rows(m, head=63)) == call(out=rows(m, token=32)) == SHAPE  # outputs on top of each other
    assert call(x=rows(m, t=m.Q8_0)) == call(out=rows(m, t=99)) == TYPE
    assert call(p=plan(m, layout=2)) == call(p=plan(m, turns=FAKE + 4)) == call(pos=FAKE + 2) == LAYOUT
    assert call(x=rows(m, ptr=FAKE + 1)) == call(x=rows(m, t=m.F32, ptr=FAKE + 2)) == LAYOUT
    assert call(out=rows(m, t=m.F32)) == call(out=rows(m, token=512)) == LAYOUT  # in place with another form
    assert call(tokens=1 << 24, x=rows(m, heads=1024, dim=1024), out=rows(m, heads=1024, dim=1024)) == SHAPE


def test_append_refuses(m27q):
    m = m27q
    def call(s=0, c=0, q=0, qo=0, k=0, v=0):
        f = [d if x == 0 else x for x, d in ((s, seqs(m)), (c, cache(m)), (q, rows(m)), (qo, rows(m, ptr=2 * FAKE)),
                                             (k, rows(m, heads=2)), (v, rows(m, heads=2)))]
        return m.lib().m27q_rope_append(ref(plan(m)), FAKE, *[ref(x) for x in f], None)
    for name in "s c q qo k v".split():
        assert call(**{name: None}) == NULL
    assert call(k=rows(m, heads=4), v=rows(m, heads=4)) == call(v=rows(m, heads=1)) == SHAPE
    assert call(q=rows(m, dim=128), qo=rows(m, dim=128, ptr=2 * FAKE)) == SHAPE
    for bad in (dict(n=0), dict(n=65536), dict(table_stride=0), dict(tokens=0), dict(max_q=0), dict(max_q=7),
                dict(max_kv=0), dict(tokens=(1 << 24) + 1)):
        assert call(s=seqs(m, **bad)) == SHAPE
    assert call(s=seqs(m, start=None)) == call(s=seqs(m, kv_len=None)) == call(s=seqs(m, table=None)) == NULL
    assert call(s=seqs(m, start=FAKE + 1)) == LAYOUT
    for bad in (dict(pages=0), dict(heads=0), dict(page_size=0), dict(page_size=8), dict(page_size=48),
                dict(page_size=8192), dict(page_stride=2047), dict(dim=0)):
        assert call(c=cache(m, **bad)) == SHAPE
    assert call(c=cache(m, k=None)) == call(c=cache(m, v=None)) == NULL
    assert call(c=cache(m, type=m.F32)) == TYPE


def test_attention_refuses(m27q):
    m = m27q
    L = m.lib()
    def call(s=0, c=0, q=0, o=0, scale=0.1, window=0, scratch=FAKE, size=1 << 30):
        f = [d if x == 0 else x for x, d in ((s, seqs(m)), (c, cache(m)), (q, rows(m)), (o, rows(m)))]
        return L.m27q_attn_paged(*[ref(x) for x in f], scale, window, scratch, size, None)
    for name in "s c q o scratch".split():
        assert call(**{name: None}) == NULL
    assert call(q=rows(m, heads=3), o=rows(m, heads=3)) == call(o=rows(m, heads=2)) == SHAPE
    assert call(c=cache(m, dim=96, page_stride=1 << 20), q=rows(m, dim=96), o=rows(m, dim=96)) == SHAPE
    assert call(q=rows(m, heads=130), o=rows(m, heads=130)) == SHAPE      # 65 query heads on one
    assert call(q=rows(m, dim=128), o=rows(m, dim=128)) == SHAPE
    assert call(q=rows(m, t=m.BF16)) == call(q=rows(m, t=m.F32)) == call(o=rows(m, t=m.BF16)) == TYPE
    assert call(scale=float("nan")) == call(scale=float("inf")) == call(window=-1) == RANGE
    assert call(q=rows(m, ptr=FAKE + 8)) == call(q=rows(m, token=260)) == call(o=rows(m, t=m.F32, ptr=FAKE + 8)) == LAYOUT
    assert call(c=cache(m, k=FAKE + 8)) == call(c=cache(m, page_stride=2052)) == call(scratch=FAKE + 8) == LAYOUT
    big = seqs(m, max_kv=1 << 20, table_stride=1 << 16)
    need = L.m27q_attn_scratch_bytes(C.byref(big), 4, C.byref(cache(m)))
    assert need > 16 and call(s=big, size=need - 1) == SCRATCH
    assert L.m27q_attn_scratch_bytes(C.byref(seqs(m)), 3, C.byref(cache(m))) == 0
    assert L.m27q_attn_scratch_bytes(None, 4, C.byref(cache(m))) == 0
    # a table bounds the keys: max_kv beyond it costs nothing
    assert (L.m27q_attn_scratch_bytes(C.byref(seqs(m, max_kv=1 << 30)), 4, C.byref(cache(m)))
            == L.m27q_attn_scratch_bytes(C.byref(seqs(m, max_kv=128)), 4, C.byref(cache(m))))


def test_delta_refuses(m27q):
    m = m27q
    L = m.lib()
    def call(scratch=FAKE, size=1 << 40, **k):
        kd = rows(m, heads=2, t=m.F32)
        vd = rows(m, heads=4, dim=32, t=m.F32)
        a = dict(start=FAKE, slots=None, g=FAKE, beta=FAKE, state_in=FAKE, state_out=FAKE, q=kd, k=kd, v=vd, out=vd, n=2,
                 tokens=200, max_len=150, n_slots=2, head_map=0, scale=0.1)
        a.update(k)
        return L.m27q_delta_rule(C.byref(m.DeltaDesc(*a.values())), scratch, size, None)
    assert L.m27q_delta_rule(None, FAKE, 1 << 30, None) == call(scratch=None) == NULL
    for name in ("start", "g", "beta"):
        assert call(**{name: None}) == NULL
    for name in ("q", "k", "v", "out"):
        assert call(**{name: rows(m, ptr=None)}) == NULL
        assert call(**{name: rows(m, heads=2 if name in "qk" else 4, dim=64 if name in "qk" else 32, t=m.BF16)}) == TYPE
    for bad in (dict(n=0), dict(tokens=0), dict(max_len=0), dict(max_len=201), dict(n=65536), dict(n_slots=(1 << 24) + 1)):
        assert call(**bad) == SHAPE
    r = lambda h, d: rows(m, heads=h, dim=d, t=m.F32)  # noqa: E731
    assert call(q=r(2, 96), k=r(2, 96)) == call(q=r(1, 64)) == call(q=r(3, 64), k=r(3, 64)) == SHAPE
    assert call(v=r(4, 40), out=r(4, 40)) == call(v=r(4, 272), out=r(4, 272)) == call(out=r(4, 64)) == SHAPE
    assert call(scale=float("nan")) == call(head_map=2) == RANGE
    assert call(state_in=FAKE + 4) == call(state_out=FAKE + 8) == call(start=FAKE + 2) == call(scratch=FAKE + 4) == LAYOUT
    assert call(v=rows(m, heads=4, dim=32, t=m.F32, ptr=FAKE + 4)) == LAYOUT
    assert call(size=L.m27q_delta_scratch_bytes(2, 200, 150, 4, 64, 32) - 1) == SCRATCH
    assert L.m27q_delta_scratch_bytes(2, 200, 201, 4, 64, 32) == L.m27q_delta_scratch_bytes(2, 200, 150, 4, 80, 32) == 0


@pytest.mark.parametrize("rot,base,scaling,factor,trained,want", [
    (0, 1e4, 0, 1, 0, SHAPE), (33, 1e4, 0, 1, 0, SHAPE), (1026, 1e4, 0, 1, 0, SHAPE), (64, 0.5, 0, 1, 0, RANGE),
    (64, float("nan"), 0, 1, 0, RANGE), (64, float("inf"), 0, 1, 0, RANGE), (64, 1e4, 4, 1, 0, RANGE),
    (64, 1e4, -1, 1, 0, RANGE), (64, 1e4, 1, 0.5, 0, RANGE), (64, 1e4, 3, 4, 0, RANGE), (64, 1.0, 3, 4, 4096, RANGE),
    (2, 1e4, 2, 4, 0, SHAPE)])
def test_turns_refuse(m27q, rot, base, scaling, factor, trained, want):
    out, s = np.zeros(1024, np.uint64), C.c_float()
    call = m27q.lib().m27q_rope_turns
    assert call(rot, base, scaling, factor, trained, out.ctypes.data, C.byref(s)) == want
    assert call(64, 1e4, 0, 1, 0, None, C.byref(s)) == call(64, 1e4, 0, 1, 0, out.ctypes.data, None) == NULL


def test_binding_refuses_tensors_that_do_not_fit(m27q):
    import torch
    m = m27q
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(m.M27QError):
        m.KVCache(k, k[:, :1])
    with pytest.raises(m.M27QError):
        m.KVCache(k.transpose(1, 2), k.transpose(1, 2))
    with pytest.raises(m.M27QError):
        m.Seqs(i32(3), i32(3), i32(2, 4), 2, 1, 16)
    with pytest.raises(m.M27QError):
        m.Seqs(i32(3).long(), i32(2), i32(2, 4), 2, 1, 16)
    with pytest.raises(m.M27QError):
        m.Rope(torch.zeros(8, dtype=torch.int64), 32)
    s, c = m.Seqs(i32(3), i32(2), i32(2, 4), 2, 1, 16), m.KVCache(k, k)
    q = torch.zeros(3, 4, 64, dtype=torch.float16)  # three rows for a call of two
    with pytest.raises(m.M27QError):
        m.attn_paged(s, c, q, q, torch.zeros(64, dtype=torch.uint8), 0.1)
    with pytest.raises(m.M27QError):
        m.attn_paged(s, c, q.transpose(1, 2)[:2], q[:2], torch.zeros(64, dtype=torch.uint8), 0.1)
    x, g = torch.zeros(4, 2, 64), torch.zeros(4, 2)
    for bad in (dict(g=g[:3]), dict(beta=g.double()), dict(state=torch.zeros(1, 2, 64, 32)), dict(start=i32(3)[::2]),
                dict(slots=i32(5))):
        a = dict(start=i32(2), q=x, k=x, v=x, g=g, beta=g, state=torch.zeros(1, 2, 64, 64), state_out=None, out=x,
                 scratch=torch.zeros(64, dtype=torch.uint8), scale=1.0, max_len=4, slots=None)
        a.update(bad)
        with pytest.raises(m.M27QError):
            m.delta_rule(**a)
