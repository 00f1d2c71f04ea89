"""What norms, attention behind shared prefixes and the sampling of rows refuse, on the host before any HIP call (no GPU
needed: the addresses are never followed)."""
import ctypes as C

import pytest

from test_mix_abi import FAKE, LAYOUT, NULL, RANGE, SCRATCH, SHAPE, TYPE, cache, ref, rows, seqs


def test_norm_refuses(m27q):
    m = m27q

    def call(x=0, add=None, tokens=3, weight=FAKE, eps=1e-6, total=None, out=0, xq=None):
        f = [rows(m, ptr=p) if v == 0 else v for v, p in ((x, FAKE), (add, 2 * FAKE), (total, 3 * FAKE), (out, 4 * FAKE))]
        return m.lib().m27q_rms_norm(ref(f[0]), ref(f[1]), tokens, weight, eps, ref(f[2]), ref(f[3]), xq, None)
    assert call(x=None) == call(out=None) == call(x=rows(m, ptr=None)) == call(add=rows(m, ptr=None)) == NULL
    assert call(total=rows(m, ptr=None)) == call(out=rows(m, ptr=None)) == NULL
    assert call(x=rows(m, t=99)) == call(add=rows(m, t=m.Q8_0, ptr=2 * FAKE)) == call(out=rows(m, t=5)) == TYPE
    assert call(tokens=0) == call(tokens=-4) == call(tokens=(1 << 24) + 1) == SHAPE
    for other in (rows(m, heads=2, ptr=9 * FAKE), rows(m, dim=32, ptr=9 * FAKE)):
        assert call(add=other) == call(total=other) == call(out=other) == SHAPE
    big = dict(heads=1, dim=(1 << 20) + 32)
    assert call(x=rows(m, **big), out=rows(m, ptr=4 * FAKE, **big)) == call(x=rows(m, heads=0)) == SHAPE
    assert call(out=rows(m, head=63, ptr=4 * FAKE)) == call(total=rows(m, token=32, ptr=3 * FAKE)) == SHAPE
    # codes: whole groups of 32, as many rows and columns as the quantizer takes
    assert call(xq=FAKE, x=rows(m, dim=40), out=rows(m, dim=40, ptr=4 * FAKE)) == call(xq=FAKE, tokens=(1 << 16) + 1) == SHAPE
    wide = dict(heads=1024, dim=1056)
    assert call(xq=FAKE, x=rows(m, **wide), out=rows(m, ptr=4 * FAKE, **wide)) == SHAPE
    # more workgroups than a launch has
    assert call(tokens=1 << 24, x=rows(m, heads=1024), out=rows(m, heads=1024, ptr=4 * FAKE)) == SHAPE
    for eps in (0.0, -1e-6, float("nan"), float("inf")):
        assert call(eps=eps) == RANGE
    assert call(weight=FAKE + 2) == call(xq=FAKE + 8) == call(x=rows(m, ptr=FAKE + 1)) == LAYOUT
    # in place, but not with another form or both outputs at one place
    assert call(out=rows(m, t=m.F32)) == call(out=rows(m, token=512)) == LAYOUT
    assert call(add=0, total=rows(m, ptr=2 * FAKE, t=m.BF16)) == LAYOUT
    assert call(total=rows(m, ptr=4 * FAKE)) == LAYOUT


def test_shared_attention_refuses(m27q):
    m = m27q

    def prefix(**k):
        a = dict(first=FAKE, len=FAKE, groups=1, max_rows=4, max_len=64, pad=0)
        a.update(k)
        return m.PrefixesDesc(*a.values())

    def call(s=0, x=0, c=0, q=0, out=0, scale=0.1, scratch=FAKE, size=1 << 40):
        f = [d if v == 0 else v for v, d in ((s, seqs(m)), (x, prefix()), (c, cache(m)), (q, rows(m)),
                                             (out, rows(m, ptr=2 * FAKE)))]
        return m.lib().m27q_attn_shared(*[ref(v) for v in f], scale, scratch, size, None)

    def size(s=0, x=0, heads=4, c=0):
        return m.lib().m27q_attn_shared_scratch_bytes(ref(seqs(m) if s == 0 else s), ref(prefix() if x == 0 else x), heads,
                                                      ref(cache(m) if c == 0 else c))
    for name in ("s", "x", "c", "q", "out", "scratch"):
        assert call(**{name: None}) == NULL
    assert call(x=prefix(first=None)) == call(x=prefix(len=None)) == call(s=seqs(m, table=None)) == NULL
    for bad in (dict(groups=0), dict(groups=3), dict(max_rows=0), dict(max_rows=7), dict(max_len=0), dict(max_len=(1 << 30) + 1)):
        assert call(x=prefix(**bad)) == SHAPE and size(x=prefix(**bad)) == 0
    assert call(q=rows(m, heads=3)) == call(q=rows(m, heads=3), out=rows(m, heads=3, ptr=2 * FAKE)) == SHAPE
    assert call(c=cache(m, dim=96, page_stride=1 << 20)) == call(s=seqs(m, max_q=0)) == SHAPE
    assert call(q=rows(m, t=m.BF16)) == call(out=rows(m, t=m.BF16, ptr=2 * FAKE)) == TYPE
    assert call(scale=float("nan")) == call(scale=float("inf")) == RANGE
    assert call(x=prefix(first=FAKE + 2)) == call(x=prefix(len=FAKE + 1)) == call(scratch=FAKE + 8) == LAYOUT
    assert call(q=rows(m, ptr=FAKE + 2)) == call(c=cache(m, k=FAKE + 2)) == LAYOUT
    assert size() > 0 and call(size=size() - 1) == SCRATCH
    # the grid: a group's rows and the sequences' rows each
    wide = dict(n=65535, tokens=1 << 24, max_q=1)
    assert call(s=seqs(m, **wide), x=prefix(groups=65535, max_rows=1 << 24)) == SHAPE


@pytest.mark.parametrize("n,max_q,max_rows,prefix,own", [(4, 1, 4, 48, 8), (9, 5, 40, 48, 14), (65, 1, 64, 21, 2)])
def test_own_keys_have_parts_beside_a_prefix(m27q, n, max_q, max_rows, prefix, own):
    """Bounds that let a sequence share anything from nothing to all of its keys: the scratch has room for the prefix's parts
    and for as many of its own as fill the 256 CUs (two places on each; of few rows of 256 half of one), two at least."""
    m = m27q
    tokens, heads, dim = n * max_q, 24, 256
    s = seqs(m, n=n, tokens=tokens, max_q=max_q, max_kv=33000, table_stride=600)
    c = cache(m, heads=4, dim=dim, page_size=64, page_stride=4 * 64 * dim, pages=100)
    x = m.PrefixesDesc(FAKE, FAKE, 1, max_rows, 33000, 0)
    assert m.lib().m27q_attn_shared_scratch_bytes(ref(s), ref(x), heads, ref(c)) >= (prefix + own) * tokens * heads * (dim * 4 + 8)


@pytest.mark.parametrize("dim,tokens", [(256, 1 << 20), (256, (1 << 20) - 64), (64, 1 << 22), (64, (1 << 22) - 64)])
def test_prefixes_of_more_rows_than_a_join_takes(m27q, dim, tokens):
    """The join has a workgroup for 1024 / dim rows, of 2^24 workgroups at most: above that each sequence reads all of its
    keys, in one part (the scratch is the paged attention's)."""
    m = m27q
    heads = 64
    s = seqs(m, n=2, tokens=tokens, max_q=tokens, max_kv=1 << 22, table_stride=1 << 16)
    c = cache(m, heads=heads, dim=dim, page_size=64, page_stride=heads * 64 * dim, pages=1 << 18)
    x = m.PrefixesDesc(FAKE, FAKE, 1, tokens, 1 << 21, 0)
    paged = m.lib().m27q_attn_scratch_bytes(ref(s), heads, ref(c))
    shared = m.lib().m27q_attn_shared_scratch_bytes(ref(s), ref(x), heads, ref(c))
    assert paged == 16 and (shared == paged) == (tokens * heads * dim // 1024 >= 1 << 24)


def test_sampling_refuses(m27q):
    m = m27q

    def call(size=1 << 40, scratch=FAKE, **k):
        a = dict(logits=FAKE, temperature=FAKE, top_k=FAKE, top_p=FAKE, min_p=FAKE, u=FAKE, token=FAKE, prob=FAKE, stride=100,
                 type=m.F32, rows=4, n=100, pad=0)
        a.update(k)
        return m.lib().m27q_sample_rows(C.byref(m.SamplingDesc(*a.values())), scratch, size, None)
    assert m.lib().m27q_sample_rows(None, FAKE, 1 << 40, None) == NULL
    assert call(logits=None) == call(u=None) == call(token=None) == call(scratch=None) == NULL
    assert call(type=m.Q8_0) == call(type=99) == TYPE
    for bad in (dict(rows=0), dict(rows=65536), dict(n=0), dict(n=(1 << 24) + 1, stride=1 << 25), dict(stride=99), dict(stride=-100)):
        assert call(**bad) == SHAPE
    for name in ("logits", "temperature", "top_k", "top_p", "min_p", "u", "token", "prob"):
        assert call(**{name: FAKE + 2}) == LAYOUT
    assert call(logits=FAKE + 1, type=m.F16) == call(scratch=FAKE + 8) == LAYOUT
    need = m.sample_rows_scratch_bytes(4, 100)
    assert need > 0 and call(size=need - 1) == SCRATCH
    assert m.sample_rows_scratch_bytes(0, 100) == m.sample_rows_scratch_bytes(4, 0) == m.sample_rows_scratch_bytes(65536, 9) == 0


@pytest.fixture
def calls(m27q):
    """Each call with arguments that fit it, all in host memory, by its name."""
    import torch
    m = m27q
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    pages = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    s, x = m.Seqs(i32(0, 1, 2), i32(5, 6), i32(1, 2, 1, 3).view(2, 2), 2, 1, 20), m.Prefixes(i32(0, 2), i32(16), 2, 16)
    q, scratch, y = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(1 << 20, dtype=torch.uint8), torch.zeros(2, 64)
    return {"m27q_rms_norm": lambda **k: m.rms_norm(y, **{"out": y.clone(), **k}),
            "m27q_attn_shared": lambda **k: m.attn_shared(s, x, m.KVCache(pages, pages), q, k.get("out", q.clone()), scratch, 0.1),
            "m27q_sample_rows": lambda **k: m.sample_rows(y, **{"u": torch.zeros(2), "token": i32(0, 0), "scratch": scratch, **k})}


@pytest.mark.parametrize("name", ["m27q_rms_norm", "m27q_attn_shared", "m27q_sample_rows"])
def test_host_tensors_are_refused(m27q, calls, name):
    with pytest.raises(m27q.M27QError, match=name + ".*current GPU's memory") as e:
        calls[name]()
    assert e.value.status == 4


def test_binding_refuses_tensors_that_do_not_fit(m27q, calls):
    import torch
    norm, sample, shared = calls["m27q_rms_norm"], calls["m27q_sample_rows"], calls["m27q_attn_shared"]
    bad = [(norm, dict(add=torch.zeros(3, 64))), (norm, dict(weight=torch.zeros(63))),
           (norm, dict(weight=torch.zeros(64).half())), (norm, dict(out=torch.zeros(2, 64, 2)[..., 0])), (norm, dict(out=torch.zeros(2))),
           (norm, dict(act=m27q.Act(3, 64, "cpu"))), (norm, dict(act=m27q.Act(2, 32, "cpu"))),
           (sample, dict(u=torch.zeros(3))), (sample, dict(temperature=torch.zeros(1))), (sample, dict(prob=torch.zeros(2).double())),
           (sample, dict(top_k=torch.zeros(3, dtype=torch.int32))), (sample, dict(token=torch.zeros(1, dtype=torch.int32))),
           (shared, dict(out=torch.zeros(3, 4, 64)))]
    for f, k in bad:
        with pytest.raises(m27q.M27QError) as e:
            f(**k)
        assert e.value.status == SHAPE, k
    with pytest.raises(m27q.M27QError) as e:
        sample(top_k=torch.zeros(2, dtype=torch.int64))
    assert e.value.status == LAYOUT
    with pytest.raises(m27q.M27QError):
        m27q.Prefixes(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1, 1)
    with pytest.raises(m27q.M27QError):
        m27q.Prefixes(torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), 1, 1)


@pytest.mark.parametrize("name", ["attn_paged", "attn_shared", "sample_rows", "delta_rule", "rms_norm"])
def test_binding_refuses_scratch_of_less_memory_than_elements(m27q, calls, name):
    """Expanded tensors: a million elements in one byte of memory."""
    import torch
    m = m27q
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    little = torch.zeros(1, dtype=torch.uint8).expand(1 << 20)
    pages = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    s, cache, q = m.Seqs(i32(0, 1, 2), i32(5, 6), i32(1, 2, 1, 3).view(2, 2), 2, 1, 20), m.KVCache(pages, pages), torch.zeros(2, 4, 64).half()
    x, g, act = torch.zeros(2, 2, 64), torch.zeros(2, 2), m.Act(2, 64, "cpu")
    act.buf = little
    call = {"attn_paged": lambda: m.attn_paged(s, cache, q, q.clone(), little, 0.1),
            "attn_shared": lambda: m.attn_shared(s, m.Prefixes(i32(0, 2), i32(16), 2, 16), cache, q, q.clone(), little, 0.1),
            "sample_rows": lambda: calls["m27q_sample_rows"](scratch=little),
            "delta_rule": lambda: m.delta_rule(i32(0, 2), x, x, x, g, g, torch.zeros(1, 2, 64, 64), None, x.clone(), little, 1.0, 2, slots=i32(0)),
            "rms_norm": lambda: m.rms_norm(torch.zeros(2, 64), act=act)}[name]
    with pytest.raises(m.M27QError) as e:
        call()
    assert e.value.status == LAYOUT and "current GPU" not in str(e.value)
