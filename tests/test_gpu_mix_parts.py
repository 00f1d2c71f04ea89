"""The sequences of a step in two calls over the same rows, each with its part of start, lengths and tables, against all of
them in one call.  Tolerances are twice those of test_gpu_attn.py and test_gpu_delta.py: both sides have theirs."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_attn import Problem as Attention
from test_gpu_delta import Problem as Delta


@pytest.mark.gpu
def test_attention_in_two_calls(m27q, dev):
    import torch
    say("attention in two calls")
    lens = [(1, 300), (1, 77), (1, 512), (90, 400), (41, 41)]
    p = Attention(m27q, dev, lens, 4, 2, 64, 16)
    whole = p.run("f32", 0.125)
    cache, q = m27q.KVCache(p.kc.to(dev), p.vc.to(dev)), p.q.to(dev)
    start, kv, table = p.start.to(dev), p.kv.to(dev), p.table.to(dev)
    out = torch.full((p.T, 4, 64), 9.0, device=dev)
    for a, b, max_q in ((0, 3, 1), (3, 5, 90)):
        seqs = m27q.Seqs(start[a: b + 1], kv[a:b], table[a:b], p.T, max_q, 512)
        scratch = torch.empty(m27q.attn_scratch_bytes(seqs, 4, cache), dtype=torch.uint8, device=dev)
        m27q.attn_paged(seqs, cache, q, out, scratch, 0.125)
    want, A, es, small = p.want(0.125)
    tol = 2 * ((2.0 ** -22 + es) * A + small + 2.0 ** -24 * np.abs(want))
    assert np.all(np.abs(out.double().cpu().numpy() - whole) <= tol)


@pytest.mark.gpu
def test_delta_rule_in_two_calls(m27q, dev):
    import torch
    say("delta rule in two calls")
    lens = [1, 1, 1, 150, 70]
    p = Delta(m27q, dev, lens, 2, 4, 64, 32)
    whole, ends = p.run()
    start, q, k, v, g, beta, st = (x.to(dev) for x in (p.start, p.q, p.k, p.v, p.g, p.beta, p.state))
    out, slots = torch.full_like(v, 9.0), torch.arange(5, dtype=torch.int32, device=dev)
    T = sum(lens)
    for a, b, most in ((0, 3, 1), (3, 5, 150)):
        scratch = torch.empty(m27q.delta_scratch_bytes(b - a, T, most, 4, 64, 32), dtype=torch.uint8, device=dev)
        m27q.delta_rule(start[a: b + 1], q, k, v, g, beta, st, st, out, scratch, 0.125, most, slots=slots[a:b])
    _, _, size, sizes = p.want()
    step = 2 * 8 * np.sqrt(150 * 128) * 2.0 ** -24
    assert np.all(np.abs(out.double().cpu().numpy() - whole) <= step * size * 0.125 * 1.01 + 2.0 ** -23 * np.abs(whole))
    assert np.all(np.abs(st.double().cpu().numpy() - ends) <= step * np.stack(sizes)[..., None])
