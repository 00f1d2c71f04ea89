"""m27q_rope_append keeps to the bounds of the call: rows past max_q and places past max_kv are not written to the cache."""
import numpy as np
import pytest

from gpu_util import say


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 40])
def test_append_keeps_to_the_bounds(m27q, dev, D):
    import torch
    say("append bounds", D)
    page, lens = 16, [(5, 5), (2, 40), (0, 3), (3, 36), (6, 38)]
    T, n = sum(a for a, _ in lens), len(lens)
    start = torch.tensor(np.concatenate([[0], np.cumsum([a for a, _ in lens])]), dtype=torch.int32)
    kv = torch.tensor([m for _, m in lens], dtype=torch.int32)
    table = torch.arange(n * 4, dtype=torch.int32).view(n, 4)
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(T, 1, D, generator=g).half().to(dev) for _ in range(3))
    pool = torch.full((2, n * 4, 1, page, D), 9.0, dtype=torch.float16, device=dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    r = m27q.Rope.make(D, 1e4, device=dev)
    turned, whole = torch.zeros_like(q), torch.empty_like(q)
    seqs = m27q.Seqs(start.to(dev), kv.to(dev), table.to(dev), T, 4, 35)
    m27q.rope_append(r, pos, seqs, m27q.KVCache(pool[0], pool[1]), q, turned, k, v)
    m27q.rope(r, pos, q, whole)
    assert torch.equal(turned, whole)  # the queries are all there
    want, t = torch.full((n * 4, page, D), 9.0, dtype=torch.float16), 0
    for s, (a, m) in enumerate(lens):
        for i in range(a):
            place = m - a + i
            if i < 4 and place < 35:
                want[4 * s + place // page, place % page] = v[t, 0].cpu()
            t += 1
    assert torch.equal(pool[1, :, 0].cpu(), want)
    assert torch.equal((pool[0, :, 0].cpu() == 9).all(-1), (want == 9).all(-1))
