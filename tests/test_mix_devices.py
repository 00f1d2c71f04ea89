"""The token mixers' Python calls refuse tensors that the GPU cannot read, before anything is launched (no GPU needed)."""
import pytest


@pytest.fixture
def calls(m27q):
    """Each call with arguments that fit it, all in host memory, by its name."""
    import torch
    m = m27q
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    rope = m.Rope.make(32, 1e4, device="cpu")
    pages = half(4, 2, 16, 64)
    cache, seqs = m.KVCache(pages, pages), m.Seqs(i32(0, 2), i32(5), i32(1, 2).view(1, 2), 2, 2, 20)
    q, k, x, g = half(2, 4, 64), half(2, 2, 64), torch.zeros(2, 2, 64), torch.zeros(2, 2)
    scratch, state = torch.zeros(1 << 20, dtype=torch.uint8), torch.zeros(1, 2, 64, 64)
    return {"m27q_rope": lambda: m.rope(rope, i32(0, 1), q, q),
            "m27q_rope_append": lambda: m.rope_append(rope, i32(0, 1), seqs, cache, q, q.clone(), k, k),
            "m27q_attn_paged": lambda: m.attn_paged(seqs, cache, q, q, scratch, 0.1),
            "m27q_delta_rule": lambda: m.delta_rule(i32(0, 2), x, x, x, g, g, state, None, x.clone(), scratch, 1.0, 2,
                                                    slots=i32(0))}


@pytest.mark.parametrize("name", ["m27q_rope", "m27q_rope_append", "m27q_attn_paged", "m27q_delta_rule"])
def test_host_tensors_are_refused(m27q, calls, name):
    with pytest.raises(m27q.M27QError, match=name + ".*current GPU's memory") as e:
        calls[name]()
    assert e.value.status == 4


def test_records_carry_where_their_tensors_lie(m27q):
    """The number of the GPU behind the record; mixed places and host memory are no GPU."""
    import struct

    class T:
        def __init__(self, device, pinned=False):
            self.is_cuda, self.device, self.pinned = device >= 0, device, pinned

        def get_device(self):
            return self.device

        def is_pinned(self):
            return self.pinned

    at = lambda *t: struct.unpack("=i", m27q._packed(b"record", *t)[6:])[0]  # noqa: E731
    assert at(T(0)) == 0 and at(T(3), T(3)) == 3
    assert at(T(-1)) == at(T(0), T(1)) == at(T(0), T(-1)) == -1
    assert at(T(-1, True)) == -2 and at(T(1), T(-1, True)) == 1 and at(T(-1), T(-1, True)) == -1


@pytest.mark.gpu
def test_pinned_lengths_are_read(m27q, dev):
    """Page-locked host memory is the GPU's too: positions, lengths and tables there give the same."""
    import torch
    from gpu_util import say
    say("pinned lengths")
    g = torch.Generator().manual_seed(2)
    q, k = (torch.randn(3, h, 64, generator=g).half().to(dev) for h in (4, 2))
    rope = m27q.Rope.make(64, 1e4, device=dev)
    outs = []
    for place in (lambda t: t.to(dev), lambda t: t.pin_memory()):
        pages = torch.zeros(2, 4, 2, 16, 64, dtype=torch.float16, device=dev)
        i32 = lambda *v: place(torch.tensor(v, dtype=torch.int32))  # noqa: E731
        seqs = m27q.Seqs(i32(0, 1, 3), i32(20, 5), i32(3, 0, 1, 2).view(2, 2), 3, 2, 32)
        cache, turned, out = m27q.KVCache(pages[0], pages[1]), torch.empty_like(q), torch.empty_like(q)
        m27q.rope_append(rope, i32(19, 3, 4), seqs, cache, q, turned, k, k)
        scratch = torch.empty(m27q.attn_scratch_bytes(seqs, 4, cache), dtype=torch.uint8, device=dev)
        m27q.attn_paged(seqs, cache, turned, out, scratch, 0.125)
        torch.cuda.synchronize()
        outs.append((pages, turned, out))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.abs().sum() > 0)
