"""The Python calls refuse a single tensor in pageable host memory beside others on the GPU.

Each call has a second fault, which the library refuses on the host, so that none of them is ever launched: what is tested is
that the binding sees the tensor before it hands the call on."""
import pytest

from gpu_util import say


@pytest.fixture
def parts(m27q, dev):
    """On the GPU and in host memory: a rope plan, a cache, scratch; and tensors that fit them."""
    import torch

    def at(d):
        pages = torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=d)
        return {"rope": m27q.Rope.make(32, 1e4, device=d), "cache": m27q.KVCache(pages, pages),
                "scratch": torch.zeros(8, dtype=torch.uint8, device=d)}
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    seqs = m27q.Seqs(i32(0, 2), i32(5), i32(1, 2).view(1, 2), 2, 2, 20)
    return at(dev), at("cpu"), i32, z, seqs, m27q.Prefixes(i32(0, 1), i32(16), 2, 16)


def calls(m, gpu, i32, z, seqs, prefixes):
    """Each call by its name and what of it is in host memory (a dict's entries in place of gpu's)."""
    import torch
    q, k, x, g = z(2, 4, 64), z(2, 2, 64), z(2, 2, 64).float(), z(2, 2).float()
    a = lambda o: {**gpu, **o}  # noqa: E731
    scores = torch.zeros(2, 100, device=q.device)
    return {
        ("m27q_rope", "rope"): lambda o: m.rope(a(o)["rope"], i32(0, 1), q, z(2, 3, 64)),
        ("m27q_rope_append", "rope"): lambda o: m.rope_append(a(o)["rope"], i32(0, 1), seqs, a(o)["cache"], q, q.clone(), z(2, 1, 64), k),
        ("m27q_rope_append", "cache"): lambda o: m.rope_append(a(o)["rope"], i32(0, 1), seqs, a(o)["cache"], q, q.clone(), z(2, 1, 64), k),
        ("m27q_attn_paged", "cache"): lambda o: m.attn_paged(seqs, a(o)["cache"], q, q.clone(), a(o)["scratch"], 0.1),
        ("m27q_attn_paged", "scratch"): lambda o: m.attn_paged(seqs, a(o)["cache"], q, q.clone(), a(o)["scratch"], 0.1),
        ("m27q_attn_shared", "cache"): lambda o: m.attn_shared(seqs, prefixes, a(o)["cache"], q, q.clone(), a(o)["scratch"], 0.1),
        ("m27q_attn_shared", "scratch"): lambda o: m.attn_shared(seqs, prefixes, a(o)["cache"], q, q.clone(), a(o)["scratch"], 0.1),
        ("m27q_delta_rule", "scratch"): lambda o: m.delta_rule(i32(0, 2), x, x, x, g, g, x.new_zeros(1, 2, 64, 64), None, x.clone(),
                                                               a(o)["scratch"], 1.0, 2, slots=i32(0), head_map=7),
        ("m27q_sample_rows", "scratch"): lambda o: m.sample_rows(scores, g.new_zeros(2), i32(0, 0), a(o)["scratch"]),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name,what", [("m27q_rope", "rope"), ("m27q_rope_append", "rope"), ("m27q_rope_append", "cache"),
                                       ("m27q_attn_paged", "cache"), ("m27q_attn_paged", "scratch"), ("m27q_attn_shared", "cache"),
                                       ("m27q_attn_shared", "scratch"), ("m27q_delta_rule", "scratch"), ("m27q_sample_rows", "scratch")])
def test_one_tensor_in_host_memory_is_refused(m27q, parts, name, what):
    say("host", name, what)
    gpu, cpu, *rest = parts
    call = calls(m27q, gpu, *rest)[name, what]
    with pytest.raises(m27q.M27QError) as e:
        call({})  # all on the GPU: the library's own refusal
    assert "current GPU's memory" not in str(e.value)
    with pytest.raises(m27q.M27QError, match=name + ".*current GPU's memory") as e:
        call({what: cpu[what]})
    assert e.value.status == 4
