"""examples/hybrid_decode.py: prompts behind a shared beginning, and sampled continuations.

Tolerance of the logits: as in the example's other test.  The two runs differ by summation orders, which move an activation
across a rounding to its int8 code (1 / 254 of its group's largest) or a key's or value's to bfloat16 (2^-9); a relative
difference (in norm) of 1 / 254 would take all of a row's."""
import importlib.util
import os

import numpy as np
import pytest

from gpu_util import say

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("hybrid_decode", os.path.join(ROOT, "examples", "hybrid_decode.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [16, 176])
def test_shared_beginning_and_sequences_alone_agree(m27q, dev, example, shared):
    say("hybrid example, shared", shared)
    rng = np.random.default_rng(6)
    prefix = rng.integers(0, example.VOCAB, shared).tolist()
    prompts = [rng.integers(0, example.VOCAB, n).tolist() for n in (5, 70, 33, 1)]
    model = example.Model(m27q, max_seqs=5, max_len=256)
    ids, logits = example.generate(model, prompts, 6, prefix=prefix)
    assert sorted(model.free_slots) == list(range(5)) and sorted(model.free_pages) == list(range(5 * 16))
    for prompt, s, rows in zip(prompts, ids, logits):
        whole = prefix + prompt
        assert s[:len(whole)] == whole and len(s) == len(whole) + 6 and len(rows) == 6
        seq, got, at = example.Sequence(model, s), [], 0
        while at < len(s) - 1:  # the same tokens alone
            n = min(31, len(whole) - at) if at < len(whole) else 1
            y = model.step([(seq, s[at: at + n])])
            at += n
            if at >= len(whole):
                got.append(y[0])
        seq.done(model)
        for a, b in zip(rows, got):
            assert float((a - b).norm() / b.norm()) < 1 / 254


@pytest.mark.gpu
def test_sampled_continuations(m27q, dev, example):
    say("hybrid example, sampled")
    rng = np.random.default_rng(7)
    prefix = rng.integers(0, example.VOCAB, 32).tolist()
    prompts = [rng.integers(0, example.VOCAB, n).tolist() for n in (4, 19)]
    model = example.Model(m27q, max_seqs=3, max_len=128)
    run = lambda **how: example.generate(model, prompts, 6, prefix=prefix, **how)[0]  # noqa: E731
    greedy = run()
    assert run(temperature=5.0, top_k=1) == greedy and run(temperature=5.0, top_p=0.0) == greedy
    warm = run(temperature=5.0, seed=3)
    assert warm == run(temperature=5.0, seed=3) and warm != run(temperature=5.0, seed=4)
    assert all(0 <= t < example.VOCAB for s in warm for t in s)


@pytest.mark.gpu
def test_prefix_of_part_of_a_page_is_refused(m27q, dev, example):
    model = example.Model(m27q, max_seqs=2, max_len=64)
    with pytest.raises(ValueError, match="whole pages"):
        example.generate(model, [[1]], 1, prefix=[1] * 17)
