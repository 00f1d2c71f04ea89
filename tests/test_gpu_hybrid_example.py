"""examples/hybrid_decode.py: rows of a batch do not see each other, and chunks of a sequence make one.

Tolerance: the two runs differ by summation orders, which move an activation across a rounding to its int8 code (1 / 254 of
its group's largest) or a key's or value's to bfloat16 (2^-9).  A few of a row's hundreds do: a relative difference of the
logits (in norm) of 1 / 254 would take all of them."""
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
def test_batch_and_single_sequences_agree(m27q, dev, example):
    say("hybrid example")
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, example.VOCAB, n).tolist() for n in (5, 90, 33, 1)]
    model = example.Model(m27q, max_seqs=4, max_len=128)
    ids, logits = example.generate(model, prompts, 8)
    assert [len(s) for s in ids] == [len(p) + 8 for p in prompts]
    assert sorted(model.free_slots) == [0, 1, 2, 3] and len(set(model.free_pages)) == 4 * 8
    for prompt, s, rows in zip(prompts, ids, logits):
        assert s[:len(prompt)] == prompt and len(rows) == 8
        # the same tokens alone, other chunks: all but the last prompt token by 7s, then what was generated, one by one
        seq, got, at = example.Sequence(model, s), [], 0
        while at < len(s) - 1:
            n = min(7, len(prompt) - at) if at < len(prompt) else 1
            y = model.step([(seq, s[at: at + n])])
            at += n
            if at >= len(prompt):
                got.append(y[0])
        seq.done(model)
        assert len(got) == 8
        for a, b in zip(rows, got):
            assert float((a - b).norm() / b.norm()) < 1 / 254
