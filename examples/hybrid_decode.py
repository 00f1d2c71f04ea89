"""A batch of prompts through a two-layer hybrid model, then token by token: the token mixers beside the quantized products.

One gated-delta layer and one attention layer with random Q8_0 weights.  Sequences of different lengths share each step:
their rows lie one after the other, `start` says where each begins.  A step has at most 64 rows (what a quantized product
takes), so prompts go in by chunks, and short ones decode beside a long one that is still being read.

    python examples/hybrid_decode.py [--new 16] [--lengths 5,90,33]
"""
import argparse
import importlib
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

HIDDEN, VOCAB = 256, 512
DELTA_K, DELTA_HEADS, DELTA_DIM = 2, 4, 64  # key heads, value heads, dk = dv
Q_HEADS, KV_HEADS, DIM, ROT = 4, 2, 64, 32
PAGE, ROWS = 16, 64


def q8_0(rng, rows, cols):
    """GGUF Q8_0 bytes of a random matrix: 32 codes under one fp16 scale."""
    w = rng.standard_normal((rows, cols // 32, 32)) / np.sqrt(cols)
    d = (np.abs(w).max(-1, keepdims=True) / 127).astype(np.float16)
    codes = np.round(w / d.astype(np.float64)).clip(-127, 127).astype(np.int8)
    return np.concatenate([d.view(np.uint8), codes.view(np.uint8)], axis=-1).reshape(-1)


class Model:
    def __init__(self, m, max_seqs=8, max_len=512, seed=0, device="cuda"):
        import torch
        self.m, self.torch, self.device = m, torch, device
        rng = np.random.default_rng(seed)
        weight = lambda rows, cols=HIDDEN: m.Weight.upload(q8_0(rng, rows, cols), m.Q8_0, cols // 32, rows)  # noqa: E731
        self.embed = weight(VOCAB)
        kd, vd = DELTA_K * DELTA_DIM, DELTA_HEADS * DELTA_DIM
        self.delta_in = [weight(kd), weight(kd), weight(vd), weight(vd)]  # q, k, v, gate
        self.delta_rates, self.delta_out = weight(2 * DELTA_HEADS), weight(HIDDEN, vd)
        self.attn_in = [weight(Q_HEADS * DIM), weight(KV_HEADS * DIM), weight(KV_HEADS * DIM)]
        self.attn_out, self.head = weight(HIDDEN, Q_HEADS * DIM), weight(VOCAB)
        # what a sequence carries: a state per head, and pages of keys and values
        pages = (max_len + PAGE - 1) // PAGE
        self.max_len, self.max_pages = max_len, pages
        self.states = torch.zeros(max_seqs, DELTA_HEADS, DELTA_DIM, DELTA_DIM, device=device)
        pool = (max_seqs * pages, KV_HEADS, PAGE, DIM)
        self.cache = m.KVCache(torch.zeros(pool, dtype=torch.bfloat16, device=device),
                               torch.zeros(pool, dtype=torch.bfloat16, device=device))
        self.rope = m.Rope.make(ROT, 10000.0, device=device)
        self.free_pages = list(range(max_seqs * pages))
        self.free_slots = list(range(max_seqs))

    def products(self, weights, x):
        rows = x.shape[0]
        act = self.m.Act(rows, x.shape[1], self.device)
        ys = [self.torch.empty(rows, w.rc, device=self.device) for w in weights]
        self.m.quant_act(x, act)
        self.m.matmul_q8_multi(weights, act, ys)
        return ys

    def add(self, x, w, residual, gate=None):
        """residual + w (x sigmoid(gate))"""
        act = self.m.Act(x.shape[0], x.shape[1], self.device)
        y = self.torch.empty_like(residual)
        self.m.quant_act(x, act, gate)
        self.m.matmul_q8(w, act, y, residual)
        return y

    def norm(self, x):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()

    def step(self, work):
        """work: (sequence, its next token ids) pairs of at most 64 ids together; the logits after each one's last."""
        m, torch, F = self.m, self.torch, self.torch.nn.functional
        lens = [len(ids) for _, ids in work]
        rows = sum(lens)
        for seq, ids in work:
            seq.grow(self, len(ids))
        table = np.full((len(work), self.max_pages), -1, np.int32)
        for row, (seq, _) in zip(table, work):
            row[:len(seq.pages)] = seq.pages
        ints = lambda a: torch.tensor(np.asarray(a, np.int32), device=self.device)  # noqa: E731
        start = ints(np.concatenate([[0], np.cumsum(lens)]))
        seqs = m.Seqs(start, ints([seq.length for seq, _ in work]), ints(table), rows, max(lens), max(s.length for s, _ in work))
        pos = ints(np.concatenate([np.arange(seq.length - n, seq.length) for (seq, _), n in zip(work, lens)]))
        x = torch.empty(rows, HIDDEN, device=self.device)
        m.embed_rows(self.embed, ints(np.concatenate([ids for _, ids in work])), x)

        # gated-delta layer
        h = self.norm(x)
        q, k, v, gate = self.products(self.delta_in, h)
        rates, = self.products([self.delta_rates], h)
        q, k = (F.normalize(y.view(rows, DELTA_K, DELTA_DIM), dim=-1) for y in (q, k))
        g = -F.softplus(rates[:, :DELTA_HEADS]).contiguous()
        beta = rates[:, DELTA_HEADS:].sigmoid().contiguous()
        v = v.view(rows, DELTA_HEADS, DELTA_DIM)
        out = torch.empty_like(v)
        scratch = torch.empty(m.delta_scratch_bytes(len(work), rows, max(lens), DELTA_HEADS, DELTA_DIM, DELTA_DIM),
                              dtype=torch.uint8, device=self.device)
        m.delta_rule(start, q, k, v, g, beta, self.states, self.states, out, scratch, DELTA_DIM ** -0.5, max(lens),
                     slots=ints([seq.slot for seq, _ in work]))
        x = self.add(out.view(rows, -1), self.delta_out, x, gate)

        # attention layer
        q, k, v = self.products(self.attn_in, self.norm(x))
        q, k, v = q.view(rows, Q_HEADS, DIM), k.view(rows, KV_HEADS, DIM), v.view(rows, KV_HEADS, DIM)
        turned, out = torch.empty(rows, Q_HEADS, DIM, dtype=torch.bfloat16, device=self.device), torch.empty_like(q)
        m.rope_append(self.rope, pos, seqs, self.cache, q, turned, k, v)
        scratch = torch.empty(m.attn_scratch_bytes(seqs, Q_HEADS, self.cache), dtype=torch.uint8, device=self.device)
        m.attn_paged(seqs, self.cache, turned, out, scratch, DIM ** -0.5)
        x = self.add(out.view(rows, -1), self.attn_out, x)

        last = torch.tensor(np.cumsum(lens) - 1, device=self.device)
        return self.products([self.head], self.norm(x[last]))[0]


class Sequence:
    def __init__(self, model, prompt):
        self.ids, self.read, self.length = list(prompt), 0, 0  # tokens, how many of them were given to a step, and cached
        self.pages, self.slot = [], model.free_slots.pop()
        model.states[self.slot].zero_()

    def grow(self, model, n):
        self.length += n
        if self.length > model.max_len:
            raise ValueError("sequence of %d tokens: the model holds %d" % (self.length, model.max_len))
        while len(self.pages) * PAGE < self.length:
            self.pages.append(model.free_pages.pop())

    def done(self, model):
        model.free_pages += self.pages
        model.free_slots.append(self.slot)


def generate(model, prompts, new, rows=ROWS):
    """Greedy continuations of `new` tokens, and each sequence's logits after its prompt and after every new token but the last."""
    seqs = [Sequence(model, p) for p in prompts]
    ends = [len(p) + new for p in prompts]
    logits = [[] for _ in seqs]
    while True:
        work, left = [], rows
        live = [i for i, s in enumerate(seqs) if s.read < len(s.ids) < ends[i] or s.read < len(s.ids) - 1]
        for i in sorted(live, key=lambda i: len(seqs[i].ids) - seqs[i].read):  # single tokens first
            n = min(left, len(seqs[i].ids) - seqs[i].read)
            if n:
                work.append((i, seqs[i].ids[seqs[i].read: seqs[i].read + n]))
                left -= n
        if not work:
            break
        y = model.step([(seqs[i], ids) for i, ids in work])
        best = y.argmax(-1).tolist()
        for (i, ids), row, token in zip(work, y, best):
            seqs[i].read += len(ids)
            if seqs[i].read == len(seqs[i].ids):
                logits[i].append(row)
                seqs[i].ids.append(token)
    for s in seqs:
        s.done(model)
    return [s.ids for s in seqs], logits


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--new", type=int, default=16)
    p.add_argument("--lengths", default="5,90,33")
    a = p.parse_args()
    m = importlib.import_module("mono-qwen27_amd").m27q
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, VOCAB, int(n)).tolist() for n in a.lengths.split(",")]
    ids, _ = generate(Model(m, len(prompts), max(map(len, prompts)) + a.new), prompts, a.new)
    for prompt, s in zip(prompts, ids):
        print("%3d tokens -> %s" % (len(prompt), s[len(prompt):]))


if __name__ == "__main__":
    main()
