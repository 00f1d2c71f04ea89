"""The token mixers of a hybrid decoder, as cases that can be timed and checked.

Between the quantized projections of a decoder layer stand the operators that move information from token to
token.  A full-attention layer rotates its queries and keys by their positions, writes keys and values into the
pages of its cache and attends over them; a gated-delta layer carries one matrix per head from token to token.
A case names one such step; `draw` gives steps of the same kinds over lengths, head layouts, types and page sizes.

A case's "op":
  append   rotary positions of q and k, k and v written to their places in the paged cache
  rope     rotary positions of one tensor, rows in, rows out
  attn     attention of each sequence's new tokens over its pages, the new ones included
  delta    the gated delta rule over each sequence's tokens from a given state, and the state after them

Where `own` is false `run` is the plain form, elementary torch operations in 32 bits; where it is true it makes
the framework's calls.
"""
import importlib
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
CHUNK = 64  # tokens per chunk of the plain delta rule, at most


def listed():
    return [
        # one decoded token of a full-attention layer: the smallest call, latency and host cost
        {"name": "append_decode_1", "op": "append", "seqs": 1, "q_len": 1, "kv_len": 1021, "ragged": False, "heads": 24,
         "kv_heads": 4, "dim": 256, "rot": 64, "half": True, "factor": 1.0, "page": 64, "types": "f32,f16,f16"},
        # a served batch, one token each, positions past the trained length scaled
        {"name": "append_batch_64", "op": "append", "seqs": 64, "q_len": 1, "kv_len": 40000, "ragged": True, "heads": 24,
         "kv_heads": 4, "dim": 256, "rot": 64, "half": True, "factor": 4.0, "page": 64, "types": "f32,bf16,bf16"},
        # two ragged prompts at once
        {"name": "append_prompts", "op": "append", "seqs": 2, "q_len": 2999, "kv_len": 5003, "ragged": True, "heads": 24,
         "kv_heads": 4, "dim": 256, "rot": 64, "half": True, "factor": 1.0, "page": 32, "types": "f32,bf16,bf16"},
        # a draft model's whole-head interleaved positions, an odd number of rows
        {"name": "rope_pairs_777", "op": "rope", "seqs": 1, "q_len": 777, "kv_len": 777, "ragged": False, "heads": 16,
         "kv_heads": 0, "dim": 128, "rot": 128, "half": False, "factor": 1.0, "page": 16, "types": "f32,f32,f32"},
        # one decoded token over a short context: latency
        {"name": "attn_decode_1", "op": "attn", "seqs": 1, "q_len": 1, "kv_len": 1021, "ragged": False, "heads": 24,
         "kv_heads": 4, "dim": 256, "window": 0, "page": 64, "types": "f16,f32"},
        # a served batch of decodes over ragged contexts: the cache's bytes
        {"name": "attn_decode_32", "op": "attn", "seqs": 32, "q_len": 1, "kv_len": 16381, "ragged": True, "heads": 24,
         "kv_heads": 4, "dim": 256, "window": 0, "page": 64, "types": "f16,f32"},
        # speculative verification: a few rows over a long context
        {"name": "attn_verify_5", "op": "attn", "seqs": 2, "q_len": 5, "kv_len": 32768, "ragged": True, "heads": 24,
         "kv_heads": 4, "dim": 256, "window": 0, "page": 16, "types": "bf16,bf16"},
        # a chunk of a long prompt over what is already cached: the largest call
        {"name": "attn_prefill_4096", "op": "attn", "seqs": 1, "q_len": 4096, "kv_len": 8192, "ragged": False,
         "heads": 24, "kv_heads": 4, "dim": 256, "window": 0, "page": 64, "types": "bf16,bf16"},
        # one decoded token of a gated-delta layer
        {"name": "delta_decode_1", "op": "delta", "seqs": 1, "q_len": 1, "ragged": False, "k_heads": 16, "heads": 48,
         "dk": 128, "dv": 128, "types": "f32"},
        # a served batch, one token each: the states' bytes
        {"name": "delta_batch_64", "op": "delta", "seqs": 64, "q_len": 1, "ragged": False, "k_heads": 16, "heads": 48,
         "dk": 128, "dv": 128, "types": "f32"},
        # a prompt of a gated-delta layer
        {"name": "delta_prompt_4096", "op": "delta", "seqs": 1, "q_len": 4096, "ragged": False, "k_heads": 16,
         "heads": 48, "dk": 128, "dv": 128, "types": "f32"},
        # four ragged prompts in 16-bit activations
        {"name": "delta_prompts_bf16", "op": "delta", "seqs": 4, "q_len": 1531, "ragged": True, "k_heads": 16,
         "heads": 48, "dk": 128, "dv": 128, "types": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case of the same ranges: one token to thousands, one sequence to a batch, odd and ragged sizes."""
    op = rng.choice(["append", "append", "rope", "attn", "attn", "attn", "delta", "delta", "delta"])
    kind = rng.choice(["decode", "verify", "prompt"])
    if op == "delta":
        seqs = {"decode": _log_int(rng, 1, 96), "verify": _log_int(rng, 1, 16), "prompt": rng.choice([1, 1, 2, 3, 5])}[kind]
        q_len = {"decode": 1, "verify": rng.randint(2, 16), "prompt": _log_int(rng, 17, 4096 // seqs)}[kind]
        k_heads = rng.choice([4, 8, 16])
        return {"op": op, "seqs": seqs, "q_len": q_len, "ragged": rng.random() < 0.5, "k_heads": k_heads,
                "heads": k_heads * rng.choice([1, 2, 3]), "dk": rng.choice([64, 128, 128]),
                "dv": rng.choice([64, 128, 128]), "types": rng.choice(["f32", "f32", "bf16", "f16"])}
    dim = rng.choice([64, 128, 256, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    seqs = {"decode": _log_int(rng, 1, 64), "verify": _log_int(rng, 1, 8), "prompt": rng.choice([1, 1, 2, 3])}[kind]
    q_len = {"decode": 1, "verify": rng.randint(2, 16), "prompt": _log_int(rng, 33, 2500)}[kind]
    most = 400000 if op == "attn" else 1000000
    kv_len = q_len + _log_int(rng, 1, max(2, min(32768, most // seqs)) if kind != "prompt" else 4096)
    case = {"op": op, "seqs": seqs, "q_len": q_len, "kv_len": kv_len, "ragged": rng.random() < 0.7, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128, 256])}
    if op == "attn":
        t = rng.choice(["f16", "bf16"])
        return dict(case, heads=min(heads, 32 // kv_heads * kv_heads),
                    window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]), types=t + "," + rng.choice([t, "f32"]))
    t = rng.choice(["f16", "bf16"])
    case = dict(case, rot=rng.choice([dim, dim // 2, dim // 4]), half=rng.random() < 0.6,
                factor=rng.choice([1.0, 1.0, 4.0]))
    if op == "rope":
        return dict(case, kv_heads=0, types=rng.choice(["f32,f32,f32", "%s,%s,%s" % (t, t, t)]))
    return dict(case, types="%s,%s,%s" % (rng.choice(["f32", t]), t, t))


def _lens(c):
    """The new tokens and the cached tokens (the new ones included) of each sequence."""
    r = random.Random("%s %d %d" % (c["op"], c["seqs"], c["q_len"]))
    q, kv = [c["q_len"]], [c.get("kv_len", c["q_len"])]
    for _ in range(c["seqs"] - 1):
        q.append(r.randint((c["q_len"] + 1) // 2, c["q_len"]) if c["ragged"] else c["q_len"])
        old = c.get("kv_len", c["q_len"]) - c["q_len"]
        kv.append(q[-1] + (r.randint(old // 2, old) if c["ragged"] else old))
    return q, kv


def _pairs(c):
    """Query-key pairs that the mask lets through, per head."""
    total = 0
    for n, m in zip(*_lens(c)):
        w = c["window"] or m
        first, last = m - n + 1, m  # keys that the first and the last new token see
        if w >= last:
            total += n * (first + last) // 2
        elif w <= first:
            total += n * w
        else:
            total += (w - first) * (first + w - 1) // 2 + (last - w + 1) * w
    return total


def work(case):
    c = case
    q, kv = _lens(c)
    T = sum(q)
    if c["op"] == "delta":
        b = BYTES[c["types"]]
        state = 2 * c["seqs"] * c["heads"] * c["dk"] * c["dv"] * 4
        rows = T * (2 * c["k_heads"] * c["dk"] * b + 2 * c["heads"] * c["dv"] * b + 2 * c["heads"] * 4)
        return {"bytes": state + rows, "flops": 6 * T * c["heads"] * c["dk"] * c["dv"]}
    t = [BYTES[x] for x in c["types"].split(",")]
    if c["op"] == "attn":
        seen = sum(min(m, n - 1 + c["window"]) if c["window"] else m for n, m in zip(q, kv))
        return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * t[0] + T * c["heads"] * c["dim"] * (t[0] + t[1]),
                "flops": 4 * c["dim"] * c["heads"] * _pairs(c)}
    heads, kvh, D = c["heads"], c["kv_heads"], c["dim"]
    return {"bytes": T * D * (heads * (t[0] + t[1]) + 2 * kvh * (t[0] + t[2])) + 4 * T,
            "flops": 3 * T * (heads + kvh) * c["rot"]}


# ------------------------------------------------------------------------------------- inputs --

def _freqs(c):
    """Radians per position of each pair: base^(-2 j / rot), scaled for long contexts by blending it with
    itself over `factor` between the pairs that turn 32 times and once in the trained length."""
    rot, base, factor, trained = c["rot"], 1e7, c["factor"], 8192
    f = [base ** (-2.0 * j / rot) for j in range(rot // 2)]
    if factor == 1.0:
        return f, 1.0
    at = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(0, math.floor(at(32))), min(rot - 1, math.ceil(at(1)))
    ramp = [min(1.0, max(0.0, (j - low) / max(high - low, 1e-3))) for j in range(rot // 2)]
    return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0


def _tables(c, kv, g):
    """Pages of the sequences, in no order, and some that belong to nobody."""
    per = -(-max(kv) // c["page"])
    n = c["seqs"] * per + 3
    return n, torch.randperm(n, generator=g, device="cuda")[: c["seqs"] * per].to(torch.int32).view(c["seqs"], per)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, kv = _lens(c)
    T = sum(q)
    start = torch.tensor([sum(q[:i]) for i in range(len(q) + 1)], dtype=torch.int32, device="cuda")
    s = {"case": c, "T": T, "max_q": max(q), "max_kv": max(kv), "start": start}
    if c["op"] == "delta":
        t, H = DTYPES[c["types"]], c["heads"]
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
        # decays as a learned rate times a softplus, mostly 0.7 to 0.999 a token; betas from a sigmoid
        rate = 1 + 15 * torch.rand(H, generator=g, device="cuda")
        return dict(s, q=unit(rand(T, c["k_heads"], c["dk"])).to(t), k=unit(rand(T, c["k_heads"], c["dk"])).to(t),
                    v=rand(T, H, c["dv"]).to(t), g=-rate * torch.log1p(torch.exp(rand(T, H) - 4)),
                    beta=torch.sigmoid(rand(T, H)), state=0.3 * rand(c["seqs"], H, c["dv"], c["dk"]),
                    scale=c["dk"] ** -0.5)
    t = [DTYPES[x] for x in c["types"].split(",")]
    D = c["dim"]
    if c["op"] != "rope":
        pages, s["table"] = _tables(c, kv, g)
        s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
        s["k_cache"] = rand(pages, c["kv_heads"], c["page"], D).to(t[-1] if c["op"] == "append" else t[0])
        s["v_cache"] = rand(pages, c["kv_heads"], c["page"], D).to(s["k_cache"].dtype)
    if c["op"] == "attn":
        return dict(s, q=(1.5 * rand(T, c["heads"], D)).to(t[0]), scale=D ** -0.5)
    f, s["mscale"] = _freqs(c)
    # turns per position as 64-bit fractions of a turn: a position's phase is their product modulo 2^64
    turns = [int(x / (2 * math.pi) * 2.0 ** 64) for x in f]
    s["turns"] = torch.tensor([u - (1 << 64) if u >> 63 else u for u in turns], dtype=torch.int64, device="cuda")
    s["pos"] = torch.cat([torch.arange(m - n, m, dtype=torch.int32) for n, m in zip(q, kv)]).to("cuda")
    if c["op"] == "rope":
        return dict(s, q=rand(T, c["heads"], D).to(t[0]))
    # the query projection gives each head's query and gate side by side
    return dict(s, q=rand(T, c["heads"], 2, D).to(t[0])[:, :, 0], k=rand(T, c["kv_heads"], D).to(t[0]),
                v=rand(T, c["kv_heads"], D).to(t[0]))


# --------------------------------------------------------------------------------- plain forms --

def _rotated(x, pos, turns, mscale, rot, half):
    """x [T, H, D] with its first `rot` dims rotated, in 32 bits."""
    phase = (pos.to(torch.int64)[:, None] * turns[None]).to(torch.float32) * (2 * math.pi / 2.0 ** 64)
    cos, sin = (phase.cos() * mscale)[:, None], (phase.sin() * mscale)[:, None]
    x = x.float()
    out = x.clone()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., a] * sin + x[..., b] * cos
    return out


def _places(s):
    """Sequence, place in its cache, page and slot of each new token."""
    t = torch.arange(s["T"], device="cuda")
    seq = (t[:, None] >= s["start"][None, 1:]).sum(1)
    at = s["kv_len"][seq] - s["start"][seq + 1] + t
    page = s["table"].long()[seq, at // s["case"]["page"]]
    return seq, at, page, at % s["case"]["page"]


def _plain_append(s):
    c = s["case"]
    t = [DTYPES[x] for x in c["types"].split(",")]
    _, _, page, slot = _places(s)
    s["k_cache"][page, :, slot] = _rotated(s["k"], s["pos"], s["turns"], s["mscale"], c["rot"], c["half"]).to(t[2])
    s["v_cache"][page, :, slot] = s["v"].to(t[2])
    q = _rotated(s["q"], s["pos"], s["turns"], s["mscale"], c["rot"], c["half"]).to(t[1])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_rope(s):
    c = s["case"]
    return _rotated(s["q"], s["pos"], s["turns"], s["mscale"], c["rot"], c["half"]).to(DTYPES[c["types"].split(",")[1]])


def _plain_attn(s):
    """All sequences at once, padded to the longest."""
    c = s["case"]
    n, H, Hk, D = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    mq, mk, G = s["max_q"], s["max_kv"], c["heads"] // c["kv_heads"]
    seq, at, _, _ = _places(s)
    row = torch.arange(s["T"], device="cuda") - s["start"][seq]
    q = torch.zeros(n, mq, H, D, device="cuda")
    q[seq, row] = s["q"].float()
    end = torch.full((n, mq), -1, dtype=at.dtype, device="cuda")  # the last key that each query sees
    end[seq, row] = at
    j = torch.arange(mk, device="cuda")
    page = s["table"].long()[:, j // c["page"]]
    keys = s["k_cache"][page, :, j % c["page"]].float()  # [n, mk, Hk, D]
    vals = s["v_cache"][page, :, j % c["page"]].float()
    q = q.view(n, mq, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(n * Hk, mq * G, D)
    keys = keys.permute(0, 2, 3, 1).reshape(n * Hk, D, mk)
    vals = vals.permute(0, 2, 1, 3).reshape(n * Hk, mk, D)
    ok = j <= end[..., None]
    if c["window"]:
        ok &= j > end[..., None] - c["window"]
    ok = ok[:, None, :, None].expand(n, 1, mq, G, mk).reshape(n, 1, mq * G, mk)
    x = (torch.bmm(q, keys) * s["scale"]).view(n, Hk, mq * G, mk).masked_fill_(~ok, float("-inf"))
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(x.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(n * Hk, mq * G, mk), vals).view(n, Hk, mq * G, D) / total.clamp(min=1e-30)
    o = o.view(n, Hk, mq, G, D).permute(0, 2, 1, 3, 4).reshape(n, mq, H, D)
    return o[seq, row].to(DTYPES[c["types"].split(",")[1]])


def _plain_delta(s):
    """Chunks of up to 64 tokens: within a chunk the rule is a triangular system, solved by doubling diagonal blocks;
    the state goes from chunk to chunk."""
    c = s["case"]
    n, Hk, H, dk, dv = c["seqs"], c["k_heads"], c["heads"], c["dk"], c["dv"]
    L = min(CHUNK, 1 << (s["max_q"] - 1).bit_length())
    N = -(-s["max_q"] // L)
    t = torch.arange(s["T"], device="cuda")
    seq = (t[:, None] >= s["start"][None, 1:]).sum(1)
    row = t - s["start"][seq]

    def chunks(x):  # [T, h, ...] -> [n, H, N, L, ...], zeros behind a sequence's end
        out = torch.zeros(n, N * L, *x.shape[1:], device="cuda")
        out[seq, row] = x.float()
        out = out.repeat_interleave(H // x.shape[1], 2)
        return out.transpose(1, 2).reshape(n, H, N, L, *x.shape[2:])

    q, k, v, g, beta = (chunks(s[x]) for x in ("q", "k", "v", "g", "beta"))
    G = g.cumsum(-1)
    low = torch.ones(L, L, device="cuda", dtype=torch.bool).tril()
    decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, float("-inf")))
    kt = k.transpose(-1, -2).contiguous()
    A = (beta[..., None] * torch.matmul(k, kt) * decay).tril(-1)
    X = torch.eye(L, device="cuda").expand_as(A).contiguous()  # becomes the inverse of 1 + A
    size = 1
    while size < L:
        m = L // (2 * size)
        blocks = lambda z: torch.diagonal(z.view(n, H, N, m, 2 * size, m, 2 * size), 0, 3, 5).permute(0, 1, 2, 5, 3, 4)  # noqa: E731
        x, a = blocks(X), blocks(A)
        corner = -torch.matmul(torch.matmul(x[..., size:, size:].contiguous(), a[..., size:, :size].contiguous()),
                               x[..., :size, :size].contiguous())
        x[..., size:, :size] = corner
        size *= 2
    W = torch.matmul(X, (beta * torch.exp(G))[..., None] * k)
    U = torch.matmul(X, beta[..., None] * v)
    P = torch.matmul(q, kt) * decay
    qg = q * torch.exp(G)[..., None]
    kg = kt * torch.exp(G[..., -1:] - G)[..., None, :]
    last = torch.exp(G[..., -1])[..., None, None]
    S = s["state"].transpose(-1, -2).contiguous()  # [n, H, dk, dv]
    out = torch.empty(n, H, N, L, dv, device="cuda")
    for i in range(N):
        u = U[:, :, i] - torch.matmul(W[:, :, i], S)
        out[:, :, i] = torch.matmul(qg[:, :, i], S) + torch.matmul(P[:, :, i], u)
        S = last[:, :, i] * S + torch.matmul(kg[:, :, i], u)
    out = out.view(n, H, N * L, dv).transpose(1, 2)[seq, row]
    return {"out": (out * s["scale"]).to(DTYPES[c["types"]]), "state": S.transpose(-1, -2).contiguous()}


# --------------------------------------------------------------------------- the framework's calls --

def _handles(s):
    """What a program makes once and keeps: the library's view of its plan, cache and sequences, outputs, scratch."""
    m = importlib.import_module("mono-qwen27_amd").m27q
    c = s["case"]
    h = {"m": m}
    if c["op"] == "delta":
        h["out"], h["state"] = torch.empty_like(s["v"]), torch.empty_like(s["state"])
        need = m.delta_scratch_bytes(c["seqs"], s["T"], s["max_q"], c["heads"], c["dk"], c["dv"])
    else:
        if c["op"] != "rope":
            h["cache"] = m.KVCache(s["k_cache"], s["v_cache"])
            h["seqs"] = m.Seqs(s["start"], s["kv_len"], s["table"], s["T"], s["max_q"], s["max_kv"])
        if c["op"] != "attn":
            h["rope"] = m.Rope(s["turns"], c["rot"], m.ROPE_HALF if c["half"] else m.ROPE_PAIRS, s["mscale"])
        h["out"] = torch.empty(s["T"], c["heads"], c["dim"], dtype=DTYPES[c["types"].split(",")[1]], device="cuda")
        need = m.attn_scratch_bytes(h["seqs"], c["heads"], h["cache"]) if c["op"] == "attn" else 0
    h["scratch"] = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    return h


def _own(s):
    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    m, op = h["m"], s["case"]["op"]
    if op == "append":
        m.rope_append(h["rope"], s["pos"], h["seqs"], h["cache"], s["q"], h["out"], s["k"], s["v"])
        return {"q": h["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "rope":
        m.rope(h["rope"], s["pos"], s["q"], h["out"])
        return h["out"]
    if op == "attn":
        m.attn_paged(h["seqs"], h["cache"], s["q"], h["out"], h["scratch"], s["scale"], s["case"]["window"])
        return h["out"]
    m.delta_rule(s["start"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], h["state"], h["out"], h["scratch"],
                 s["scale"], s["max_q"])
    return {"out": h["out"], "state": h["state"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "rope": _plain_rope, "attn": _plain_attn, "delta": _plain_delta}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ definitions --

def _exact_rotated(x, s):
    c = s["case"]
    f, mscale = _freqs(c)
    a = s["pos"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
    z = mscale * torch.polar(torch.ones_like(a), a)[:, None]  # e^(i angle) [T, 1, rot / 2]
    x = x.double()
    head = x[..., : c["rot"]]
    head = head.unflatten(-1, (2, -1)).transpose(-1, -2) if c["half"] else head.unflatten(-1, (-1, 2))
    turned = torch.view_as_real(torch.view_as_complex(head.contiguous()) * z)
    turned = turned.transpose(-1, -2).flatten(-2) if c["half"] else turned.flatten(-2)
    return torch.cat([turned, x[..., c["rot"]:]], -1)


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence (attention) or token by token (the delta rule)."""
    s = prepare(case, seed)
    c = case
    if c["op"] == "rope":
        return _exact_rotated(s["q"], s)
    q_lens, kv_lens = _lens(c)
    if c["op"] == "append":
        new, vals = _exact_rotated(s["k"], s), s["v"].double()
        kc, vc, t = s["k_cache"].double(), s["v_cache"].double(), 0
        for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
            at = torch.arange(m - n, m, device="cuda")
            page, slot = s["table"][i].long()[at // c["page"]], at % c["page"]
            kc[page, :, slot], vc[page, :, slot] = new[t: t + n], vals[t: t + n]
            t += n
        return {"q": _exact_rotated(s["q"], s), "k_cache": kc, "v_cache": vc}
    if c["op"] == "attn":
        out, t, G = [], 0, c["heads"] // c["kv_heads"]
        for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
            pages = s["table"][i].long()[: -(-m // c["page"])]
            k, v = (x[pages].double().transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :m]
                    for x in (s["k_cache"], s["v_cache"]))
            last = torch.arange(m - n, m, device="cuda")[:, None]
            j = torch.arange(m, device="cuda")[None]
            hidden = (j > last) | (j <= last - c["window"]) if c["window"] else j > last
            o = torch.empty(n, c["heads"], c["dim"], dtype=torch.float64, device="cuda")
            for h in range(c["heads"]):
                x = s["q"][t: t + n, h].double() @ k[h // G].T * s["scale"]
                o[:, h] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ v[h // G]
            out.append(o)
            t += n
        return torch.cat(out)
    # S <- e^g S; u = beta (v - S k); S <- S + u k^T; o = scale S q, for all sequences that have such a token
    S, out = s["state"].double(), torch.empty(s["T"], c["heads"], c["dv"], dtype=torch.float64, device="cuda")
    r = c["heads"] // c["k_heads"]
    starts = s["start"].tolist()
    for i in range(max(q_lens)):
        live = [a for a, n in enumerate(q_lens) if n > i]
        rows = torch.tensor([starts[a] + i for a in live], device="cuda")
        live = slice(None) if len(live) == len(q_lens) else torch.tensor(live, device="cuda")
        q, k = (s[x][rows].double().repeat_interleave(r, 1)[..., None] for x in ("q", "k"))
        old = S[live] * torch.exp(s["g"][rows].double())[..., None, None]
        u = s["beta"][rows].double()[..., None, None] * (s["v"][rows].double()[..., None] - old @ k)
        S[live] = old + u * k.transpose(-1, -2)
        out[rows] = s["scale"] * (S[live] @ q)[..., 0]
    return {"out": out, "state": S}
