"""The steps of a served batch around its products, as cases that can be timed and checked.

A batch that decodes together adds each layer's output to the residual stream, norms it and quantizes it for the next
product; attends over contexts that begin with the same system prompt or document; and at the end picks a token for each
sequence with that request's own temperature and cuts.  A case names one such step; `draw` gives steps of the same kinds.

A case's "op":
  norm    root-mean-square norm of x + residual: the sum, the normed rows, and their 8-bit codes with a scale for 32
  shared  attention of each sequence's new tokens over a prefix that a group of sequences shares and its own tokens behind it
  sample  a token for each row of logits: temperature, top-k, min-p, top-p, from given uniforms

Where `own` is false `run` is the plain form, elementary torch operations in 32 bits (the sampler's weights and running
sums in 64: a token is picked where a sum of 250000 of them passes a border); where it is true it makes the framework's calls.
"""
import importlib
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def listed():
    return [
        # one decoded token between two products: the smallest call, latency and host cost
        {"name": "norm_decode_1", "op": "norm", "rows": 1, "heads": 1, "dim": 5120, "add": True, "codes": True, "types": "f32,f32"},
        # a served batch, one token each
        {"name": "norm_batch_64", "op": "norm", "rows": 64, "heads": 1, "dim": 5120, "add": True, "codes": True, "types": "f32,f32"},
        # a prompt's chunk
        {"name": "norm_prompt_4096", "op": "norm", "rows": 4096, "heads": 1, "dim": 5120, "add": True, "codes": True, "types": "f32,f32"},
        # a prompt's query heads, each normed by itself in front of its rotation, in 16 bits
        {"name": "norm_heads_1531", "op": "norm", "rows": 1531, "heads": 24, "dim": 256, "add": False, "codes": False, "types": "bf16,bf16"},
        # four chats behind one short system prompt, a token each: latency
        {"name": "shared_decode_4", "op": "shared", "groups": 1, "seqs": 4, "q_len": 1, "prefix": 2048, "own_len": 300, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 64, "types": "f16,f32"},
        # 64 questions to one long document, a token each
        {"name": "shared_decode_64", "op": "shared", "groups": 1, "seqs": 64, "q_len": 1, "prefix": 32768, "own_len": 1021, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 64, "types": "f16,f32"},
        # three system prompts, speculative verification of five tokens a sequence
        {"name": "shared_verify_3x8", "op": "shared", "groups": 3, "seqs": 8, "q_len": 5, "prefix": 12000, "own_len": 700, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 16, "types": "bf16,bf16"},
        # eight new prompts behind one document: the largest
        {"name": "shared_prompts_8", "op": "shared", "groups": 1, "seqs": 8, "q_len": 301, "prefix": 8192, "own_len": 301, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 64, "types": "bf16,bf16"},
        # one row of the vocabulary, the chat program's usual settings: latency
        {"name": "sample_1", "op": "sample", "rows": 1, "n": 248320, "kind": "chat", "types": "f32"},
        # a served batch, every request with settings of its own
        {"name": "sample_64_mixed", "op": "sample", "rows": 64, "n": 248320, "kind": "mixed", "types": "f32"},
        # a large batch with a nucleus alone, no number of candidates to bound it
        {"name": "sample_200_top_p", "op": "sample", "rows": 200, "n": 248320, "kind": "top_p", "types": "f32"},
        # a draft model's small vocabulary, an odd size
        {"name": "sample_33_small", "op": "sample", "rows": 33, "n": 32003, "kind": "plain", "types": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case of the same ranges: one row to thousands, odd and ragged sizes, each type."""
    op = rng.choice(["norm", "shared", "sample"])
    if op == "norm":
        t = rng.choice(["f32", "f16", "bf16"])
        if rng.random() < 0.3:
            heads, dim = rng.choice([1, 4, 8, 16, 24, 48]), rng.choice([64, 128, 256])
            codes = rng.random() < 0.3
        else:
            heads, dim, codes = 1, 32 * _log_int(rng, 4, 600), rng.random() < 0.8
        rows = _log_int(rng, 1, max(2, min(4096, 20000000 // (heads * dim))))
        return {"op": op, "rows": rows, "heads": heads, "dim": dim, "add": rng.random() < 0.7, "codes": codes,
                "types": "%s,%s" % (t, rng.choice([t, "f32"]))}
    if op == "shared":
        kind = rng.choice(["decode", "decode", "verify", "prompts"])
        groups = rng.choice([1, 1, 1, 2, 3])
        seqs = {"decode": _log_int(rng, 2, 96), "verify": _log_int(rng, 2, 16), "prompts": rng.randint(2, 6)}[kind] // groups + 1
        q_len = {"decode": 1, "verify": rng.randint(2, 8), "prompts": _log_int(rng, 20, 300)}[kind]
        dim, kv_heads = rng.choice([64, 128, 256, 256]), rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 6, 8])
        t = rng.choice(["f16", "bf16"])
        most = {"decode": 32768, "verify": 16384, "prompts": 6000}[kind]
        return {"op": op, "groups": groups, "seqs": seqs, "q_len": q_len, "prefix": _log_int(rng, 100, most),
                "own_len": q_len + _log_int(rng, 1, 1500), "heads": min(heads, 32 // kv_heads * kv_heads), "kv_heads": kv_heads,
                "dim": dim, "page": rng.choice([16, 32, 64, 128]), "types": t + "," + rng.choice([t, "f32"])}
    n = rng.choice([248320, 248320, _log_int(rng, 1000, 160000)])
    return {"op": op, "rows": _log_int(rng, 1, min(200, 40000000 // n)), "n": n, "kind": rng.choice(["chat", "mixed", "top_p", "plain", "wide"]),
            "types": rng.choice(["f32", "f32", "bf16", "f16"])}


def _lens(c):
    """Of each sequence of each group, its new tokens and its own cached ones behind the prefix (the new ones included); the
    groups' prefixes."""
    r = random.Random("%d %d %d" % (c["seqs"], c["q_len"], c["own_len"]))
    n = c["groups"] * c["seqs"]
    q = [c["q_len"]] + [r.randint((c["q_len"] + 1) // 2, c["q_len"]) for _ in range(n - 1)]
    old = c["own_len"] - c["q_len"]
    mine = [a + (old if i == 0 else r.randint(old // 4, old)) for i, a in enumerate(q)]
    page = c["page"]  # whole pages are shared
    prefix = [max(1, (c["prefix"] if g == 0 else r.randint(c["prefix"] // 2, c["prefix"])) // page) * page for g in range(c["groups"])]
    return q, mine, prefix


def work(case):
    c = case
    if c["op"] == "norm":
        t = [BYTES[x] for x in c["types"].split(",")]
        n = c["rows"] * c["heads"] * c["dim"]
        each = t[0] * (1 + c["add"]) + t[1] * c["add"] + (1 + 8 / 32 if c["codes"] else t[1])
        return {"bytes": int(n * each) + 4 * c["dim"], "flops": 6 * n}
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (c["n"] * BYTES[c["types"]] + 28), "flops": 20 * c["rows"] * c["n"]}
    t = [BYTES[x] for x in c["types"].split(",")]
    q, mine, prefix = _lens(c)
    keys = sum(mine) + sum(prefix)
    pairs = sum(a * (prefix[i // c["seqs"]] + m - a) + a * (a + 1) // 2 for i, (a, m) in enumerate(zip(q, mine)))
    return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] * t[0] + sum(q) * c["heads"] * c["dim"] * (t[0] + t[1]),
            "flops": 4 * c["dim"] * c["heads"] * pairs}


# ------------------------------------------------------------------------------------- inputs --

def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    uniform = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    s = {"case": c}
    if c["op"] == "norm":
        t = DTYPES[c["types"].split(",")[0]]
        shape = (c["rows"], c["heads"], c["dim"])
        # a residual stream has a few channels far above the others
        big = 1 + 30 * (uniform(c["dim"]) < 0.002)
        s.update(x=rand(*shape).to(t), weight=1 + 0.2 * rand(c["dim"]))
        if c["add"]:
            s["add"] = (3 * big * rand(*shape)).to(t)
        return s
    if c["op"] == "sample":
        rows, n = c["rows"], c["n"]
        # a model's logits: a bulk, and a few dozen tokens that stand out; some tokens are banned
        x = 2.2 * rand(rows, n)
        peaks = torch.randint(0, n // 40, (rows, 40), generator=g, device="cuda") + n // 40 * torch.arange(40, device="cuda")
        x.scatter_(1, peaks, 6 + 3 * rand(rows, 40) + 8 * uniform(rows, 1))
        x.masked_fill_(uniform(rows, n) < 1e-4, float("-inf"))
        s.update(logits=x.to(DTYPES[c["types"]]), u=uniform(rows))
        i = torch.arange(rows, device="cuda")
        if c["kind"] == "chat":
            kinds = torch.zeros_like(i)
        else:
            kinds = {"mixed": i % 6, "top_p": 1 + 0 * i, "plain": 2 + 0 * i, "wide": 5 + 0 * i}[c["kind"]]
        # by kind:                   chat  top-p  plain  greedy  min-p  many candidates
        pick = lambda *v: torch.tensor(v, device="cuda")[kinds]  # noqa: E731
        s["temperature"] = pick(0.7, 1.0, 1.0, 0.0, 1.5, 1.3)
        s["top_k"] = pick(40, 0, 0, 0, 0, 2500).to(torch.int32)
        s["top_p"] = pick(0.95, 0.9, 1.0, 1.0, 1.0, 0.98)
        s["min_p"] = pick(0.05, 0.0, 0.0, 0.0, 0.02, 0.0)
        return s
    t = DTYPES[c["types"].split(",")[0]]
    q, mine, prefix = _lens(c)
    n, page, T, D = len(q), c["page"], sum(q), c["dim"]
    kv = [m + prefix[i // c["seqs"]] for i, m in enumerate(mine)]
    per = -(-max(kv) // page)
    # pages in no order; the sequences of a group name the same ones for its prefix
    total = sum(p // page for p in prefix) + sum(-(-m // page) for m in mine) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((n, per), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(prefix):
        table[i * c["seqs"]: (i + 1) * c["seqs"], : p // page] = order[at: at + p // page]
        at += p // page
    for i, m in enumerate(mine):
        first, count = prefix[i // c["seqs"]] // page, -(-m // page)
        table[i, first: first + count] = order[at: at + count]
        at += count
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(s, T=T, max_q=max(q), max_kv=max(kv), max_rows=max(sum(q[i: i + c["seqs"]]) for i in range(0, n, c["seqs"])),
                max_own=max(mine), max_prefix=max(prefix), table=table, start=ints([sum(q[:i]) for i in range(n + 1)]), kv_len=ints(kv),
                first=ints([i * c["seqs"] for i in range(c["groups"] + 1)]), prefix=ints(prefix),
                k_cache=rand(total, c["kv_heads"], page, D).to(t), v_cache=rand(total, c["kv_heads"], page, D).to(t),
                q=(1.5 * rand(T, c["heads"], D)).to(t), scale=D ** -0.5)


# --------------------------------------------------------------------------------- plain forms --

def _plain_norm(s):
    c = s["case"]
    out_t = DTYPES[c["types"].split(",")[1]]
    x = s["x"].float()
    out = {}
    if c["add"]:
        x = x + s["add"].float()
        out["sum"] = x.to(out_t)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"]
    if not c["codes"]:
        out["out"] = y.to(out_t)
        return out
    y = y.view(c["rows"], -1, 32)
    d = y.abs().amax(-1, keepdim=True) / 127
    codes = torch.floor((y / d.clamp(min=1e-37)).abs() + 0.5).clamp(max=127) * y.sign()
    out["codes"] = (codes * d).to(torch.float16)  # what the codes stand for
    return out


def _plain_shared(s):
    """The prefix once for all rows of a group, each sequence's own keys behind it, one softmax over both."""
    c = s["case"]
    G, n, Hk, D, page = c["groups"], c["groups"] * c["seqs"], c["kv_heads"], c["dim"], c["page"]
    H, R, P, mq, mk, T = c["heads"], s["max_rows"], s["max_prefix"], s["max_q"], s["max_own"], s["T"]
    Q = H // Hk
    t = torch.arange(T, device="cuda")
    seq = (t[:, None] >= s["start"][None, 1:]).sum(1)
    group = seq // c["seqs"]
    place = s["kv_len"][seq] - s["start"][seq + 1] + t
    row_g = t - s["start"][s["first"].long()][group]
    row_s = t - s["start"][seq]
    q = s["q"].float().view(T, Hk, Q, D)

    def part(rows, count, longest, tables, first, last):
        """Scores of rows (their batch and row in it) over the keys first + 0 .. longest - 1 of their batch, up to each one's last."""
        j = torch.arange(longest, device="cuda")
        at = first[:, None] + j  # [batch, keys]
        pages = torch.gather(tables.long(), 1, (at // page).clamp(max=tables.shape[1] - 1)).clamp(min=0)
        keys = s["k_cache"][pages, :, at % page].float().permute(0, 2, 3, 1).reshape(count * Hk, D, longest)
        vals = s["v_cache"][pages, :, at % page].float().permute(0, 2, 1, 3).reshape(count * Hk, longest, D)
        m = int(rows[2])
        padded = torch.zeros(count, m, Hk, Q, D, device="cuda")
        padded[rows[0], rows[1]] = q
        end = torch.full((count, m), -1, dtype=last.dtype, device="cuda")
        end[rows[0], rows[1]] = last
        x = torch.bmm(padded.permute(0, 2, 1, 3, 4).reshape(count * Hk, m * Q, D), keys) * s["scale"]
        hidden = at[:, None, :] > end[..., None]  # [batch, row, key]
        x = x.view(count, Hk, m, Q, longest).masked_fill_(hidden[:, None, :, None], float("-inf"))
        top = x.amax(-1, keepdim=True).clamp(min=-1e30)
        p = torch.exp(x.sub_(top))
        sums = torch.bmm(p.view(count * Hk, m * Q, longest), vals).view(count, Hk, m, Q, D)
        back = lambda z: z.permute(0, 2, 1, 3, 4)[rows[0], rows[1]]  # noqa: E731
        return back(top), back(p.sum(-1, keepdim=True)), back(sums)

    shared = s["prefix"].long()
    zero = torch.zeros_like(shared)
    a = part((group, row_g, R), G, P, s["table"][s["first"][:-1].long()], zero, torch.minimum(place, shared[group] - 1))
    b = part((seq, row_s, mq), n, mk, s["table"], shared.repeat_interleave(c["seqs"]), place)
    top = torch.maximum(a[0], b[0])
    fa, fb = torch.exp(a[0] - top), torch.exp(b[0] - top)
    out = (a[2] * fa + b[2] * fb) / (a[1] * fa + b[1] * fb)
    return out.reshape(T, H, D).to(DTYPES[c["types"].split(",")[1]])


def _plain_sample(s):
    x, order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    rows, n = x.shape
    x = x.double()
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    k = torch.where(s["top_k"] > 0, s["top_k"], n).clamp(max=n)[:, None].long()
    rank = torch.arange(n, device="cuda")[None]
    run = w.cumsum(-1)
    among = run.gather(1, k - 1)  # the sum of the first k
    kept = (rank < k) & (w >= s["min_p"].double()[:, None])
    reach = s["top_p"].double()[:, None] * among
    kept[:, 1:] &= (run[:, :-1] < reach) | (s["top_p"][:, None] >= 1)
    kept[:, 0] = True
    last = kept.sum(-1, keepdim=True) - 1
    total = run.gather(1, last)
    pick = (run < s["u"].double()[:, None] * total).sum(-1, keepdim=True).minimum(last)
    pick = torch.where(greedy, torch.zeros_like(pick), pick)
    prob = torch.where(greedy, torch.ones_like(total), w.gather(1, pick) / total)
    return {"token": order.gather(1, pick)[:, 0].to(torch.int32), "prob": prob[:, 0].float()}


# --------------------------------------------------------------------------- the framework's calls --

def _handles(s):
    """What a program makes once and keeps: the library's view of its weights, cache and sequences, outputs, scratch."""
    m = importlib.import_module("mono-qwen27_amd").m27q
    c = s["case"]
    h = {"m": m}
    if c["op"] == "norm":
        t = DTYPES[c["types"].split(",")[1]]
        h["sum"] = torch.empty(s["x"].shape, dtype=t, device="cuda") if c["add"] else None
        h["out"] = None if c["codes"] else torch.empty(s["x"].shape, dtype=t, device="cuda")
        if c["codes"]:
            h["act"] = m.Act(c["rows"], c["heads"] * c["dim"])
            codes, d, _ = h["act"].parts()
            h["parts"] = codes.view(c["rows"], -1, 32), d.unsqueeze(-1)
            h["values"] = torch.empty(h["parts"][0].shape, dtype=torch.float16, device="cuda")
        return h
    if c["op"] == "sample":
        h["token"] = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
        h["prob"] = torch.empty(c["rows"], device="cuda")
        need = m.sample_rows_scratch_bytes(c["rows"], c["n"])
    else:
        h["cache"] = m.KVCache(s["k_cache"], s["v_cache"])
        h["seqs"] = m.Seqs(s["start"], s["kv_len"], s["table"], s["T"], s["max_q"], s["max_kv"])
        h["prefixes"] = m.Prefixes(s["first"], s["prefix"], s["max_rows"], s["max_prefix"])
        h["out"] = torch.empty(s["T"], c["heads"], c["dim"], dtype=DTYPES[c["types"].split(",")[1]], device="cuda")
        need = m.attn_shared_scratch_bytes(h["seqs"], h["prefixes"], c["heads"], h["cache"])
    h["scratch"] = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    return h


def _own(s):
    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    m, op = h["m"], s["case"]["op"]
    if op == "sample":
        m.sample_rows(s["logits"], s["u"], h["token"], h["scratch"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                      prob=h["prob"])
        return {"token": h["token"], "prob": h["prob"]}
    if op == "shared":
        m.attn_shared(h["seqs"], h["prefixes"], h["cache"], s["q"], h["out"], h["scratch"], s["scale"])
        return h["out"]
    m.rms_norm(s["x"], s["weight"], EPS, add=s.get("add"), sum=h["sum"], out=h["out"], act=h.get("act"))
    out = {"sum": h["sum"]} if s["case"]["add"] else {}
    if s["case"]["codes"]:
        # what the codes stand for, as a user who looks at them reads them
        out["codes"] = torch.mul(*h["parts"], out=h["values"])
    else:
        out["out"] = h["out"]
    return out


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "shared": _plain_shared, "sample": _plain_sample}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ definitions --

def exact(case, seed):
    """The definitions in 64 bits, row by row or sequence by sequence."""
    s = prepare(case, seed)
    c = case
    if c["op"] == "norm":
        out = {}
        x = s["x"].double()
        if c["add"]:
            x += s["add"]
            out["sum"] = x
        y = s["weight"].double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + EPS)
        if c["codes"]:
            y = y.reshape(c["rows"], -1, 32)
            step = torch.linalg.vector_norm(y, float("inf"), -1, keepdim=True) / 127
            z = torch.where(step > 0, y / step, torch.zeros_like(y))
            out["codes"] = torch.copysign(torch.trunc(z.abs() + 0.5), z) * step
        else:
            out["out"] = y
        return out
    if c["op"] == "shared":
        q_lens, mine, prefix = _lens(c)
        out, t, Q = [], 0, c["heads"] // c["kv_heads"]
        for i, (a, m) in enumerate(zip(q_lens, mine)):
            n = prefix[i // c["seqs"]] + m
            pages = s["table"][i].long()[: -(-n // c["page"])]
            k, v = (x[pages].double().transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :n] for x in (s["k_cache"], s["v_cache"]))
            hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - a, n, device="cuda")[:, None]
            o = torch.empty(a, c["heads"], c["dim"], dtype=torch.float64, device="cuda")
            for h in range(c["heads"]):
                x = s["q"][t: t + a, h].double() @ k[h // Q].T * s["scale"]
                o[:, h] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ v[h // Q]
            out.append(o)
            t += a
        return torch.cat(out)
    # row by row: the candidates that a threshold leaves, in order, and the first whose running sum passes the pick
    tokens, probs = [], []
    for r in range(c["rows"]):
        x = s["logits"][r].double()
        t, k, top_p, min_p, u = (float(s[a][r]) for a in ("temperature", "top_k", "top_p", "min_p", "u"))
        best = x.max()
        if t <= 0:
            tokens.append(int((x == best).nonzero()[0]))
            probs.append(1.0)
            continue
        k = min(int(k), c["n"]) or c["n"]
        among = (x >= x.kthvalue(c["n"] - k + 1).values).nonzero()[:, 0]
        among = among[torch.argsort(x[among], descending=True, stable=True)][:k]
        w = torch.exp((x[among] - best) / t)
        run = torch.cumsum(w, 0)
        count = int((w >= min_p).sum())
        if top_p < 1:
            count = min(count, int(torch.searchsorted(run, top_p * run[-1])) + 1)
        count = max(count, 1)
        i = min(int(torch.searchsorted(run, u * run[count - 1])), count - 1)
        tokens.append(int(among[i]))
        probs.append(float(w[i] / run[count - 1]))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}
