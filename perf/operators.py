"""The operators of a serving step over a key / value cache in pages, as cases that can be timed and compared, in their plain form and as this library's kernels:

  store    rotary positions (one axis, or several) of the new rows' queries and keys; keys and values into the pages of their sequences
  decode   attention of one new token per sequence over its pages
  prompt   causal attention of whole prompts (or of pieces behind what is cached already), packed one behind another
  sample   one token per row of logits: top-k, top-p, min-p, temperature, from given random numbers

Shapes are the benchmark configurations': "small" 14 query heads on 2 key / value heads of 64, "8b" 32 on 8 of 128, "32b" 40 on 8 of 128. Lengths belong to the
case, values and the order of the pages to the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False        # True: run() calls the library; False: elementary torch operations

SHAPES = {"small": (14, 2, 64, True, 1e6), "8b": (32, 8, 128, False, 5e5), "32b": (40, 8, 128, True, 1e6)}      # query heads, key / value heads, head size, split halves, base
VOCAB = {"small": 151936, "8b": 128256, "32b": 152064}


def listed():
    return [
        # one step of 64 conversations; and the rows of a batch of prompts, some of them images with three position axes, written behind what is cached
        {"name": "store_step_64", "op": "store", "model": "small", "io": "f32", "page": 16, "axes": 1, "sequences": 64, "new": 1, "cached": 3000},
        {"name": "store_images_6x1000", "op": "store", "model": "32b", "io": "f16", "page": 64, "axes": 3, "sequences": 6, "new": 1000, "cached": 1500},
        # one conversation; a batch of ragged conversations; the serving load's batch; one document of 131071 positions; long contexts in f16
        {"name": "decode_one_2311", "op": "decode", "model": "8b", "io": "f32", "page": 64, "rows": 1, "shortest": 2311, "longest": 2311},
        {"name": "decode_16_ragged", "op": "decode", "model": "small", "io": "f32", "page": 16, "rows": 16, "shortest": 1, "longest": 1500},
        {"name": "decode_serving_256", "op": "decode", "model": "small", "io": "f32", "page": 16, "rows": 256, "shortest": 32, "longest": 4096},
        {"name": "decode_document_131071", "op": "decode", "model": "32b", "io": "f32", "page": 128, "rows": 1, "shortest": 131071, "longest": 131071},
        {"name": "decode_long_48", "op": "decode", "model": "8b", "io": "f16", "page": 32, "rows": 48, "shortest": 4000, "longest": 16384},
        # short questions packed; the next 512 tokens of documents that are cached already; a whole document
        {"name": "prompt_questions_24", "op": "prompt", "model": "small", "page": 16, "sequences": 24, "shortest": 1, "longest": 97, "cached": 0},
        {"name": "prompt_chunks_4", "op": "prompt", "model": "8b", "page": 32, "sequences": 4, "shortest": 300, "longest": 512, "cached": 6000},
        {"name": "prompt_document_8192", "op": "prompt", "model": "32b", "page": 128, "sequences": 1, "shortest": 8192, "longest": 8192, "cached": 0},
        # one conversation with the usual filters; the serving load's batch, each row with its own
        {"name": "sample_one", "op": "sample", "vocab": 151936, "rows": 1, "kind": "chat"},
        {"name": "sample_serving_256", "op": "sample", "vocab": 128256, "rows": 256, "kind": "mixed"},
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["store", "decode", "decode", "prompt", "prompt", "sample"])
    model, page = rng.choice(["small", "8b", "32b"]), rng.choice([16, 32, 64, 128, 256])
    if op == "store":
        sequences = size(1, 256)
        return {"op": op, "model": model, "io": rng.choice(["f32", "f16"]), "page": page, "axes": rng.choice([1, 2, 3, 4]), "sequences": sequences,
                "new": size(1, max(1, 6000 // sequences)), "cached": rng.choice([0, size(1, 4000)])}
    if op == "decode":
        rows = size(1, 256)
        longest = size(1, min(131071, 500000 // rows))
        return {"op": op, "model": model, "io": rng.choice(["f32", "f16"]), "page": page, "rows": rows, "shortest": rng.choice([0, 1, max(1, longest // 2), longest]), "longest": longest}
    if op == "prompt":
        sequences = size(1, 32)
        longest = size(1, 4000 // sequences)
        return {"op": op, "model": model, "page": page, "sequences": sequences, "shortest": rng.choice([1, longest]), "longest": longest, "cached": rng.choice([0, 0, size(1, 3000)])}
    return {"op": op, "vocab": rng.choice([size(500, 32000), VOCAB["small"], VOCAB["8b"], VOCAB["32b"]]), "rows": size(1, 200), "kind": rng.choice(["chat", "open", "mixed"])}


# ---------------------------------------------------------------- inputs

def _case_rng(case):
    """What belongs to the case (lengths), apart from the seed."""
    return np.random.Generator(np.random.PCG64([ord(c) for c in repr(sorted((k, v) for k, v in case.items() if k != "name"))]))


def _lengths(case):
    """(new rows, cached positions before them) of every sequence of a store or prompt case; (positions) of every row of a decode case."""
    g = _case_rng(case)
    if case["op"] == "decode":
        n = g.integers(case["shortest"], case["longest"] + 1, case["rows"])
        n[0] = case["longest"]
        return n
    lo = case["new"] if case["op"] == "store" else case["shortest"]
    hi = case["new"] if case["op"] == "store" else case["longest"]
    new = g.integers(lo, hi + 1, case["sequences"])
    new[0] = hi
    return new, g.integers(0, case["cached"] + 1, case["sequences"])


def _pages(lengths, page, g):
    """A page table (-1 where a sequence has no page) whose pages lie in any order in a pool with a few unused ones, and the pool's size."""
    need = -(-np.asarray(lengths) // page)
    pool = int(need.sum()) + 3
    order = g.permutation(pool).astype(np.int32)
    table = np.full((len(need), max(1, int(need.max()))), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += int(n)
    return table, pool


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _positions(case, new, cached, g):
    """Rotary positions [axes][rows]: text counts on along every axis; a third of a prompt's rows is an image, whose rows share the first axis' position and count
    along the others by row and column (what follows goes on behind the largest of them)."""
    out = []
    for n, c in zip(new, cached):
        p = np.repeat(np.arange(c, c + n)[None], case["axes"], axis=0)
        if case["axes"] > 1 and n >= 12:
            at, count = int(n // 3), int(n // 3)
            wide = max(1, int(math.sqrt(count)))
            i = np.arange(count)
            grid = [np.zeros(count, dtype=np.int64), i // wide, i % wide, i % 3]
            for a in range(case["axes"]):
                p[a, at:at + count] = c + at + grid[a]
            p[:, at + count:] = c + at + 1 + max(count // wide, wide) + np.arange(n - at - count)
        out.append(p)
    return np.concatenate(out, axis=1).astype(np.int32)


def _sections(case):
    """Rotary pairs per axis: a fourth of them for the first, the rest dealt over the others."""
    pairs, axes = SHAPES[case["model"]][2] // 2, case["axes"]
    if axes == 1:
        return [pairs]
    rest = pairs - pairs // 4
    return [pairs // 4] + [rest // (axes - 1) + (1 if i < rest % (axes - 1) else 0) for i in range(axes - 1)]


def prepare(case, seed):
    g = np.random.Generator(np.random.PCG64(seed))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(std)
    state = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        state["logits"] = normal(rows, vocab, std=2.5)
        state["logits"][:, g.integers(0, vocab, 40)] = -math.inf            # tokens that a grammar rules out
        state["logits"][:, g.integers(0, vocab, 8)] += 8.0
        kind = np.array(["chat", "open", "greedy", "narrow"])[g.choice(4, rows, p=[0.5, 0.3, 0.1, 0.1]) if case["kind"] == "mixed" else np.full(rows, {"chat": 0, "open": 1}[case["kind"]])]
        state["temperature"] = _cuda(np.where(kind == "greedy", 0.0, g.uniform(0.6, 1.3, rows)).astype(np.float32))
        state["top_k"] = _cuda(np.where(kind == "chat", g.integers(20, 65, rows), np.where(kind == "narrow", g.integers(1, 2000, rows), 0)).astype(np.int32))
        state["top_p"] = _cuda(np.where(kind == "open", np.where(g.random(rows) < 0.5, 1.0, g.uniform(0.8, 0.99, rows)), np.where(kind == "chat", 0.95, 0.999)).astype(np.float32))
        state["min_p"] = _cuda(np.where(kind == "open", 0.0, np.where(kind == "chat", 0.05, 0.001)).astype(np.float32))
        state["uniform"] = torch.rand(rows, generator=gen, device="cuda")
        state["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        state["probability"] = torch.zeros(rows, device="cuda")
        return state
    H, K, D = SHAPES[case["model"]][:3]
    io = torch.float16 if case.get("io", "f16") == "f16" else torch.float32
    if case["op"] == "decode":
        lengths = _lengths(case)
    else:
        new, cached = _lengths(case)
        lengths = new + cached
    table, pool = _pages(lengths, case["page"], g)
    state["table"] = _cuda(table)
    state["keys"] = normal(pool, case["page"], K, D, dtype=torch.float16)
    state["values"] = normal(pool, case["page"], K, D, dtype=torch.float16)
    state["lengths"] = _cuda(lengths.astype(np.int32))
    if case["op"] == "decode":
        state["q"] = normal(case["rows"], H, D, dtype=io, std=1.5)
        state["out"] = torch.zeros(case["rows"], H, D, dtype=io, device="cuda")
        state["sequence"] = torch.arange(case["rows"], dtype=torch.int32, device="cuda")
        state["longest"] = case["longest"]
    elif case["op"] == "store":
        rows = int(new.sum())
        state["qkv"] = normal(rows, (H + 2 * K) * D)
        state["sequence"] = _cuda(np.repeat(np.arange(len(new)), new).astype(np.int32))
        state["at"] = _cuda(np.concatenate([np.arange(c, c + n) for n, c in zip(new, cached)]).astype(np.int32))
        state["positions"] = _cuda(_positions(case, new, cached, g))
        state["q"] = torch.zeros(rows, H, D, dtype=io, device="cuda")
        state["sections"] = _sections(case)
    else:
        starts = np.concatenate([[0], np.cumsum(new)])
        rows = int(starts[-1]) + 5                                           # the batch's buffer is a little longer than its prompts
        state["q"] = normal(rows, H, D, dtype=io, std=1.5)
        state["out"] = torch.zeros(rows, H, D, dtype=io, device="cuda")
        state["starts"] = _cuda(starts.astype(np.int32))
        state["host"] = [(int(a), int(b), int(n)) for a, b, n in zip(starts[:-1], starts[1:], lengths)]
        state["sequence"] = torch.arange(case["sequences"], dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------- the plain forms

def _gathered(state, rows, longest):
    """The rows' keys and values in f32, [rows][key / value head][position][head size], up to `longest` positions; which of them there are."""
    page = state["keys"].shape[1]
    table = state["table"][state["sequence"][rows].long()][:, :-(-longest // page)].clamp_min(0).long()
    there = torch.arange(longest, device="cuda") < state["lengths"][rows][:, None]

    def rows_of(pool):
        x = pool[table].flatten(1, 2)[:, :longest].transpose(1, 2).float()
        return torch.where(there[:, None, :, None], x, 0.0)
    return rows_of(state["keys"]), rows_of(state["values"]), there


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v over the positions that are seen; rows that see none are zero. q [..][queries][d]."""
    s = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    return (e @ v) / torch.where(total > 0, total, 1.0)


def _plain_decode(state):
    H, K, D = SHAPES[state["case"]["model"]][:3]
    rows = torch.arange(state["q"].shape[0], device="cuda")
    if state["longest"] == 0:
        return torch.zeros_like(state["q"])
    k, v, there = _gathered(state, rows, state["longest"])
    q = state["q"].float().view(-1, K, H // K, D)
    return _attend(q, k, v, there[:, None, None, :]).reshape(-1, H, D).to(state["q"].dtype)


def _plain_prompt(state):
    H, K, D = SHAPES[state["case"]["model"]][:3]
    out = torch.zeros_like(state["q"])
    for i, (a, b, n) in enumerate(state["host"]):
        if b > a:
            k, v, _ = _gathered(state, torch.tensor([i], device="cuda"), n)
            q = state["q"][a:b].float().view(b - a, K, H // K, D).permute(1, 2, 0, 3)
            seen = torch.arange(n, device="cuda") <= torch.arange(n - (b - a), n, device="cuda")[:, None]
            o = _attend(q.reshape(1, K, -1, D), k, v, seen.repeat(H // K, 1))
            out[a:b] = o.view(K, H // K, b - a, D).permute(2, 0, 1, 3).reshape(b - a, H, D).to(out.dtype)
    return out


def _plain_store(state):
    H, K, D, halves, base = SHAPES[state["case"]["model"]]
    page, rows = state["keys"].shape[1], state["qkv"].shape[0]
    axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device="cuda"), torch.tensor(state["sections"], device="cuda"))
    pair = torch.arange(D // 2, device="cuda", dtype=torch.float64)
    angle = state["positions"][axis].double().T * torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"), -2.0 * pair / D)      # [rows][pairs]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = state["qkv"].view(rows, H + 2 * K, D)

    def turned(y):
        one, two = (y[..., :D // 2], y[..., D // 2:]) if halves else (y[..., 0::2], y[..., 1::2])
        a, b = one * cos - two * sin, one * sin + two * cos
        return torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)
    where = state["table"][state["sequence"].long(), (state["at"] // page).long()].long(), (state["at"] % page).long()
    state["keys"][where] = turned(x[:, H:H + K]).half()
    state["values"][where] = x[:, H + K:].half()
    return {"q": turned(x[:, :H]).to(state["q"].dtype), "keys": state["keys"], "values": state["values"]}


def _plain_sample(state):
    value, token = torch.sort(state["logits"], dim=-1, descending=True, stable=True)
    value = value.double()
    place = torch.arange(value.shape[1], device="cuda")
    top, t = value[:, :1], state["temperature"].double()[:, None]
    k = torch.where(state["top_k"] > 0, state["top_k"], value.shape[1])[:, None]
    kept = place < k
    mass = torch.where(kept, torch.exp(value - top), 0.0)
    before = mass.cumsum(-1) - mass                                          # a token stays while what is before it has not reached top_p
    kept &= (before < state["top_p"].double()[:, None] * mass.sum(-1, keepdim=True)) | (place == 0)
    kept &= (mass >= state["min_p"].double()[:, None]) | (place == 0)
    kept &= (t > 0) | (place == 0)
    weight = torch.where(kept, torch.exp((value - top) / torch.where(t > 0, t, 1.0)), 0.0)
    total = weight.sum(-1, keepdim=True)
    at = (weight.cumsum(-1) <= state["uniform"].double()[:, None] * total).sum(-1, keepdim=True)
    at = torch.minimum(at, (weight > 0).sum(-1, keepdim=True) - 1)
    return {"tokens": token.gather(1, at)[:, 0].int(), "probability": (weight.gather(1, at) / total)[:, 0].float()}


# ---------------------------------------------------------------- the library's operators

def _library(state):
    """The call as a program that keeps its cache, its plan and its workspace makes it."""
    from dooms_b200 import paged
    case, stream = state["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "sample":
        paged.sample_rows(state["logits"], state["uniform"], state["tokens"], state["probability"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                          min_p=state["min_p"], stream=stream)
        return {"tokens": state["tokens"], "probability": state["probability"]}
    H, K, D, halves, base = SHAPES[case["model"]]
    if "cache" not in state:
        state["cache"] = paged.PagedCache(state["keys"], state["values"], state["table"])
        state["scratch"] = torch.empty(state["cache"].scratch_bytes(H), dtype=torch.uint8, device="cuda") if case["op"] != "store" else None
    cache = state["cache"]
    if case["op"] == "store":
        cache.rope_store(state["qkv"], state["sequence"], state["at"], state["positions"], state["q"], base=base, neox=halves, sections=state["sections"], stream=stream)
        return {"q": state["q"], "keys": state["keys"], "values": state["values"]}
    if case["op"] == "decode":
        cache.attention(state["q"], state["sequence"], state["lengths"], state["longest"], state["out"], state["scratch"], stream=stream)
    else:
        cache.attention_prompt(state["q"], state["sequence"], state["starts"], state["lengths"], state["out"], state["scratch"], stream=stream)
    return state["out"]


def run(state):
    if own:
        return _library(state)
    return {"store": _plain_store, "decode": _plain_decode, "prompt": _plain_prompt, "sample": _plain_sample}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    H, K, D, halves, base = SHAPES[case["model"]]
    page, table = case["page"], s["table"].cpu().numpy()
    if case["op"] == "store":
        x = s["qkv"].double().view(-1, H + 2 * K, D)
        freq = [base ** (-2.0 * i / D) for i in range(D // 2)]
        axis = sum([[a] * n for a, n in enumerate(s["sections"])], [])
        pos = s["positions"].double()
        for i in range(D // 2):
            a = (pos[axis[i]] * freq[i])[:, None]
            i1, i2 = (i, i + D // 2) if halves else (2 * i, 2 * i + 1)
            u, w = x[:, :H + K, i1].clone(), x[:, :H + K, i2].clone()
            x[:, :H + K, i1], x[:, :H + K, i2] = u * torch.cos(a) - w * torch.sin(a), u * torch.sin(a) + w * torch.cos(a)
        keys, values = s["keys"].double(), s["values"].double()
        seq, at = s["sequence"].cpu().numpy(), s["at"].cpu().numpy()
        line = _cuda(table[seq, at // page].astype(np.int64) * page + at % page)
        keys.view(-1, K, D)[line], values.view(-1, K, D)[line] = x[:, H:H + K], x[:, H + K:]
        return {"q": x[:, :H], "keys": keys, "values": values}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    jobs = s["host"] if case["op"] == "prompt" else [(r, r + 1, n) for r, n in enumerate(s["lengths"].tolist())]
    for i, (a, b, n) in enumerate(jobs):
        line = torch.from_numpy(table[i].astype(np.int64)).cuda().repeat_interleave(page)[:n] * page + torch.arange(n, device="cuda") % page
        k, v = s["keys"].view(-1, K, D)[line].double(), s["values"].view(-1, K, D)[line].double()
        for h in range(H if n else 0):
            scores = s["q"][a:b, h].double() @ k[:, h // (H // K)].T / math.sqrt(D)
            scores.masked_fill_(torch.ones_like(scores, dtype=torch.bool).triu(n - (b - a) + 1), -math.inf)
            out[a:b, h] = torch.softmax(scores, -1) @ v[:, h // (H // K)]
    return out


def _exact_sample(s):
    logits = s["logits"].cpu().numpy().astype(np.float64)
    temperature, top_k, top_p, min_p, uniform = (s[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    tokens, probability = np.zeros(len(logits), dtype=np.int32), np.zeros(len(logits))
    for r, x in enumerate(logits):
        n = int(top_k[r]) if 0 < top_k[r] < len(x) else len(x)
        border = np.partition(x, len(x) - n)[len(x) - n]
        few = np.nonzero(x >= border)[0]
        few = few[np.lexsort((few, -x[few]))][:n]
        x = x[few] - x[few[0]]
        p = np.exp(x)
        reached = np.nonzero(np.cumsum(p) >= top_p[r] * p.sum())[0]
        n = int(reached[0]) + 1 if len(reached) else len(p)
        n = max(1, min(n, int((p >= min_p[r]).sum())))
        if temperature[r] == 0:
            n = 1
        w = np.exp(x[:n] / (temperature[r] or 1.0))
        ahead = np.nonzero(np.cumsum(w) > uniform[r] * w.sum())[0]
        i = int(ahead[0]) if len(ahead) else int(np.nonzero(w)[0][-1])
        tokens[r], probability[r] = few[i], w[i] / w.sum()
    return {"tokens": torch.from_numpy(tokens), "probability": torch.from_numpy(probability)}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (4.0 * case["vocab"] + 28), "flops": 4.0 * case["rows"] * case["vocab"]}
    H, K, D = SHAPES[case["model"]][:3]
    io = 2 if case.get("io", "f16") == "f16" else 4
    if case["op"] == "store":
        rows = int(_lengths(case)[0].sum())
        return {"bytes": rows * ((H + 2 * K) * D * 4.0 + H * D * io + 2 * K * D * 2 + 4 * (2 + case["axes"])), "flops": 6.0 * rows * (H + K) * D / 2}
    if case["op"] == "decode":
        n = _lengths(case)
        return {"bytes": int(n.sum()) * 4.0 * K * D + case["rows"] * 2.0 * H * D * io, "flops": 4.0 * H * D * int(n.sum())}
    new, cached = _lengths(case)
    pairs = float((new * cached + new * (new + 1) / 2).sum())
    return {"bytes": int((new + cached).sum()) * 4.0 * K * D + int(new.sum()) * 2.0 * H * D * io, "flops": 4.0 * H * D * pairs}
