"""Cases that measure the operators for drafted tokens, streams and scored tokens of ``nanopointllm_b200``.

Three operators:

* ``tree``     - attention of a tree of drafted tokens over the paged cache (``paged_attention.paged_tree_attention``)
* ``window``   - attention with a sliding window and a few first tokens that stay visible, over the paged cache, for
                 single tokens and for prompts (``paged_attention.paged_window_attention``)
* ``logprobs`` - log probabilities of given tokens, the entropy of their distributions and the top alternatives
                 (``logprobs.token_logprobs``)

``own`` False computes them in elementary torch operations, True calls the
package. Sizes are those of the repository's 7B shape (32 heads of 128,
vocabulary 32003, cache pages of 256, a 20 x 800-token prefill batch) and
generic ones: grouped key/value heads, pages of 16, longer contexts.
"""
from __future__ import annotations

import importlib
import importlib.util
import math
import pathlib
import sys

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
CHUNK = 512  # queries that the plain form takes at a time


# ------------------------------------------------------------------- cases
def listed():
    mha = {"heads": 32, "kv_heads": 32, "dim": 128, "page": 256, "type": "fp16"}  # the 7B shape and its cache
    gqa = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16"}  # grouped heads, small pages
    one = {"tokens_min": 1, "tokens_max": 1}
    return [
        # one sequence of the 7B shape, a small tree of drafts: latency counts
        {"name": "tree, 1 x 16 nodes", "op": "tree", "batch": 1, "nodes": 16, "prefix_min": 1024, "prefix_max": 1024,
         **mha},
        # a batch of the 7B shape, one prompt's length and more, each with a full tree
        {"name": "tree, 8 x 64 nodes", "op": "tree", "batch": 8, "nodes": 64, "prefix_min": 560, "prefix_max": 2000,
         **mha},
        # long contexts in small pages: what a larger server holds
        {"name": "tree, 32 x 25 nodes, 32/8 heads", "op": "tree", "batch": 32, "nodes": 25, "prefix_min": 500,
         "prefix_max": 8000, **gqa},
        # an odd group of seven heads of 64, a large tree
        {"name": "tree, 4 x 61 nodes, 28/4 heads", "op": "tree", "batch": 4, "nodes": 61, "prefix_min": 1000,
         "prefix_max": 4000, "heads": 28, "kv_heads": 4, "dim": 64, "page": 32, "type": "fp16"},
        # one stream of the 7B shape: its next token
        {"name": "window, 1 token", "op": "window", "batch": 1, **one, "prefix_min": 4000, "prefix_max": 4000,
         "window": 1024, "sinks": 4, **mha},
        # the largest decode batch of streams, some of them shorter than the window
        {"name": "window, 64 tokens", "op": "window", "batch": 64, **one, "prefix_min": 199, "prefix_max": 4000,
         "window": 1024, "sinks": 4, **mha},
        # a long window
        {"name": "window, 16 tokens, 32/8 heads", "op": "window", "batch": 16, **one, "prefix_min": 3000,
         "prefix_max": 16000, "window": 4096, "sinks": 16, **gqa},
        # the repository's prefill batch under a short window
        {"name": "window, 20 x 800 tokens", "op": "window", "batch": 20, "tokens_min": 800, "tokens_max": 800,
         "prefix_min": 0, "prefix_max": 0, "window": 256, "sinks": 4, **mha},
        # one long document
        {"name": "window, 16000 tokens, 32/8 heads", "op": "window", "batch": 1, "tokens_min": 16000,
         "tokens_max": 16000, "prefix_min": 0, "prefix_max": 0, "window": 1024, "sinks": 4, **gqa},
        # the tokens that a decode batch of 8 has chosen
        {"name": "logprobs, 8 rows", "op": "logprobs", "rows": 8, "vocab": 32003, "top": 5, "type": "fp16"},
        # the largest decode batch, 32-bit logits, as many alternatives as clients ask for
        {"name": "logprobs, 64 rows", "op": "logprobs", "rows": 64, "vocab": 32003, "top": 20, "type": "fp32"},
        # scoring the tokens of a whole prefill batch
        {"name": "logprobs, 16000 rows", "op": "logprobs", "rows": 16000, "vocab": 32003, "top": 5, "type": "fp16"},
    ]


def _size(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], often one that no tile divides."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.25:
        v = (v + 7) // 16 * 16
    return max(lo, min(hi, v))


def _shape(rng):
    heads, kv_heads = rng.choice(((32, 32), (32, 8), (28, 4), (16, 16), (40, 8), (8, 1), (12, 3)))
    return {"heads": heads, "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128)),
            "page": rng.choice((8, 16, 32, 64, 256)), "type": rng.choice(("fp16", "bf16"))}


def draw(rng):
    op = rng.choice(("tree", "window", "window", "logprobs"))
    if op == "logprobs":
        case = {"op": op, "rows": _size(rng, 1, 16000), "vocab": _size(rng, 1000, 160001), "top": rng.randint(0, 20),
                "type": rng.choice(("fp16", "bf16", "fp32"))}
        while case["rows"] > 1 and case["rows"] * case["vocab"] * BYTES[case["type"]] > 1 << 30:
            case["rows"] //= 2
        return case
    longest = _size(rng, 16, 16000)
    case = {"op": op, "batch": _size(rng, 1, 64), "prefix_min": rng.randint(0, longest), "prefix_max": longest,
            **_shape(rng)}
    if op == "tree":
        case["nodes"] = _size(rng, 1, 128)
    else:
        most = 1 if rng.random() < 0.5 else _size(rng, 2, 4000)
        case["tokens_min"], case["tokens_max"] = (most if rng.random() < 0.5 else 1), most
        case["window"] = _size(rng, 16, 4096)
        case["sinks"] = rng.choice((0, 1, 4, 16, 65))
    while case["batch"] > 1 and (work(case)["flops"] > 2e11 or work(case)["bytes"] > 1e9
                                 or _held(case) > 5e9):
        case["batch"] //= 2
    return case


def _spread(case, key):
    """One length for each sequence, spread over the case's (least, most)."""
    lo, hi = case[key + "_min"], case[key + "_max"]
    return [lo + int((hi - lo) * ((i * 0.6180339887 + 0.5) % 1.0) + 0.5) for i in range(case["batch"])]


def _lengths(case):
    """(new tokens, tokens before them) of each sequence."""
    new = [case["nodes"]] * case["batch"] if case["op"] == "tree" else _spread(case, "tokens")
    return new, _spread(case, "prefix")


def _held(case):
    """Bytes of the cache that holds every token of every sequence."""
    new, prefix = _lengths(case)
    return (sum(new) + sum(prefix)) * case["kv_heads"] * case["dim"] * 2 * BYTES[case["type"]]


def work(case):
    b = BYTES[case["type"]]
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * v * b + n * (8 + 4 + 4 + k * 12), "flops": 6 * n * v}
    new, prefix = _lengths(case)
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    rows = 2 * sum(new) * h * d * b  # the queries in, their outputs out
    if case["op"] == "tree":
        keys = sum(n + p for n, p in zip(new, prefix))
        pairs = sum(n * (p + 1) for n, p in zip(new, prefix))  # every node sees the prefix and itself
        return {"bytes": rows + keys * hkv * d * 2 * b + sum(n * n for n in new), "flops": 4 * d * h * pairs}
    w, s = case["window"], case["sinks"]
    keys = pairs = 0
    for n, p in zip(new, prefix):
        first = max(0, p - w + 1)  # the first key that the first query's window holds
        keys += n + p - first + min(s, first)
        # query at position t: its window, and the sinks before the window
        low = min(n, max(0, w - p))  # queries whose window starts at the first token
        pairs += low * p + low * (low + 1) // 2
        for t in range(p + low, min(p + n, w + s)):
            pairs += w + min(s, t - w + 1)
        pairs += max(0, n - max(low, min(n, w + s - p))) * (w + s)
    return {"bytes": rows + keys * hkv * d * 2 * b, "flops": 4 * d * h * pairs}


# ------------------------------------------------------------------ inputs
def _parents(n, g):
    """A tree of n drafts: each one's parent (-1: the last token of the cache) among the few before it."""
    back = (torch.rand(n, generator=g) ** 2 * 6).long()
    return [max(-1, i - 1 - int(back[i])) for i in range(n)]


def _ancestors(n, g):
    """bool [n, n]: what each draft sees of the others, itself and those that it follows."""
    seen = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(_parents(n, g)):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    if case["op"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        logits = torch.empty(n, v, dtype=dtype, device="cuda")
        for i in range(0, n, 2048):  # a language model's: wide, and a few tokens far above the others
            part = torch.randn(min(2048, n - i), v, generator=g, device="cuda").mul_(2.5)
            hot = torch.randint(0, v, (part.shape[0], 4), generator=g, device="cuda")
            part.scatter_add_(1, hot, torch.rand(hot.shape, generator=g, device="cuda") * 12.0)
            logits[i:i + part.shape[0]] = part
        # most tokens are likely ones, the others any
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.7, logits.argmax(1),
                          torch.randint(0, v, (n,), generator=g, device="cuda"))
        return {"op": "logprobs", "logits": logits, "ids": ids, "top": case["top"]}
    new, prefix = _lengths(case)
    h, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    total = sum(new)
    ctx = [n + p for n, p in zip(new, prefix)]
    pages = [-(-c // page) for c in ctx]
    pool = sum(pages) + 3
    order = torch.randperm(pool, generator=g, device="cuda").tolist()
    table = torch.zeros(len(ctx), max(pages), dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    offsets = [sum(new[:i]) for i in range(len(new))]
    q = torch.randn(total, h, d, generator=g, device="cuda")
    q *= torch.exp(torch.randn(total, h, 1, generator=g, device="cuda") * 0.5)  # some rows look at few keys
    k = torch.randn(pool, page, hkv, d, generator=g, device="cuda", dtype=dtype)
    v = torch.randn(pool, page, hkv, d, generator=g, device="cuda", dtype=dtype)
    s = {"op": case["op"], "q": q.to(dtype), "k": k, "v": v, "table": table.cuda(), "scale": d ** -0.5,
         "groups": h // hkv, "new": new, "ctx": ctx,
         "ctx_gpu": torch.tensor(ctx, dtype=torch.int32, device="cuda"),
         "new_gpu": torch.tensor(new, dtype=torch.int32, device="cuda"),
         "offsets": torch.tensor(offsets, dtype=torch.int32, device="cuda")}
    if case["op"] == "tree":
        cpu = torch.Generator().manual_seed(seed)
        s["mask"] = torch.cat([_ancestors(n, cpu) for n in new]).cuda()  # all trees have the same size
    else:
        s["window"], s["sinks"] = case["window"], case["sinks"]
    return s


# ------------------------------------------------------------- plain forms
def _gather(s, i, first, last):
    """Keys and values first .. last - 1 of sequence i as fp32 [Hkv, n, D]."""
    page = s["k"].shape[1]
    at = torch.arange(first, last, device="cuda")
    block = s["table"][i].long()[at // page]
    return (s["k"][block, at % page].float().transpose(0, 1), s["v"][block, at % page].float().transpose(0, 1))


def _softmax_rows(s, q, k, v, seen):
    """Attention of q [n, H, D] over k, v [Hkv, m, D] where seen [n, m]."""
    n, h, d = q.shape
    hkv = k.shape[0]
    x = q.float().view(n, hkv, h // hkv, d).permute(1, 2, 0, 3)  # [Hkv, G, n, D]
    score = (x @ k.transpose(1, 2)[:, None]) * s["scale"]
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v[:, None]) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(2, 0, 1, 3).reshape(n, h, d).to(q.dtype)


def _plain_tree(s):
    out, row = torch.empty_like(s["q"]), 0
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        k, v = _gather(s, i, 0, c)
        seen = torch.ones(n, c, dtype=torch.bool, device="cuda")
        seen[:, c - n:] = s["mask"][row:row + n, :n]
        out[row:row + n] = _softmax_rows(s, s["q"][row:row + n], k, v, seen)
        row += n
    return out


def _plain_window(s):
    out, row, w, sinks = torch.empty_like(s["q"]), 0, s["window"], s["sinks"]
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        for a in range(0, n, CHUNK):
            m = min(CHUNK, n - a)
            p0 = c - n + a  # the position of the first query
            first, last = max(0, p0 - w + 1), p0 + m
            k, v = _gather(s, i, first, last)
            key = torch.arange(first, last, device="cuda")
            if min(sinks, first) > 0:
                ks, vs = _gather(s, i, 0, min(sinks, first))
                k, v = torch.cat([ks, k], 1), torch.cat([vs, v], 1)
                key = torch.cat([torch.arange(min(sinks, first), device="cuda"), key])
            pos = torch.arange(p0, p0 + m, device="cuda")[:, None]
            seen = (key <= pos) & ((key > pos - w) | (key < sinks))
            out[row + a:row + a + m] = _softmax_rows(s, s["q"][row + a:row + a + m], k, v, seen)
        row += n
    return out


def _plain_logprobs(logits, ids, top):
    n, v = logits.shape
    outs = []
    index = torch.arange(v, device="cuda")
    for i in range(0, n, 1024):
        x = logits[i:i + 1024].float()
        shifted = x - x.amax(-1, keepdim=True)
        e = torch.exp(shifted)
        total = e.sum(-1, keepdim=True)
        lse = torch.log(total)
        entropy = (lse - (shifted * e).sum(-1, keepdim=True) / total).squeeze(-1)
        logp = (shifted.gather(1, ids[i:i + 1024, None]) - lse).squeeze(-1)
        # one whole number for each logit and its place, larger for a larger logit and, of equal ones, for the first
        bits = x.view(torch.int32).long()
        bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        best = torch.topk((bits << 32) + (v - 1 - index), top, dim=1).values
        top_ids = v - 1 - (best & 0xFFFFFFFF)
        outs.append((logp, entropy, top_ids, shifted.gather(1, top_ids) - lse))
    return tuple(torch.cat(parts) for parts in zip(*outs))


# ----------------------------------------------------------------- one pass
_modules = None


def _package():
    """(paged_attention, logprobs) of nanopointllm_b200; its folder has a hyphen, so it is registered by hand."""
    global _modules
    if _modules is None:
        if "nanopointllm_b200" not in sys.modules:
            folder = pathlib.Path(__file__).resolve().parent.parent / "nano-pointllm_b200"
            spec = importlib.util.spec_from_file_location("nanopointllm_b200", folder / "__init__.py",
                                                          submodule_search_locations=[str(folder)])
            module = importlib.util.module_from_spec(spec)
            sys.modules["nanopointllm_b200"] = module
            spec.loader.exec_module(module)
        _modules = (importlib.import_module("nanopointllm_b200.paged_attention"),
                    importlib.import_module("nanopointllm_b200.logprobs"))
    return _modules


def run(state):
    s, op = state, state["op"]
    if own:
        attention, scores = _package()
        if op == "logprobs":
            r = scores.token_logprobs(s["logits"], s["ids"], top_k=s["top"])
            return r.logprobs, r.entropy, r.top_ids, r.top_logprobs
        if op == "tree":
            return attention.paged_tree_attention(s["q"], s["k"], s["v"], s["table"], s["ctx_gpu"], s["new_gpu"],
                                                  s["offsets"], s["scale"], s["groups"], s["mask"],
                                                  max_q_len=max(s["new"]))
        if max(s["new"]) == 1:  # one token of each sequence
            return attention.paged_window_attention(s["q"], s["k"], s["v"], s["table"], s["ctx_gpu"], None, None,
                                                    s["scale"], s["groups"], s["window"], s["sinks"])
        return attention.paged_window_attention(s["q"], s["k"], s["v"], s["table"], s["ctx_gpu"], s["new_gpu"],
                                                s["offsets"], s["scale"], s["groups"], s["window"], s["sinks"],
                                                max_q_len=max(s["new"]))
    if op == "logprobs":
        return _plain_logprobs(s["logits"], s["ids"], s["top"])
    return _plain_tree(s) if op == "tree" else _plain_window(s)


# -------------------------------------------------------------------- exact
def _exact_sequence(s, i, start, mask_of):
    """Sequence i's outputs in 64 bits, a few queries at a time over all of its keys; mask_of(queries, keys) says
    what is seen."""
    n, c, g = s["new"][i], s["ctx"][i], s["groups"]
    page, hkv, d = s["k"].shape[1:]
    used = s["table"][i, :-(-c // page)].long()
    keys = s["k"][used].reshape(-1, hkv, d)[:c].double()
    values = s["v"][used].reshape(-1, hkv, d)[:c].double()
    q = s["q"][start:start + n].double()
    out = torch.zeros_like(q)
    step = max(1, min(n, int(2.5e8) // max(1, c * g)))
    for a in range(0, n, step):
        rows = torch.arange(a, min(n, a + step), device="cuda")
        hidden = ~mask_of(rows, torch.arange(c, device="cuda"))
        for h in range(q.shape[1]):
            z = (q[rows, h] @ keys[:, h // g].t()) * s["scale"]
            z[hidden] = -math.inf
            p = torch.softmax(z, -1)
            out[rows, h] = torch.nan_to_num(p) @ values[:, h // g]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        parts = []
        for i in range(0, case["rows"], 512):
            x = s["logits"][i:i + 512].double()
            lp = torch.log_softmax(x, -1)
            p = lp.exp()
            order = torch.sort(s["logits"][i:i + 512].float(), dim=-1, descending=True, stable=True).indices
            order = order[:, :case["top"]]
            parts.append((lp.gather(1, s["ids"][i:i + 512, None])[:, 0], -(p * lp).sum(-1), order,
                          lp.gather(1, order)))
        return tuple(torch.cat(p) for p in zip(*parts))
    outs, start = [], 0
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        if case["op"] == "tree":
            seen = s["mask"][start:start + n]

            def mask_of(rows, keys, seen=seen, before=c - n):
                inside = torch.nn.functional.pad(seen[rows], (before, 0), value=True)
                return inside[:, :keys.numel()]
        else:
            def mask_of(rows, keys, before=c - n):
                distance = (before + rows)[:, None] - keys[None]
                return (distance >= 0) & ((distance < case["window"]) | (keys[None] < case["sinks"]))
        outs.append(_exact_sequence(s, i, start, mask_of))
        start += n
    return torch.cat(outs)
