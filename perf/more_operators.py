"""The operators that score and serve texts from a paged cache of 16-bit values, as
cases that a timing program can list, draw, prepare, run and check.

* ``append``: RoPE of q and k, k and v stored by the slot map
  (``kernels.kv16.kv16_append``);
* ``attention``: attention over the cache -- one new token per request, chunks of
  prompts behind a context, whole prompts -- whose scores may be capped by a
  tanh or carry a bias for the distance, and whose rows may see a sliding window, a
  document or a prefix (``kernels.kv16.kv16_attention``);
* ``logprobs``: the log-probabilities of given tokens under the output projection,
  without its logits (``kernels.logprobs.token_logprobs``).

``run`` computes them in elementary torch operations, or with ``own`` set by the
framework's kernels.  Both take the same state.  The cache of a layer is one tensor
``[pages, kv heads, 2, page size, head size]``: K and V of a page and head.

The model's sizes are those of the Qwen2-7B configuration (28 / 4 heads of
128, hidden size 3584, vocabulary 152064); the others are generic.
"""
import math
import os
import sys

import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, HIDDEN, VOCAB, THETA = 28, 4, 128, 3584, 152064, 1e6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _framework():
    # The package's folder name is no Python identifier: its parts are imported from inside it.
    pkg = os.path.abspath("qwen2-7b-triton_engine_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from kernels import kv16, logprobs
    return kv16, logprobs


def listed():
    heads = {"heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM}
    plain = {"softcap": 0.0, "slopes": False, "window": 0, "documents": 0, "prefix": False}
    return [
        # The new tokens of a decode step.
        {"name": "append_t64", "kind": "append", "tokens": 64, "max_pos": 4096, "dtype": "fp16", "page": 64, **heads},
        # Prompts of ragged length, small pages.
        {"name": "append_t2011", "kind": "append", "tokens": 2011, "max_pos": 4096, "dtype": "bf16", "page": 16, **heads},
        # A single sequence: the smallest call, where latency counts.
        {"name": "decode_b1", "kind": "attention", "requests": 1, "longest": 1100, "chunk": 1, "dtype": "fp16", "page": 64,
         **heads, **plain},
        # A serving batch with lengths from a few tokens to thousands.
        {"name": "decode_b64", "kind": "attention", "requests": 64, "longest": 4096, "chunk": 1, "dtype": "fp16", "page": 64,
         **heads, **plain},
        # Long contexts of a layer with a sliding window and capped scores, eight kv heads, small pages.
        {"name": "decode_window", "kind": "attention", "requests": 8, "longest": 32768, "chunk": 1, "dtype": "bf16", "page": 16,
         "heads": 32, "kv_heads": 8, "head_dim": 128, **plain, "softcap": 50.0, "window": 4096},
        # Chunks of long prompts behind thousands of cached tokens, heads of 64, a bias for the distance.
        {"name": "chunks_b3", "kind": "attention", "requests": 3, "longest": 4000, "chunk": 389, "dtype": "fp16", "page": 32,
         "heads": 14, "kv_heads": 2, "head_dim": 64, **plain, "slopes": True},
        # Short instructions, each followed by an answer: all tokens of an instruction see each other.
        {"name": "prefix_b5", "kind": "attention", "requests": 5, "longest": 700, "chunk": 700, "dtype": "fp16", "page": 64,
         "heads": 32, "kv_heads": 8, "head_dim": 128, **plain, "prefix": True},
        # Texts packed into one sequence to be scored together, capped scores.
        {"name": "packed_s2500", "kind": "attention", "requests": 1, "longest": 2500, "chunk": 2500, "dtype": "bf16", "page": 64,
         "heads": 16, "kv_heads": 16, "head_dim": 128, **plain, "softcap": 30.0, "documents": 9},
        # A whole long prompt of ragged length: the largest.
        {"name": "prompt_s6001", "kind": "attention", "requests": 1, "longest": 6001, "chunk": 6001, "dtype": "fp16", "page": 64,
         **heads, **plain},
        # The token that a single sequence took.
        {"name": "logprobs_t1", "kind": "logprobs", "tokens": 1, "vocab": VOCAB, "hidden": HIDDEN, "dtype": "fp16"},
        # The tokens of a serving batch, an odd vocabulary.
        {"name": "logprobs_t61", "kind": "logprobs", "tokens": 61, "vocab": 50257, "hidden": 4096, "dtype": "bf16"},
        # A text to be scored.
        {"name": "logprobs_t2047", "kind": "logprobs", "tokens": 2047, "vocab": VOCAB, "hidden": HIDDEN, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (heads, kv heads, head size): the model's, then groups of one to sixteen query heads
_LAYOUTS = ((HEADS, KV_HEADS, HEAD_DIM), (HEADS, KV_HEADS, HEAD_DIM), (32, 8, 128), (14, 2, 64), (16, 1, 128), (12, 12, 64))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "attention", "logprobs", "logprobs"])
    dtype = rng.choice(["fp16", "fp16", "bf16"])
    if kind == "logprobs":
        return {"kind": kind, "tokens": _log_int(rng, 1, 2047), "vocab": _log_int(rng, 1000, VOCAB),
                "hidden": 64 * rng.randint(4, HIDDEN // 64), "dtype": dtype}
    heads, kv_heads, head_dim = rng.choice(_LAYOUTS)
    case = {"kind": kind, "dtype": dtype, "page": rng.choice([16, 32, 64, 128]), "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim}
    if kind == "append":
        return {**case, "tokens": _log_int(rng, 1, 2048), "max_pos": _log_int(rng, 2048, 8192)}
    case.update(softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.25,
                window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]))
    if rng.random() < 0.5:      # one token for each request; at most the cache of the largest listed batch
        requests = _log_int(rng, 1, 64)
        most = 64 * 4096 * KV_HEADS * HEAD_DIM // (requests * kv_heads * head_dim)
        return {**case, "requests": requests, "longest": _log_int(rng, 1, min(16384, most)), "chunk": 1, "documents": 0,
                "prefix": False}
    requests, longest = rng.randint(1, 4), _log_int(rng, 33, 2500)
    return {**case, "requests": requests, "longest": longest, "chunk": _log_int(rng, 2, longest),
            "documents": rng.choice([0, 0, rng.randint(1, 12)]), "prefix": rng.random() < 0.25}


# ---- inputs ----------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(case, seed):
    """(length, new tokens) of each request after the step: the first is the
    longest with the largest chunk, the others' lengths are spread from one token up."""
    g = torch.Generator()
    g.manual_seed(seed)
    part = torch.rand(case["requests"], generator=g).tolist()
    new = [max(1, case["chunk"] - case["chunk"] * i // (2 * case["requests"])) for i in range(case["requests"])]
    return [max(m, int(case["longest"] * (1.0 if i == 0 else part[i]))) for i, m in enumerate(new)], new


def _tables(lengths, page, width, g):
    """Block tables of the requests, pages handed out in random order; (tables, pages)."""
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, pages


def _rope_tables(max_pos, head_dim):
    inv = 1.0 / (THETA ** (torch.arange(0, head_dim, 2, device="cuda", dtype=torch.float32) / head_dim))
    f = torch.outer(torch.arange(max_pos, device="cuda", dtype=torch.float32), inv)
    return torch.cat((f, f), -1).cos(), torch.cat((f, f), -1).sin()


def _append_inputs(case, seed):
    g = _generator(seed)
    heads, kvh, hd, tokens, page = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"], case["page"]
    qkv = torch.randn((tokens, (heads + 2 * kvh) * hd), generator=g, device="cuda")
    # Keys have channels that are much larger than the others.
    qkv[:, heads * hd:(heads + kvh) * hd] *= 1.0 + 3.0 * torch.rand(kvh * hd, generator=g, device="cuda").pow(8)
    pages = -(-tokens // page) + 3
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].sort().values.to(torch.int32)
    positions = torch.randint(0, case["max_pos"], (tokens,), generator=g, device="cuda", dtype=torch.int32)
    data = torch.randn((pages, kvh, 2, page, hd), generator=g, device="cuda").to(DTYPES[case["dtype"]])
    return qkv.to(DTYPES[case["dtype"]]), slots, positions, data


def _attention_inputs(case, seed):
    g = _generator(seed)
    heads, kvh, hd, page, dtype = (case[k] for k in ("heads", "kv_heads", "head_dim", "page", "dtype"))
    lengths, new = _lengths(case, seed)
    tables, pages = _tables(lengths, page, -(-max(lengths) // page) + 1, g)
    # Capped scores are those that would grow large.
    gain = 6.0 if case["softcap"] else 1.0
    q = (torch.randn((sum(new), heads * hd), generator=g, device="cuda") * gain).to(DTYPES[dtype])
    data = torch.randn((pages, kvh, 2, page, hd), generator=g, device="cuda")
    data[:, :, 0] *= 1.0 + 3.0 * torch.rand((kvh, 1, hd), generator=g, device="cuda").pow(8)
    slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if case["slopes"] else None
    prefix = first = None
    if case["prefix"]:
        share = torch.rand(len(lengths), generator=g, device="cuda")
        prefix = (share * _i32(lengths)).to(torch.int32)
    if case["documents"]:
        starts = []
        for n, m in zip(lengths, new):
            # where the documents of this request begin, the first at 0
            cuts = torch.cat([_i32([0]), torch.randint(0, n, (case["documents"],), generator=g, device="cuda")]).sort().values
            pos = torch.arange(n - m, n, device="cuda")
            starts.append(cuts[torch.searchsorted(cuts, pos, right=True) - 1])
        first = torch.cat(starts).to(torch.int32)
    return q, lengths, new, tables, data.to(DTYPES[dtype]), slopes, prefix, first


def _logprobs_inputs(case, seed):
    g = _generator(seed)
    T, V, K, dtype = case["tokens"], case["vocab"], case["hidden"], DTYPES[case["dtype"]]
    hidden = torch.randn((T, K), generator=g, device="cuda")
    weight = (torch.randn((V, K), generator=g, device="cuda") * (2.0 / math.sqrt(K))).to(dtype)
    targets = torch.randint(0, V, (T,), generator=g, device="cuda")
    # A text's tokens are likelier than others: one hidden state in three points along its token's row.
    hidden[::3] += 1.5 * weight[targets[::3]].float()
    hidden = hidden.to(dtype)
    return hidden, weight, targets


def prepare(case, seed):
    kind = case["kind"]
    if kind == "append":
        qkv, slots, positions, data = _append_inputs(case, seed)
        cos, sin = _rope_tables(case["max_pos"], case["head_dim"])
        return {"kind": kind, "heads": case["heads"], "qkv": qkv, "slots": slots, "positions": positions, "data": data, "cos": cos,
                "sin": sin}
    if kind == "attention":
        q, lengths, new, tables, data, slopes, prefix, first = _attention_inputs(case, seed)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        return {"kind": kind, "heads": case["heads"], "q": q, "data": data, "tables": tables, "lengths": _i32(lengths),
                "starts": _i32(starts), "longest": max(lengths), "most_new": max(new), "slopes": slopes, "prefix": prefix,
                "first": first, "softcap": case["softcap"] or None, "window": case["window"] or None}
    hidden, weight, targets = _logprobs_inputs(case, seed)
    return {"kind": kind, "hidden": hidden, "weight": weight, "targets": targets}


# ---- one pass ----------------------------------------------------------------------


def run(state):
    return _RUN[state["kind"]](state)


def _rotate_half(x):
    half = x.shape[-1] // 2
    return torch.cat((-x[..., half:], x[..., :half]), -1)


def _run_append(s):
    heads, data = s["heads"], s["data"]
    if own:
        kv16, _ = _framework()
        cache = kv16.Kv16Cache.of(data)
        q = kv16.kv16_append(s["qkv"], cache, s["slots"], s["positions"], s["cos"], s["sin"], heads)
        return {"q": q, "cache": cache.data}
    qkv, slots = s["qkv"], s["slots"].long()
    _, kvh, _, page, hd = data.shape
    cos, sin = s["cos"][s["positions"].long()].unsqueeze(1), s["sin"][s["positions"].long()].unsqueeze(1)
    qk = qkv[:, :(heads + kvh) * hd].float().view(-1, heads + kvh, hd)
    qk = (qk * cos + _rotate_half(qk) * sin).to(qkv.dtype)
    data[slots // page, :, 0, slots % page] = qk[:, heads:]
    data[slots // page, :, 1, slots % page] = qkv[:, (heads + kvh) * hd:].view(-1, kvh, hd)
    return {"q": qk[:, :heads].reshape(-1, heads * hd), "cache": data}


def _run_attention(s):
    q, data = s["q"], s["data"]
    if own:
        kv16, _ = _framework()
        return kv16.kv16_attention(q, kv16.Kv16Cache.of(data), s["tables"], s["lengths"], s["starts"], s["most_new"],
                                   softcap=s["softcap"], slopes=s["slopes"], window=s["window"], prefix=s["prefix"],
                                   first=s["first"])
    heads = s["heads"]
    _, kvh, _, page, hd = data.shape
    groups, B, L, S = heads // kvh, s["tables"].shape[0], s["longest"], s["most_new"]
    lengths, starts = s["lengths"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    # every request's rows and keys, padded to the longest
    key = torch.arange(L, device="cuda")
    number = s["tables"].long().clamp(min=0)[:, key // page]                                         # [B, L]
    k, v = (data[number, :, i, key % page].float().permute(0, 2, 1, 3).reshape(B * kvh, L, hd) for i in (0, 1))
    row = torch.arange(S, device="cuda")
    at = (starts[:-1, None] + row).clamp(max=q.shape[0] - 1)                                         # [B, S]
    pos = (lengths - new)[:, None] + row                                                             # [B, S]
    qs = q.float().view(-1, kvh, groups, hd)[at].permute(0, 2, 3, 1, 4).reshape(B * kvh, groups * S, hd)
    scores = torch.bmm(qs, k.transpose(1, 2).contiguous()).div_(math.sqrt(hd)).view(B, kvh, groups, S, L)
    if s["softcap"]:
        scores = s["softcap"] * torch.tanh(scores / s["softcap"])
    if s["slopes"] is not None:
        scores -= s["slopes"].view(kvh, groups, 1, 1) * (pos[..., None] - key).abs()[:, None, None]
    end = pos + 1
    if s["prefix"] is not None:
        end = torch.maximum(end, s["prefix"].long()[:, None])
    end = torch.minimum(end, lengths[:, None])[..., None]                                            # [B, S, 1]
    seen = key < end
    if s["window"] is not None:
        seen &= key > pos[..., None] - s["window"]
    if s["first"] is not None:
        seen &= key >= s["first"].long()[at][..., None]
    scores = scores.masked_fill_(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)                          # a row that sees nothing gives zeros
    out = torch.bmm(p.view(B * kvh, groups * S, L), v).view(B, kvh, groups, S, hd)
    out = out.permute(0, 3, 1, 2, 4).reshape(B * S, heads * hd)
    b = torch.searchsorted(starts[1:], torch.arange(q.shape[0], device="cuda"), right=True)
    return out[b * S + torch.arange(q.shape[0], device="cuda") - starts[b]].to(q.dtype)


def _run_logprobs(s):
    if own:
        _, logprobs = _framework()
        chosen, total = logprobs.token_logprobs(s["hidden"], s["weight"], s["targets"])
        return {"logprobs": chosen, "logsumexp": total}
    logits = torch.mm(s["hidden"].float(), s["weight"].float().t())
    top = logits.amax(-1, keepdim=True)
    total = top + torch.exp(logits - top).sum(-1, keepdim=True).log()
    return {"logprobs": (logits.gather(1, s["targets"][:, None]) - total)[:, 0], "logsumexp": total[:, 0]}


_RUN = {"append": _run_append, "attention": _run_attention, "logprobs": _run_logprobs}


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        T, V, K = case["tokens"], case["vocab"], case["hidden"]
        return {"bytes": 2 * K * (T + V) + 16 * T, "flops": 2 * T * V * K + 3 * T * V}
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        T = case["tokens"]
        # qkv in, q and the new keys and values out, the positions' cos and sin
        return {"bytes": 2 * T * (2 * heads + 4 * kvh) * hd + 8 * T * hd + 8 * T, "flops": 6 * T * (heads + kvh) * hd}
    pairs = tokens = 0
    lengths, new = _lengths(case, 1)
    for n, m in zip(lengths, new):
        pos = torch.arange(n - m, n)
        low = (pos + 1 - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(pos)
        end = pos + 1
        if case["prefix"]:
            end = end.clamp(min=n // 2)
        if case["documents"]:      # on average a document more than are cut
            low = torch.maximum(low, pos - n // (case["documents"] + 1)).clamp(min=0)
        pairs += int((end - low).clamp(min=0).sum())
        tokens += n - int(low.min())
    return {"bytes": 4 * kvh * hd * tokens + 4 * sum(new) * heads * hd, "flops": 4 * heads * hd * pairs}


# ---- the same in 64 bits, from the definitions ---------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind == "append":
        return _exact_append(case, seed)
    if kind == "attention":
        return _exact_attention(case, seed)
    return _exact_logprobs(case, seed)


def _exact_append(case, seed):
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    qkv, slots, positions, data = _append_inputs(case, seed)
    cos, sin = (t[positions.long()].double()[:, None, :hd // 2] for t in _rope_tables(case["max_pos"], hd))
    x = qkv.double().view(-1, heads + 2 * kvh, hd)
    a, b = x[:, :heads + kvh, :hd // 2], x[:, :heads + kvh, hd // 2:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    cache = data.double().permute(0, 3, 1, 2, 4).reshape(-1, kvh, 2, hd)          # by slots
    cache[slots.long()] = torch.stack((turned[:, heads:], x[:, heads + kvh:]), 2)
    cache = cache.view(-1, page, kvh, 2, hd).permute(0, 2, 3, 1, 4).contiguous()
    return {"q": turned[:, :heads].reshape(-1, heads * hd), "cache": cache}


def _exact_attention(case, seed):
    q, lengths, new, tables, data, slopes, prefix, first = _attention_inputs(case, seed)
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    out, at = [], 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        pages = data[tables[b, :-(-n // case["page"])].long()]
        rows = q[at:at + m].double().view(m, heads, hd)
        i, j = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = j <= i
        if prefix is not None:
            seen = seen | (j < prefix[b])
        if case["window"]:
            seen = seen & (i - j < case["window"])
        if first is not None:
            seen = seen & (j >= first[at:at + m, None])
        o = torch.empty_like(rows)
        for h in range(heads):
            k, v = (pages[:, h // (heads // kvh), c].reshape(-1, hd)[:n].double() for c in (0, 1))
            scores = rows[:, h] @ k.t().contiguous() / math.sqrt(hd)
            if case["softcap"]:
                scores = case["softcap"] * torch.tanh(scores / case["softcap"])
            if slopes is not None:
                scores = scores - slopes[h].double() * (i - j).abs()
            o[:, h] = torch.softmax(torch.where(seen, scores, -math.inf), -1) @ v
        o[~seen.any(1)] = 0.0
        out.append(o.view(m, -1))
        at += m
    return torch.cat(out)


def _exact_logprobs(case, seed):
    hidden, weight, targets = _logprobs_inputs(case, seed)
    x = hidden.double()
    parts = [torch.logsumexp(x @ w.double().t().contiguous(), 1) for w in weight.split(16384)]
    total = torch.logsumexp(torch.stack(parts), 0)
    return {"logprobs": (x * weight[targets].double()).sum(1) - total, "logsumexp": total}
