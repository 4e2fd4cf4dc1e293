"""The operators that serve many requests from one paged 4-bit cache, as cases
that a timing program can list, draw, prepare, run and check.

* ``step``: the block tables, slots and positions of a step's new tokens, from
  the requests' lengths (``kernels.paged.paged_step``);
* ``append``: RoPE of q and k, k and v quantised to 4 bits and stored by the
  slot map, then read back (``kernels.kv4.kv4_append``, ``kv4_gather``);
* ``attention``: attention over the cache -- one new token per request, or
  chunks of prompts with the context before them (``kernels.kv4.kv4_attention``);
* ``logits``: penalties for repeated tokens, biases, a grammar's mask and the
  greedy token (``kernels.logits.process_logits``).

``run`` computes them in elementary torch operations, or with ``own`` set by the
framework's kernels.  Both take the same state: the packed cache among it,
whose format is written out in ``_pack`` and ``_unpack``.

The model's sizes are those of the Qwen2-7B configuration (28 / 4 heads of
128, vocabulary 152064); the others are generic.
"""
import math
import os
import sys

import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, VOCAB, THETA = 28, 4, 128, 152064, 1e6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _framework():
    # The package's folder name is no Python identifier: its parts are imported from inside it.
    pkg = os.path.abspath("qwen2-7b-triton_engine_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from kernels import kv4, logits, paged
    return kv4, logits, paged


def listed():
    model = {"heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM, "dtype": "fp16"}
    cache = {"page": 64, "group": 64}
    return [
        # One decode step of a serving batch: a new token for each request.
        {"name": "step_b64", "kind": "step", "requests": 64, "longest": 4096, "tokens": 64, "page": 64},
        # Prompts of many requests at once, beside requests that decode.
        {"name": "step_prompts", "kind": "step", "requests": 256, "longest": 8192, "tokens": 16384, "page": 16},
        # The new tokens of a decode step.
        {"name": "append_t64", "kind": "append", "tokens": 64, "max_pos": 4096, **model, **cache},
        # An ordinary prompt of ragged length.
        {"name": "append_t2011", "kind": "append", "tokens": 2011, "max_pos": 4096, **model, **cache},
        # A single sequence: the smallest call, where latency counts.
        {"name": "decode_b1", "kind": "attention", "requests": 1, "longest": 1100, "chunk": 1, **model, **cache},
        # A serving batch with lengths from a few tokens to thousands.
        {"name": "decode_b64", "kind": "attention", "requests": 64, "longest": 4096, "chunk": 1, **model, **cache},
        # Two long contexts in small pages and groups, eight kv heads.
        {"name": "decode_long", "kind": "attention", "requests": 2, "longest": 32768, "chunk": 1, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "page": 16, "group": 32},
        # A whole prompt of ragged length.
        {"name": "prompt_s1777", "kind": "attention", "requests": 1, "longest": 1777, "chunk": 1777, **model, **cache},
        # Chunks of long prompts: a few hundred rows behind thousands of cached tokens, heads of 64.
        {"name": "chunks_b3", "kind": "attention", "requests": 3, "longest": 4000, "chunk": 389, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "dtype": "fp16", "page": 32, "group": 64},
        # The last step of a single sequence.
        {"name": "logits_b1", "kind": "logits", "requests": 1, "vocab": VOCAB, "history": 1200, "biases": 40,
         "mask": True, "dtype": "fp16"},
        # The last step of a serving batch.
        {"name": "logits_b64", "kind": "logits", "requests": 64, "vocab": VOCAB, "history": 4096, "biases": 100,
         "mask": True, "dtype": "fp16"},
        # Logits in 32 bits of an odd vocabulary, long histories, no grammar.
        {"name": "logits_b8_fp32", "kind": "logits", "requests": 8, "vocab": 50257, "history": 16000, "biases": 300,
         "mask": False, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (heads, kv heads, head size): the model's, then groups of one to sixteen query heads
_LAYOUTS = ((HEADS, KV_HEADS, HEAD_DIM), (HEADS, KV_HEADS, HEAD_DIM), (32, 8, 128), (14, 2, 64), (16, 1, 128), (12, 12, 64))


def draw(rng):
    kind = rng.choice(["step", "append", "attention", "attention", "attention", "logits"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "step":
        requests = _log_int(rng, 1, 256)
        return {"kind": kind, "requests": requests, "longest": _log_int(rng, 256, 8192),
                "tokens": _log_int(rng, requests, 16384), "page": page}
    if kind == "logits":
        requests = _log_int(rng, 1, 64)
        return {"kind": kind, "requests": requests, "vocab": _log_int(rng, 1000, VOCAB),
                "history": _log_int(rng, 16, 4096), "biases": rng.randint(0, 100), "mask": rng.random() < 0.6,
                "dtype": rng.choice(["fp16", "fp16", "bf16", "fp32"])}
    heads, kv_heads, head_dim = rng.choice(_LAYOUTS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": rng.choice(["fp16", "fp16", "bf16"]), "page": page,
            "group": rng.choice([32, 64, 64] + [128] * (head_dim == 128))}
    if kind == "append":
        return {**case, "tokens": _log_int(rng, 1, 2048), "max_pos": _log_int(rng, 2048, 8192)}
    if rng.random() < 0.6:      # one token for each request; at most the cache of the largest listed batch
        requests = _log_int(rng, 1, 64)
        most = 64 * 4096 * KV_HEADS * HEAD_DIM // (requests * kv_heads * head_dim)
        return {**case, "requests": requests, "longest": _log_int(rng, 1, min(16384, most)), "chunk": 1}
    requests, longest = rng.randint(1, 4), _log_int(rng, 33, 2048)
    return {**case, "requests": requests, "longest": longest, "chunk": _log_int(rng, 2, max(2, longest // requests))}


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
    pages = sum(held) + 8
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, pages, order[at:]


def _step_inputs(case, seed):
    """Lengths before the step and new tokens: `tokens` rows in all, the requests' shares uneven."""
    g = torch.Generator()
    g.manual_seed(seed)
    requests, page, longest = case["requests"], case["page"], case["longest"]
    left = case["tokens"] - requests
    cuts = sorted(torch.randint(0, left + 1, (requests - 1,), generator=g).tolist())
    new = [1 + b - a for a, b in zip([0] + cuts, cuts + [left])]
    lengths = [min(longest, int(longest * p)) for p in torch.rand(requests, generator=g).tolist()]
    width = -(-(longest + case["tokens"]) // page)
    gg = _generator(seed)
    tables, _, free = _tables(lengths, page, width, gg)
    more = sum(-(-(a + b) // page) + -(-a // page) for a, b in zip(lengths, new)) + 8
    free = torch.cat([free, free.numel() + torch.randperm(more, generator=gg, device="cuda").to(torch.int32) + sum(
        -(-n // page) for n in lengths)])
    return lengths, new, tables, free


def _rope_tables(max_pos, head_dim):
    inv = 1.0 / (THETA ** (torch.arange(0, head_dim, 2, device="cuda", dtype=torch.float32) / head_dim))
    f = torch.outer(torch.arange(max_pos, device="cuda", dtype=torch.float32), inv)
    return torch.cat((f, f), -1).cos(), torch.cat((f, f), -1).sin()


def _append_inputs(case, g):
    heads, kvh, hd, tokens = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
    qkv = torch.randn((tokens, (heads + 2 * kvh) * hd), generator=g, device="cuda")
    # Keys have channels that are much larger than the others.
    qkv[:, heads * hd:(heads + kvh) * hd] *= 1.0 + 3.0 * torch.rand(kvh * hd, generator=g, device="cuda").pow(8)
    pages = -(-tokens // case["page"]) + 3
    slots = torch.randperm(pages * case["page"], generator=g, device="cuda")[:tokens].sort().values.to(torch.int32)
    positions = torch.randint(0, case["max_pos"], (tokens,), generator=g, device="cuda", dtype=torch.int32)
    return qkv.to(DTYPES[case["dtype"]]), slots, positions, pages


def _attention_inputs(case, seed):
    """Queries, and the codes, scales and zeros of every slot of the cache."""
    g = _generator(seed)
    heads, kvh, hd, page, group = (case[k] for k in ("heads", "kv_heads", "head_dim", "page", "group"))
    lengths, new = _lengths(case, seed)
    width = -(-case["longest"] // page) + 1
    tables, pages, _ = _tables(lengths, page, width, g)
    q = torch.randn((sum(new), heads * hd), generator=g, device="cuda").to(DTYPES[case["dtype"]])
    parts = []
    for gain in (3.0, 0.0):
        x = torch.randn((pages * page, kvh, hd), generator=g, device="cuda")
        x *= 1.0 + gain * torch.rand((kvh, hd), generator=g, device="cuda").pow(8)
        parts.append(_quantise(x, group))
    return q, lengths, new, tables, pages, parts


def _logits_inputs(case, seed):
    g = _generator(seed)
    B, V, L = case["requests"], case["vocab"], case["history"]
    x = (torch.randn((B, V), generator=g, device="cuda") * 3.0).to(DTYPES[case["dtype"]])
    rand = lambda lo, hi: lo + (hi - lo) * torch.rand(B, generator=g, device="cuda")  # noqa: E731
    lengths = (rand(0.3, 1.0) * L).to(torch.int32).clamp(min=1)
    prompt = (lengths * rand(0.1, 0.9)).to(torch.int32)
    # Texts repeat themselves: two tokens in three come from a few hundred.
    often = torch.randint(0, V, (256,), generator=g, device="cuda")
    tokens = torch.randint(0, V, (B, L), generator=g, device="cuda")
    pick = torch.randint(0, 256, (B, L), generator=g, device="cuda")
    tokens = torch.where(pick < 170, often[pick], tokens)
    n = case["biases"]
    bias_tokens = torch.rand((B, V), generator=g, device="cuda").topk(n, dim=1).indices.to(torch.int32).reshape(-1)
    bias_start = torch.arange(B + 1, dtype=torch.int32, device="cuda") * n
    bias_values = torch.randn(B * n, generator=g, device="cuda") * 5.0
    words = -(-V // 32)
    mask = None
    if case["mask"]:
        word = lambda: torch.randint(-2**31, 2**31 - 1, (B, words), generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
        mask = word() & word()                              # a quarter of the tokens allowed
    return {"logits": x, "tokens": tokens, "lengths": lengths, "prompt_lens": prompt,
            "repetition": rand(1.0, 1.3), "presence": rand(0.0, 0.8), "frequency": rand(0.0, 0.5),
            "bias": (bias_start, bias_tokens, bias_values), "mask": mask}


def prepare(case, seed):
    kind = case["kind"]
    if kind == "step":
        lengths, new, tables, free = _step_inputs(case, seed)
        return {"kind": kind, "page": case["page"], "tokens": case["tokens"], "tables": tables, "free": free,
                "lengths": _i32(lengths + [free.numel()]), "new": _i32(new)}
    if kind == "append":
        qkv, slots, positions, pages = _append_inputs(case, _generator(seed))
        cos, sin = _rope_tables(case["max_pos"], case["head_dim"])
        meta = {k: case[k] for k in ("heads", "kv_heads", "head_dim", "page", "group")}
        data = torch.zeros((pages, case["kv_heads"], _block_bytes(case)), dtype=torch.uint8, device="cuda")
        return {"kind": kind, **meta, "qkv": qkv, "slots": slots, "positions": positions, "cos": cos, "sin": sin, "data": data}
    if kind == "attention":
        q, lengths, new, tables, pages, (k, v) = _attention_inputs(case, seed)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        meta = {k_: case[k_] for k_ in ("heads", "kv_heads", "head_dim", "page", "group")}
        return {"kind": kind, **meta, "q": q, "data": _pack(k, v, case, pages), "tables": tables, "lengths": _i32(lengths),
                "starts": _i32(starts), "longest": max(lengths), "most_new": max(new)}
    return {"kind": kind, **_logits_inputs(case, seed)}


# ---- the cache's format ------------------------------------------------------------


def _quantise(x, group):
    """Codes 0 .. 15, scales and zeros (fp16) of fp32 [n, heads, head_dim], by
    groups of columns: zero = fp16(min), scale = (max - zero) / 15 rounded up to
    seven significant bits (so that code * scale is exact in fp16)."""
    n, heads, hd = x.shape
    x = x.view(n, heads, hd // group, group)
    zero = x.amin(-1, keepdim=True).half()
    # divided by a tensor: by a number, torch multiplies with its rounded reciprocal
    r = ((x.amax(-1, keepdim=True) - zero.float()) / torch.full_like(x[..., :1], 15.0)).clamp(min=0.0).contiguous()
    r = ((r.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32)
    scale = torch.where(r < 2.0 ** -17, torch.ceil(r * 2.0 ** 24) * 2.0 ** -24, r).half()
    s = scale.float()
    codes = torch.round((x - zero.float()) / torch.where(s > 0, s, torch.ones_like(s))).clamp(0, 15) * (s > 0)
    return codes.to(torch.int32).view(n, heads, hd), scale.squeeze(-1), zero.squeeze(-1)


def _block_bytes(case):
    return case["page"] * (case["head_dim"] + 8 * (case["head_dim"] // case["group"]))


def _words(nibbles):
    """int32 words of [..., 8] codes, the first in the lowest four bits."""
    shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int64)
    word = (nibbles.to(torch.int64) << shift).sum(-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def _nibbles(words):
    shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    return (words.unsqueeze(-1) >> shift) & 15


# K words: columns 0, 2, 4, 6, 1, 3, 5, 7 from the lowest four bits up.
_K_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)


def _pack(k, v, case, pages):
    """uint8 [pages, kv heads, block]: a block holds K's words [token][4][head_dim / 32]
    (the word (t, s) is columns 32 s + 8 t ..), V's words [token / 4][head_dim / 8][token % 4],
    K's (scale, zero) [token][group] and V's [token / 4][group][scales, zeros][token % 4]."""
    kvh, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    groups = hd // case["group"]
    bytes_of = lambda t: t.contiguous().view(pages, kvh, -1).view(torch.uint8)  # noqa: E731
    kw = _words(k[0].view(pages, page, kvh, hd // 32, 4, 8)[..., list(_K_ORDER)]).permute(0, 2, 1, 4, 3)
    vw = _words(v[0].view(pages, page // 4, 4, kvh, hd // 8, 8)).permute(0, 3, 1, 4, 2)
    ks = torch.stack(k[1:], -1).view(pages, page, kvh, groups, 2).permute(0, 2, 1, 3, 4)
    vs = torch.stack(v[1:], -1).view(pages, page // 4, 4, kvh, groups, 2).permute(0, 3, 1, 4, 5, 2)
    return torch.cat([bytes_of(kw), bytes_of(vw), bytes_of(ks), bytes_of(vs)], -1).contiguous()


def _unpack(data, s):
    """fp32 values (k, v) [pages * page, kv heads, head_dim] of a packed cache."""
    pages, kvh = data.shape[:2]
    hd, page, group = s["head_dim"], s["page"], s["group"]
    groups, half = hd // group, page * hd // 2
    part = lambda lo, n, t: data[..., lo:lo + n].contiguous().view(t)  # noqa: E731
    kw = _nibbles(part(0, half, torch.int32).view(pages, kvh, page, 4, hd // 32))
    inverse = [_K_ORDER.index(c) for c in range(8)]
    kc = kw[..., inverse].permute(0, 2, 1, 4, 3, 5).reshape(-1, kvh, groups, group)
    vw = _nibbles(part(half, half, torch.int32).view(pages, kvh, page // 4, hd // 8, 4))
    vc = vw.permute(0, 2, 4, 1, 3, 5).reshape(-1, kvh, groups, group)
    ks = part(2 * half, 4 * page * groups, torch.float16).view(pages, kvh, page, groups, 2)
    ks = ks.permute(0, 2, 1, 3, 4).reshape(-1, kvh, groups, 2).float()
    vs = part(2 * half + 4 * page * groups, 4 * page * groups, torch.float16).view(pages, kvh, page // 4, groups, 2, 4)
    vs = vs.permute(0, 2, 5, 1, 3, 4).reshape(-1, kvh, groups, 2).float()
    value = lambda c, z: (c.float() * z[..., :1] + z[..., 1:]).reshape(-1, kvh, hd)  # noqa: E731
    return value(kc, ks), value(vc, vs)


# ---- one pass ----------------------------------------------------------------------


def run(state):
    return _RUN[state["kind"]](state)


def _run_step(s):
    if own:
        _, _, paged = _framework()
        tables = paged.PagedTables.of(s["tables"], s["lengths"], s["free"], page_size=s["page"])
        r = paged.paged_step(tables, s["new"], s["tokens"])
        return {"state": r.state, "query_start": r.query_start, "slots": r.slots, "positions": r.positions,
                "failed": r.failed, "tables": s["tables"]}
    page, rows, tables, free = s["page"], s["tokens"], s["tables"], s["free"]
    old, count, new = s["lengths"][:-1], s["lengths"][-1:], s["new"]
    ends = torch.cumsum(new, 0)
    room = ((old + new) <= tables.shape[1] * page) & (ends <= rows) & (new >= 0)
    held = (old + page - 1) // page
    need = torch.where(room, (old + new + page - 1) // page - held, 0)
    taken = torch.cumsum(need, 0)
    served = room & ((need == 0) | (taken <= count))
    query_start = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    row = torch.arange(rows, dtype=torch.int32, device="cuda")
    b = torch.searchsorted(ends, row, right=True).clamp(max=new.shape[0] - 1)
    pos = old[b] + row - query_start[b]
    fine = served[b] & (row < ends[-1])
    index = pos // page
    fresh = (taken - need)[b] + index - held[b]             # its page's place among the step's new ones
    top = (count - 1 - fresh).clamp(0, free.shape[0] - 1)
    index = torch.where(fine, index, 0)
    from_table = tables[b, index]
    number = torch.where(fine & (index >= held[b]), free[top], from_table)
    tables[b, index] = number
    slots = torch.where(fine, number * page + pos % page, -1)
    got = torch.where(served, new, 0)
    left = count - torch.where(served, need, 0).sum()
    return {"state": torch.cat([old + got, left]).to(torch.int32), "query_start": query_start,
            "slots": slots.to(torch.int32), "positions": torch.where(fine, pos, -1).to(torch.int32),
            "failed": (~served).to(torch.int32), "tables": tables}


def _rotate_half(x):
    half = x.shape[-1] // 2
    return torch.cat((-x[..., half:], x[..., :half]), -1)


def _run_append(s):
    heads, kvh, hd = s["heads"], s["kv_heads"], s["head_dim"]
    if own:
        kv4, _, _ = _framework()
        cache = kv4.Kv4Cache.of(s["data"], head_dim=hd, page_size=s["page"], group_size=s["group"])
        q = kv4.kv4_append(s["qkv"], cache, s["slots"], s["positions"], s["cos"], s["sin"], heads)
        k, v = kv4.kv4_gather(cache, s["slots"], dtype=s["qkv"].dtype)
        return {"q": q, "k": k, "v": v}
    qkv, slots = s["qkv"], s["slots"].long()
    cos, sin = s["cos"][s["positions"].long()].unsqueeze(1), s["sin"][s["positions"].long()].unsqueeze(1)
    qk = qkv[:, :(heads + kvh) * hd].float().view(-1, heads + kvh, hd)
    qk = qk * cos + _rotate_half(qk) * sin
    v = qkv[:, (heads + kvh) * hd:].float().view(-1, kvh, hd)
    parts = []
    for x in (qk[:, heads:].contiguous(), v.contiguous()):
        codes, scale, zero = _quantise(x, s["group"])
        # a cache of plain tensors: one byte a code, the scales and zeros beside them
        shape = (s["data"].shape[0] * s["page"], kvh)
        cache = (torch.zeros((*shape, hd), dtype=torch.uint8, device="cuda"),
                 torch.zeros((*shape, hd // s["group"], 2), dtype=torch.float16, device="cuda"))
        cache[0][slots] = codes.to(torch.uint8)
        cache[1][slots] = torch.stack((scale, zero), -1)
        c, z = cache[0][slots].float().view(-1, kvh, hd // s["group"], s["group"]), cache[1][slots].float()
        parts.append((c * z[..., :1] + z[..., 1:]).view(-1, kvh, hd).to(qkv.dtype))
    return {"q": qk[:, :heads].reshape(-1, heads * hd).to(qkv.dtype), "k": parts[0], "v": parts[1]}


def _run_attention(s):
    if own:
        kv4, _, _ = _framework()
        cache = kv4.Kv4Cache.of(s["data"], head_dim=s["head_dim"], page_size=s["page"], group_size=s["group"])
        return kv4.kv4_attention(s["q"], cache, s["tables"], s["lengths"], s["starts"], s["most_new"])
    heads, kvh, hd, page = s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    groups, B, L, S = heads // kvh, s["tables"].shape[0], s["longest"], s["most_new"]
    q, lengths, starts = s["q"], s["lengths"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    # every request's rows and keys, padded to the longest
    key = torch.arange(L, device="cuda")
    slot = (s["tables"].long().clamp(min=0) * page)[:, key // page] + key % page                    # [B, L]
    k, v = (x[slot].permute(0, 2, 1, 3) for x in _unpack(s["data"], s))                              # [B, kvh, L, hd]
    row = torch.arange(S, device="cuda")
    at = (starts[:-1, None] + row).clamp(max=q.shape[0] - 1)                                        # [B, S]
    qs = q.float().view(-1, kvh, groups, hd)[at].permute(0, 2, 3, 1, 4).reshape(B * kvh, groups * S, hd)
    hidden = key > (lengths - new)[:, None, None] + row[:, None]                                     # [B, S, L]
    scores = torch.bmm(qs, k.reshape(B * kvh, L, hd).transpose(1, 2).contiguous()) / math.sqrt(hd)
    scores = scores.view(B, kvh, groups, S, L).masked_fill_(hidden[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(B * kvh, groups * S, L), v.reshape(B * kvh, L, hd).contiguous()).view(B, kvh, groups, S, hd)
    out = out.permute(0, 3, 1, 2, 4).reshape(B * S, heads * hd)
    b = torch.searchsorted(starts[1:], torch.arange(q.shape[0], device="cuda"), right=True)
    return out[b * S + torch.arange(q.shape[0], device="cuda") - starts[b]].to(q.dtype)


def _run_logits(s):
    x, tokens = s["logits"], s["tokens"]
    if own:
        _, logits, _ = _framework()
        out, token = logits.process_logits(x, tokens=tokens, lengths=s["lengths"], prompt_lens=s["prompt_lens"],
                                           repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                                           bias=s["bias"], mask=s["mask"])
        return {"logits": out, "token": token}
    B, V = x.shape
    y = x.float()
    place = torch.arange(tokens.shape[1], device="cuda")
    live = place < s["lengths"][:, None]
    made = live & (place >= s["prompt_lens"][:, None])
    seen = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, tokens, live.to(torch.int32)) > 0
    times = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, tokens, made.to(torch.int32))
    rep = s["repetition"][:, None]
    y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
    y = y - s["frequency"][:, None] * times
    y = y - torch.where(times > 0, s["presence"][:, None], 0.0)
    start, ids, values = s["bias"]
    b = torch.searchsorted(start[1:].contiguous(), torch.arange(ids.shape[0], dtype=torch.int32, device="cuda"), right=True)
    y[b, ids.long()] += values
    if s["mask"] is not None:
        v = torch.arange(V, device="cuda")
        y = torch.where((s["mask"][:, v // 32] >> (v % 32)) & 1 > 0, y, float("-inf"))
    y = y.to(x.dtype)
    top = y.amax(-1, keepdim=True)
    first = torch.where(y == top, torch.arange(V, device="cuda"), V).amin(-1)
    return {"logits": y, "token": torch.where(top[:, 0] == float("-inf"), -1, first)}


_RUN = {"step": _run_step, "append": _run_append, "attention": _run_attention, "logits": _run_logits}


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "step":
        B, T = case["requests"], case["tokens"]
        # lengths and new tokens in; lengths, row offsets, flags, slots and positions out; a page number in and out
        return {"bytes": 4 * (5 * B + 2 * T + 2 * (T // case["page"])), "flops": 8 * T}
    if kind == "logits":
        B, V = case["requests"], case["vocab"]
        size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
        return {"bytes": B * (2 * size * V + (V // 8 if case["mask"] else 0) + 8 * case["history"] * 65 // 100 +
                              8 * case["biases"]), "flops": 6 * B * V}
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    token = kvh * (hd + 8 * (hd // case["group"]))          # a token's codes, scales and zeros, K and V
    if kind == "append":
        T = case["tokens"]
        rows = 2 * T * (2 * heads + 4 * kvh) * hd            # qkv in, q and the values read back out
        return {"bytes": rows + 8 * T * hd + 2 * T * token, "flops": T * hd * (6 * heads + 20 * kvh)}
    lengths, new = _lengths(case, 1)
    pairs = sum(n * length - n * (n - 1) // 2 for length, n in zip(lengths, new))
    return {"bytes": sum(lengths) * token + 4 * sum(new) * heads * hd, "flops": 4 * heads * hd * pairs}


# ---- the same in 64 bits, from the definitions ---------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind == "step":
        return _exact_step(case, seed)
    if kind == "append":
        return _exact_append(case, seed)
    if kind == "attention":
        return _exact_attention(case, seed)
    return _exact_logits(case, seed)


def _exact_step(case, seed):
    """Request by request, on the host."""
    lengths, new, tables, free = _step_inputs(case, seed)
    page, stack = case["page"], free.tolist()
    after, starts, slots, positions, failed = [], [0], [], [], []
    table = [[p for p in row if p >= 0] for row in tables.tolist()]
    for b, (n, m) in enumerate(zip(lengths, new)):
        for p in range(n, n + m):
            if p // page == len(table[b]):
                table[b].append(stack.pop())
            positions.append(p)
            slots.append(table[b][p // page] * page + p % page)
        after.append(n + m)
        starts.append(starts[-1] + m)
        failed.append(0)
    full = [row + [-1] * (tables.shape[1] - len(row)) for row in table]
    return {"state": _i32(after + [len(stack)]), "query_start": _i32(starts), "slots": _i32(slots),
            "positions": _i32(positions), "failed": _i32(failed), "tables": _i32(full)}


def _exact_append(case, seed):
    """q after RoPE and the values that v's codes stand for.  k's have no such
    value: after RoPE in 32 and in 64 bits a few of them lie on different sides
    of the middle between two codes."""
    heads, kvh, hd, group = case["heads"], case["kv_heads"], case["head_dim"], case["group"]
    qkv, _, positions, _ = _append_inputs(case, _generator(seed))
    cos, sin = (t[positions.long()].double()[:, None] for t in _rope_tables(case["max_pos"], hd))
    q = qkv[:, :heads * hd].double().view(-1, heads, hd)
    a, b = q[..., :hd // 2], q[..., hd // 2:]
    q = torch.cat((a * cos[..., :hd // 2] - b * sin[..., :hd // 2], b * cos[..., hd // 2:] + a * sin[..., hd // 2:]), -1)
    v = qkv[:, (heads + kvh) * hd:].double().view(-1, kvh, hd // group, group)
    low = v.min(-1, keepdim=True).values.half().double()
    step = ((v.max(-1, keepdim=True).values - low) / 15).clamp(min=0)
    power = torch.tensor([2.0 ** e for e in range(-24, 17)], dtype=torch.float64, device="cuda")
    unit = power[(torch.frexp(step).exponent - 7).clamp(-24, 16).long() + 24]       # the seventh bit's weight
    step = torch.ceil(step / unit) * unit
    code = torch.where(step > 0, torch.round((v - low) / step), torch.zeros_like(v)).clamp(0, 15)
    return {"q": q.reshape(-1, heads * hd), "k": None, "v": (code * step + low).reshape(-1, kvh, hd)}


def _exact_attention(case, seed):
    q, lengths, new, tables, _, parts = _attention_inputs(case, seed)
    kvh, hd, page, group = case["kv_heads"], case["head_dim"], case["page"], case["group"]
    each = case["heads"] // kvh
    out, at = [], 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        slots = torch.cat([torch.arange(page, device="cuda") + page * p for p in tables[b, :-(-n // page)].tolist()])[:n]
        k, v = ((c[slots].double() * s[slots].double().repeat_interleave(group, -1) +
                 z[slots].double().repeat_interleave(group, -1)) for c, s, z in parts)
        rows = q[at:at + m].double().view(m, case["heads"], hd)
        seen = torch.arange(n, device="cuda") <= torch.arange(n - m, n, device="cuda")[:, None]
        o = torch.empty_like(rows)
        for h in range(case["heads"]):
            scores = rows[:, h] @ k[:, h // each].t().contiguous() / math.sqrt(hd)
            o[:, h] = torch.softmax(torch.where(seen, scores, -math.inf), -1) @ v[:, h // each].contiguous()
        out.append(o.view(m, -1))
        at += m
    return torch.cat(out)


def _exact_logits(case, seed):
    """Row by row.  The token is the first largest logit as stored, and so has
    no value of its own in 64 bits."""
    s = _logits_inputs(case, seed)
    rows = []
    start, ids, values = s["bias"]
    for b in range(case["requests"]):
        x = s["logits"][b].double()
        n, prompt = int(s["lengths"][b]), int(s["prompt_lens"][b])
        text = s["tokens"][b, :n]
        known = text.unique()
        x[known] = torch.where(x[known] > 0, x[known] / s["repetition"][b].double(), x[known] * s["repetition"][b].double())
        made, times = text[prompt:].unique(return_counts=True)
        x[made] -= s["frequency"][b].double() * times + s["presence"][b].double()
        mine = slice(int(start[b]), int(start[b + 1]))
        x[ids[mine].long()] += values[mine].double()
        if s["mask"] is not None:
            bits = s["mask"][b].view(torch.uint8)[:, None] >> torch.arange(8, device="cuda", dtype=torch.uint8) & 1
            x[bits.reshape(-1)[:x.shape[0]] == 0] = -math.inf
        rows.append(x)
    return {"logits": torch.stack(rows), "token": None}
