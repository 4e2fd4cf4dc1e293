"""``kernels/logits.py`` against the same steps in torch on the CPU.  Each step is
one correctly rounded fp32 operation and the result is rounded once: logits and
tokens have to be equal."""
import math
import random

import pytest
import torch

from kernels.logits import process_logits

pytestmark = pytest.mark.gpu


def _reference(x, tokens=None, lengths=None, prompt=None, rep=None, pres=None, freq=None, bias=None, mask=None):
    y = x.float().clone()
    B, V = y.shape
    for b in range(B):
        if tokens is not None:
            text = tokens[b, :min(int(lengths[b]), tokens.shape[1])].tolist() if int(lengths[b]) > 0 else []
            made = text[int(prompt[b]):] if int(prompt[b]) > 0 else text
            for v in {t for t in text if 0 <= t < V}:
                n = made.count(v)
                e = y[b, v]
                if rep is not None:
                    e = e / rep[b] if e > 0 else e * rep[b]
                if freq is not None and n:
                    e = e - freq[b] * torch.tensor(float(n))
                if pres is not None and n:
                    e = e - pres[b]
                y[b, v] = e
        if bias is not None:
            start, ids, values = bias
            last = {int(ids[i]): i for i in range(max(0, int(start[b])), min(int(start[b + 1]), ids.shape[0]))}
            for v, i in last.items():
                if 0 <= v < V:
                    y[b, v] = y[b, v] + values[i]
        if mask is not None:
            for v in range(V):
                if not (int(mask[b, v // 32]) >> (v % 32)) & 1:
                    y[b, v] = -math.inf
    y = y.to(x.dtype)
    token = torch.argmax(y.float(), -1)          # the first largest on the CPU; a NaN counts as the largest
    token[(y.float() == -math.inf).all(-1)] = -1
    return y, token


def _check(gpu, x, **kw):
    names = {"prompt": "prompt_lens", "rep": "repetition", "pres": "presence", "freq": "frequency"}
    dev = {names.get(k, k): (tuple(t.to(gpu) for t in v) if isinstance(v, tuple) else v.to(gpu)) for k, v in kw.items()
           if v is not None}
    y, token = process_logits(x.to(gpu), **dev)
    ref, want = _reference(x, **kw)
    same = (y.cpu() == ref) | (torch.isnan(y.cpu()) & torch.isnan(ref))
    assert same.all(), f"{(~same).sum().item()} logits differ"
    assert token.tolist() == want.tolist()
    return y, token


def _inputs(B, V, L, dtype, seed, ids=torch.int64):
    g = torch.Generator().manual_seed(seed)
    rnd = random.Random(seed)
    lengths = torch.tensor([rnd.randint(0, L) for _ in range(B)], dtype=torch.int32)
    often = torch.randint(0, V, (8,), generator=g)
    tokens = torch.where(torch.rand((B, L), generator=g) < 0.5, often[torch.randint(0, 8, (B, L), generator=g)],
                         torch.randint(0, V, (B, L), generator=g)).to(ids)
    counts = [rnd.randint(0, 6) for _ in range(B)]
    start = torch.tensor([0] + [sum(counts[:i + 1]) for i in range(B)], dtype=torch.int32)
    n = sum(counts)
    return {"x": (torch.randn((B, V), generator=g) * 4).to(dtype), "tokens": tokens, "lengths": lengths,
            "prompt": (lengths * torch.rand(B, generator=g)).to(torch.int32),
            "rep": 1 + torch.rand(B, generator=g), "pres": torch.rand(B, generator=g), "freq": torch.rand(B, generator=g),
            "bias": (start, torch.randint(0, V, (n,), generator=g, dtype=torch.int32), torch.randn(n, generator=g) * 5),
            "mask": torch.randint(-2**31, 2**31 - 1, (B, (V + 31) // 32), generator=g, dtype=torch.int32)}


@pytest.mark.parametrize("B,V,L,dtype", [
    (1, 1, 3, torch.float16), (1, 33, 40, torch.float32), (3, 2048, 300, torch.float16), (2, 2049, 2300, torch.bfloat16),
    (5, 8192, 50, torch.bfloat16), (4, 9001, 64, torch.float16), (2, 10248, 5000, torch.float32),
    (300, 4104, 20, torch.float16), (520, 515, 9, torch.float16), (260, 8200, 12, torch.bfloat16)])
def test_everything_at_once(gpu, B, V, L, dtype):
    _check(gpu, **_inputs(B, V, L, dtype, B * 7 + V))


def test_each_rule_alone_and_none(gpu):
    full = _inputs(4, 3000, 200, torch.float16, 5)
    x = full["x"]
    history = {k: full[k] for k in ("tokens", "lengths", "prompt")}
    _check(gpu, x)
    _check(gpu, x, mask=full["mask"])
    _check(gpu, x, bias=full["bias"])
    _check(gpu, x, **history)
    for rule in ("rep", "pres", "freq"):
        _check(gpu, x, **history, **{rule: full[rule]})
    _check(gpu, x, **{**history, "tokens": history["tokens"].int()}, rep=full["rep"], freq=full["freq"])


def test_history_edges(gpu):
    """No history, one longer than its tensor, a prompt longer than the history, ids outside the vocabulary."""
    full = _inputs(6, 500, 70, torch.float32, 6)
    full["lengths"] = torch.tensor([0, 70, 500, 30, -4, 1], dtype=torch.int32)
    full["prompt"] = torch.tensor([0, 0, 80, 100, 0, -1], dtype=torch.int32)
    full["tokens"][:, ::3] = torch.tensor([-1, 500, 2**40, 499, -2**33, 0]).unsqueeze(1)
    _check(gpu, **full)
    empty = {"tokens": torch.zeros((6, 0), dtype=torch.int64), "lengths": full["lengths"], "prompt": full["prompt"]}
    _check(gpu, full["x"], **empty, rep=full["rep"])


def test_biases_listed_twice_and_outside(gpu):
    x = torch.zeros((2, 100))
    ids = torch.tensor([5, 5, -1, 100, 7, 5, 2**31 - 1, 9, 5], dtype=torch.int32)
    values = torch.arange(9, dtype=torch.float32) + 1
    _check(gpu, x, bias=(torch.tensor([0, 6, 9], dtype=torch.int32), ids, values))
    _check(gpu, x, bias=(torch.tensor([-5, 2, 50], dtype=torch.int32), ids, values))
    _check(gpu, x, bias=(torch.tensor([0, 0, 0], dtype=torch.int32), ids[:0], values[:0]))


def test_ties_infinities_nan_and_rows_with_nothing_left(gpu):
    V = 20000
    x = torch.full((9, V), -1.0)
    x[0, [17, 12345, 19999]] = 3.0                            # the first of equals
    x[1, 9000] = math.nan
    x[1, 15000] = math.inf
    x[2, :] = -math.inf
    x[3, 11] = math.inf
    x[4, :] = math.nan
    x[5, :] = 0.0
    x[5, ::2] = -0.0                                          # the zeros are equal
    x[6, :] = -math.inf
    x[6, 19999] = -3.4e38
    x[7, :] = -3.4e38
    mask = torch.full((9, V // 32), -1, dtype=torch.int32)
    mask[8] = 0                                               # a grammar that leaves nothing
    y, token = _check(gpu, x, mask=mask)
    assert token.tolist() == [17, 9000, -1, 11, 0, 0, 19999, 0, -1]
    for dtype in (torch.float16, torch.bfloat16):             # -3.4e38 becomes -inf in fp16
        _check(gpu, x.to(dtype), mask=mask)


def test_in_place_strides_and_offsets(gpu):
    full = _inputs(3, 4096, 100, torch.float16, 8)
    ref, want = _reference(**full)
    kw = {"tokens": full["tokens"].to(gpu), "lengths": full["lengths"].to(gpu), "prompt_lens": full["prompt"].to(gpu),
          "repetition": full["rep"].to(gpu), "presence": full["pres"].to(gpu), "frequency": full["freq"].to(gpu),
          "bias": tuple(t.to(gpu) for t in full["bias"]), "mask": full["mask"].to(gpu)}
    x = full["x"].to(gpu)
    wide = torch.empty((3, 5000), dtype=torch.float16, device=gpu)
    wide[:, 100:4196] = x
    odd = torch.empty(3 * 4096 + 1, dtype=torch.float16, device=gpu)[1:].view(3, 4096).copy_(x)
    for logits in (wide[:, 100:4196], odd, x.t().contiguous().t()):
        y, token = process_logits(logits, **kw)
        assert torch.equal(y.cpu(), ref) and token.tolist() == want.tolist()
    out = torch.empty(3 * 4096 + 1, dtype=torch.float16, device=gpu)[1:].view(3, 4096)
    y, token = process_logits(x, out=out, **kw)
    assert y is out and torch.equal(out.cpu(), ref)
    y, token = process_logits(x, out=x, **kw)
    assert y is x and torch.equal(x.cpu(), ref) and token.tolist() == want.tolist()


def test_in_a_graph(gpu):
    full = _inputs(2, 5000, 64, torch.float16, 9)
    x, tokens, lengths = full["x"].to(gpu), full["tokens"].to(gpu), full["lengths"].to(gpu)
    prompt, rep = torch.zeros_like(lengths), full["rep"].to(gpu)
    run = lambda: process_logits(x, tokens=tokens, lengths=lengths, prompt_lens=prompt, repetition=rep, frequency=rep)  # noqa: E731
    run()
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, token = run()
    torch.cuda.current_stream(gpu).wait_stream(side)
    for i in range(4):
        lengths.fill_(10 * i + 3)
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        a, b = run()
        assert torch.equal(y, a) and torch.equal(token, b), f"replay {i}"


def test_refusals(gpu):
    full = _inputs(2, 64, 10, torch.float16, 10)
    x = full["x"].to(gpu)
    tokens, lengths, rep = full["tokens"].to(gpu), full["lengths"].to(gpu), full["rep"].to(gpu)
    history = {"tokens": tokens, "lengths": lengths, "prompt_lens": lengths}
    for bad in (lambda: process_logits(x.double()), lambda: process_logits(x[0]), lambda: process_logits(full["x"]),
                lambda: process_logits(x, repetition=rep), lambda: process_logits(x, tokens=tokens),
                lambda: process_logits(x, **{**history, "tokens": tokens.short()}),
                lambda: process_logits(x, **{**history, "lengths": lengths.long()}),
                lambda: process_logits(x, **history, presence=rep.half()),
                lambda: process_logits(x, **history, presence=rep[:1]),
                lambda: process_logits(x, mask=torch.zeros((2, 3), dtype=torch.int32, device=gpu)),
                lambda: process_logits(x, mask=torch.zeros((2, 2), dtype=torch.int64, device=gpu)),
                lambda: process_logits(x, bias=(lengths, lengths, rep)),
                lambda: process_logits(x, out=torch.empty((2, 64), device=gpu))):
        with pytest.raises(ValueError):
            bad()
