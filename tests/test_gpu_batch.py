"""The batch engine (``engine/qwen2_batch.py``): paged 4-bit cache, attention and
logits rules together, on a small model."""
import math

import pytest
import torch

from engine.qwen2_batch import Qwen2BatchDecoder
from engine.qwen2_decode import Qwen2AwqDecoder, Qwen2Shape
from kernels.kv4 import kv4_append, kv4_gather

pytestmark = pytest.mark.gpu

SHAPE = Qwen2Shape(vocab_size=1003, hidden_size=512, intermediate_size=1024, num_layers=2, num_heads=4, num_kv_heads=2)
SMALL = Qwen2Shape(vocab_size=640, hidden_size=384, intermediate_size=512, num_layers=2, num_heads=6, num_kv_heads=2)


def _model(shape, seed, dev):
    """Random weights small enough for the embedding to show through to the last
    layer, and an output projection that answers each token with one clear successor."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    H, I, V = shape.hidden_size, shape.intermediate_size, shape.vocab_size
    embed = torch.randn((V, H), generator=g, device=dev).half()
    successor = torch.randperm(V, generator=g, device=dev)
    head = torch.empty_like(embed)
    head[successor] = embed * 0.02

    def awq(k, n):
        word = dict(generator=g, device=dev, dtype=torch.int32)
        return (torch.randint(-2**31, 2**31 - 1, (k, n // 8), **word),
                torch.randint(-2**31, 2**31 - 1, (k // 128, n // 8), **word),
                (torch.rand((k // 128, n), generator=g, device=dev) * 0.0025 + 0.0005).half())

    qkv = (shape.num_heads + 2 * shape.num_kv_heads) * shape.head_dim
    layers = [{"ln1": torch.ones(H, dtype=torch.float16, device=dev), "ln2": torch.ones(H, dtype=torch.float16, device=dev),
               "qkv_bias": (torch.randn(qkv, generator=g, device=dev) * 0.5).half(), "qkv": awq(H, qkv), "o": awq(H, H),
               "gate_up": awq(H, 2 * I), "down": awq(I, H)} for _ in range(shape.num_layers)]
    weights = {"embed": embed, "lm_head": head, "final_norm": torch.ones(H, dtype=torch.float16, device=dev), "layers": layers}
    return Qwen2AwqDecoder(shape, max_seq_len=256, device=dev, weights=weights), successor.cpu()


class PlainAttention(Qwen2BatchDecoder):
    """The same engine with its attention in torch, in 32 bits, over the values that the cache holds."""

    def _attention(self, li, qkv, step, max_query):
        m, s, cache = self.model, self.s, self.caches[li]
        q = kv4_append(qkv, cache, step.slots, step.positions, m.cos, m.sin, s.num_heads).float()
        page = cache.page_size
        out = torch.zeros_like(q).view(-1, s.num_heads, s.head_dim)
        starts, lengths = step.query_start.tolist(), step.lengths.tolist()
        for b, n in enumerate(lengths):
            lo, hi = starts[b], starts[b + 1]
            if lo == hi:
                continue
            table = self.tables.block_tables[b].tolist()
            slots = torch.tensor([table[i // page] * page + i % page for i in range(n)], dtype=torch.int32, device=self.dev)
            k, v = (x.float() for x in kv4_gather(cache, slots))
            k, v = (x.repeat_interleave(s.num_heads // s.num_kv_heads, 1) for x in (k, v))
            rows = q[lo:hi].view(hi - lo, s.num_heads, s.head_dim)
            hidden = torch.arange(n, device=self.dev) > torch.arange(n - (hi - lo), n, device=self.dev)[:, None]
            scores = torch.einsum("rhd,khd->hrk", rows, k) / math.sqrt(s.head_dim)
            out[lo:hi] = torch.einsum("hrk,khd->rhd", torch.softmax(scores.masked_fill(hidden, -math.inf), -1), v)
        return out.view(q.shape).half()


def _prompts(rng, shape, lens):
    return [torch.randint(0, shape.vocab_size, (n,), generator=rng) for n in lens]


@pytest.mark.parametrize("shape,page,group,lens", [(SHAPE, 16, 32, [1, 16, 33, 90, 5]), (SMALL, 64, 64, [64, 7, 130])])
def test_logits_of_prompts_and_steps(gpu, shape, page, group, lens):
    """Against the same engine with plain attention: fp16 activations through two
    layers.  A rounding of the attention's output (2^-11) reaches the logits through two layers and
    the final norm: 4 x 2^-11 of their size bounds it."""
    rng = torch.Generator().manual_seed(1)
    model, _ = _model(shape, 2, gpu)
    prompts = [p.to(gpu) for p in _prompts(rng, shape, lens)]
    engines = [cls(model, len(lens) + 1, page_size=page, group_size=group) for cls in (Qwen2BatchDecoder, PlainAttention)]
    ids, new = torch.cat(prompts), torch.tensor(lens + [0], dtype=torch.int32, device=gpu)
    for step in range(4):
        a, b = (e.step(ids, new, int(new.max())).float() for e in engines)
        assert torch.isfinite(a).all()
        rel = ((a - b).norm() / b.norm()).item()
        assert rel <= 4 * 2.0**-11, f"step {step}: {rel}"
        ids = torch.randint(0, shape.vocab_size, (len(lens),), generator=rng).to(gpu)
        new = torch.tensor([1] * len(lens) + [0], dtype=torch.int32, device=gpu)
        assert torch.equal(engines[0].tables.state, engines[1].tables.state)


def test_generate_follows_the_successors(gpu):
    rng = torch.Generator().manual_seed(3)
    model, successor = _model(SHAPE, 4, gpu)
    engine = Qwen2BatchDecoder(model, 12, page_size=16)
    for lens in ([1, 40, 17], [3] * 12):
        prompts = _prompts(rng, SHAPE, lens)
        tokens = engine.generate(prompts, 20)
        for p, row in zip(prompts, tokens):
            want, last = [], p[-1]
            for _ in range(20):
                last = successor[last]
                want.append(int(last))
            assert row.tolist() == want
        assert engine.tables.free_count.item() == engine.tables.free_pages.shape[0], "all pages are back"


def test_generate_under_rules(gpu):
    """A bias that decides, a mask that forbids the successor, a penalty that breaks a loop."""
    rng = torch.Generator().manual_seed(5)
    model, successor = _model(SHAPE, 6, gpu)
    engine = Qwen2BatchDecoder(model, 4, page_size=16)
    prompts = _prompts(rng, SHAPE, [9, 30])
    tokens = engine.generate(prompts, 5, biases=[{77: 1000.0}, {}])
    assert tokens[0].tolist() == [77] * 5 and int(tokens[1][0]) == int(successor[prompts[1][-1]])
    allowed = torch.zeros((2, (SHAPE.vocab_size + 31) // 32), dtype=torch.int64)
    allowed[0, 2] = 1 << 3                                                # token 67 only
    allowed[1, :] = 2**32 - 1
    allowed = torch.where(allowed >= 2**31, allowed - 2**32, allowed).int().to(gpu)
    tokens = engine.generate(prompts, 3, mask=allowed)
    assert tokens[0].tolist() == [67] * 3 and int(tokens[1][0]) == int(successor[prompts[1][-1]])
    # the biased token again, unless its presence costs more than the bias gives
    tokens = engine.generate(prompts, 3, presence=2000.0, biases=[{77: 1000.0}, {77: 1000.0}])
    assert (tokens[:, 0] == 77).all() and (tokens[:, 1:] != 77).all()
    with pytest.raises(RuntimeError):
        engine.generate(prompts, 2, mask=torch.zeros_like(allowed))


def test_refusals(gpu):
    model, _ = _model(SHAPE, 7, gpu)
    engine = Qwen2BatchDecoder(model, 2, num_pages=4, page_size=16)
    one = torch.zeros(1, dtype=torch.int64)
    for bad in (lambda: engine.generate([], 3), lambda: engine.generate([one] * 3, 3), lambda: engine.generate([one[:0]], 3),
                lambda: engine.generate([one], 0), lambda: engine.generate([one], 256),
                lambda: engine.generate([one.repeat(30), one.repeat(30)], 10)):
        with pytest.raises(ValueError):
            bad()
