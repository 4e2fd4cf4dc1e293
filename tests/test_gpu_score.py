"""The batch engine over a 16-bit cache, and scoring (``Qwen2BatchDecoder.score``): paged steps, append, attention and
log-probabilities together, on a small model."""
import math

import pytest
import torch
from test_gpu_batch import SHAPE, SMALL, _model, _prompts

from engine.qwen2_batch import Qwen2BatchDecoder
from kernels.kv16 import Kv16Cache
from kernels.paged import paged_release

pytestmark = pytest.mark.gpu


def _plain_logits(engine, text):
    """Logits in 64 bits of every position of one text, attention in torch over unrounded keys and values; the rest on
    the engine's own kernels."""
    m, s = engine.model, engine.s
    seen = []

    class Plain(Qwen2BatchDecoder):
        def _attention(self, li, qkv, step, max_query):
            T, nh, kvh, hd = qkv.shape[0], s.num_heads, s.num_kv_heads, s.head_dim
            x = qkv.double().view(T, nh + 2 * kvh, hd)
            cos, sin = m.cos[:T].double()[:, None], m.sin[:T].double()[:, None]
            rot = torch.cat((-x[..., hd // 2:], x[..., :hd // 2]), -1)
            q, k = torch.split((x * cos + rot * sin)[:, :nh + kvh], [nh, kvh], 1)
            k, v = (t.repeat_interleave(nh // kvh, 1) for t in (k, x[:, nh + kvh:]))
            hidden = torch.ones((T, T), dtype=torch.bool, device=qkv.device).triu(1)
            scores = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
            p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
            return torch.einsum("hij,jhd->ihd", p, v).reshape(T, nh * hd).half()

        def _rows(self, ids, step, max_query):
            h = super()._rows(ids, step, max_query)
            seen.append(h)
            return h

    plain = Plain(m, 1, page_size=16, cache_bits=16)
    plain.step(text, torch.tensor([text.shape[0]], dtype=torch.int32, device=text.device), text.shape[0])
    h = seen[0].double()
    h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + s.rms_norm_eps) * m.final_norm.double()
    return h @ m.lm_head.double().t().contiguous()


@pytest.mark.parametrize("shape,page,lens,chunk", [(SHAPE, 16, [1, 2, 33, 90, 17], 4096), (SMALL, 64, [130, 64, 7], 4096),
                                                   (SHAPE, 32, [100, 3, 57], 40), (SMALL, 16, [50, 1], 7)])
def test_scores_of_texts(gpu, shape, page, lens, chunk):
    """Against the model with plain attention.  Roundings to fp16 of the attention's operands and output (2^-11 each, four of
    them) pass through two layers and the final norm to logits of up to 12: 12 x 2 x 4 x 2^-11 bounds a logit's error, and a
    log-probability's is twice that."""
    rng = torch.Generator().manual_seed(3)
    model, _ = _model(shape, 2, gpu)
    texts = [p.to(gpu) for p in _prompts(rng, shape, lens)]
    engine = Qwen2BatchDecoder(model, len(lens) + 1, page_size=page, cache_bits=16)
    got = engine.score(texts, chunk)
    assert [g.shape[0] for g in got] == [n - 1 for n in lens] and not engine.tables.lengths.any()
    for text, scores in zip(texts, got):
        if text.shape[0] == 1:
            continue
        z = _plain_logits(engine, text)
        want = torch.log_softmax(z[:-1], -1).gather(1, text[1:, None])[:, 0].cpu()
        bound = 2 * z.abs().max().item() * 2 * 4 * 2.0**-11
        assert (scores.double() - want).abs().max() <= bound
    # the pages are returned: the same again, and in other chunks within the same bound
    again = engine.score(texts, chunk)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_sixteen_bits_against_four(gpu):
    """Greedy tokens of a model whose every answer is clear, over both caches and against their known successors."""
    model, successor = _model(SHAPE, 4, gpu)
    rng = torch.Generator().manual_seed(5)
    prompts = _prompts(rng, SHAPE, [3, 20, 64])
    want = []
    for p in prompts:
        t, out = int(p[-1]), []
        for _ in range(12):
            t = int(successor[t])
            out.append(t)
        want.append(out)
    for bits in (4, 16):
        engine = Qwen2BatchDecoder(model, 4, cache_bits=bits)
        assert engine.generate(prompts, 12).tolist() == want
    assert all(isinstance(c, Kv16Cache) for c in engine.caches)
    # a text of successors scores higher than one of other tokens
    text = torch.tensor([int(prompts[0][-1])] + want[0])
    likely, other = engine.score([text, text.flip(0)])
    assert likely.mean() > other.mean() + 1


def test_score_up_to_max_seq_len_and_refusals(gpu):
    model, _ = _model(SHAPE, 6, gpu)
    engine = Qwen2BatchDecoder(model, 2, page_size=16, cache_bits=16)
    rng = torch.Generator().manual_seed(7)
    full = _prompts(rng, SHAPE, [model.max_seq_len])[0]
    assert engine.score([full])[0].shape[0] == model.max_seq_len - 1
    for texts, chunk in (([], 8), ([full] * 3, 8), ([torch.cat((full, full[:1]))], 8), ([full], 0), ([full[None]], 8), ([full[:0]], 8),
                         ([torch.tensor([1, SHAPE.vocab_size])], 8), ([torch.tensor([1, -1])], 8)):
        with pytest.raises(ValueError):
            engine.score(texts, chunk)
    with pytest.raises(ValueError):
        Qwen2BatchDecoder(model, 2, cache_bits=8)
    with pytest.raises(ValueError):
        engine.generate([full[:5]], 0)
    small = Qwen2BatchDecoder(model, 2, num_pages=3, page_size=16, cache_bits=16)
    assert small.score([full[:33], full[:17]])[0].shape[0] == 32      # 2 pages and 1
    with pytest.raises(ValueError):
        small.score([full[:34], full[:17]])
    # requests that a caller of step began keep their pages
    new = torch.tensor([5, 0], dtype=torch.int32, device=gpu)
    engine.step(full[:5].to(gpu), new, 5)
    with pytest.raises(RuntimeError):
        engine.score([full[:9]])
    assert engine.tables.lengths.tolist() == [5, 0]
    paged_release(engine.tables, torch.zeros_like(new))
    assert engine.score([full[:9]])[0].shape[0] == 8
