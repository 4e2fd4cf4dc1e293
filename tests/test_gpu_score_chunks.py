"""Scores of texts (``Qwen2BatchDecoder.score``) in passes of few and of many rows, over both caches."""
import pytest
import torch
from test_gpu_batch import SHAPE, SMALL, _model, _prompts
from test_gpu_score import _plain_logits

from engine.qwen2_batch import Qwen2BatchDecoder
from kernels.paged import paged_release

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,page,lens", [(SHAPE, 16, [1, 33, 90, 17]), (SMALL, 64, [130, 64, 2])])
def test_the_same_texts_in_other_chunks(gpu, shape, page, lens):
    """Each against the model with plain attention, within the bound that ``test_scores_of_texts`` derives."""
    model, _ = _model(shape, 2, gpu)
    texts = [p.to(gpu) for p in _prompts(torch.Generator().manual_seed(8), shape, lens)]
    engine = Qwen2BatchDecoder(model, len(lens), page_size=page, cache_bits=16)
    want, bound = [], []
    for text in texts:
        z = _plain_logits(engine, text)
        want.append(torch.log_softmax(z[:-1], -1).gather(1, text[1:, None])[:, 0].cpu())
        bound.append(2 * z.abs().max().item() * 2 * 4 * 2.0**-11)
    for chunk in (1, 7, 40, 65, 4096):
        got = engine.score(texts, chunk)
        assert [g.shape[0] for g in got] == [n - 1 for n in lens] and not engine.tables.lengths.any()
        for g, w, b in zip(got, want, bound):
            assert not g.numel() or (g.double() - w).abs().max() <= b, chunk


@pytest.mark.parametrize("bits", [4, 16])
def test_scores_are_those_of_step(gpu, bits):
    """Token by token both run the same passes: the logits that ``step`` gives, rounded to fp16 (2^-12 of the largest below 2 z),
    give the same log-probabilities, off by twice a logit's rounding."""
    model, _ = _model(SHAPE, 2, gpu)
    engine = Qwen2BatchDecoder(model, 2, page_size=16, cache_bits=bits)
    text = _prompts(torch.Generator().manual_seed(9), SHAPE, [50])[0].to(gpu)
    got = engine.score([text], 1)[0]
    new = torch.tensor([1, 0], dtype=torch.int32, device=gpu)
    logits = torch.cat([engine.step(text[i:i + 1], new, 1, 1) for i in range(49)]).double()
    paged_release(engine.tables, torch.zeros_like(new))
    want = torch.log_softmax(logits, -1).gather(1, text[1:, None])[:, 0].cpu()
    assert (got.double() - want).abs().max() <= 2 * logits.abs().max().item() * 2.0**-11
    # and in one pass, over a cache that rounds its keys and values alike whatever the pass
    whole = engine.score([text])[0]
    assert torch.isfinite(whole).all() and whole.shape == got.shape
