"""Scores of texts (``Qwen2BatchDecoder.score``) in passes of few and of many rows, over a 16-bit cache."""
import pytest
import torch
from test_gpu_batch import SHAPE, SMALL, _model, _prompts
from test_gpu_score import _plain_logits

from engine.qwen2_batch import Qwen2BatchDecoder

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
