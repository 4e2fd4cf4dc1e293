"""The batch engine where a request cannot be served, and calls that meet what earlier
ones left."""
import pytest
import torch
from test_gpu_batch import SHAPE, _model, _prompts

from engine.qwen2_batch import Qwen2BatchDecoder
from engine.qwen2_decode import Qwen2AwqDecoder
from kernels.paged import paged_release

pytestmark = pytest.mark.gpu


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _step(engine, prompts, dev):
    """Logits of a step that adds prompts[b] to request b (None: nothing)."""
    new = [0 if p is None else len(p) for p in prompts]
    ids = torch.cat([p for p in prompts if p is not None]).to(dev)
    return engine.step(ids, _i32(new, dev), max(new))


def _near(a, b):
    """The same rows through the same kernels, in a batch of other rows: roundings of fp16 activations."""
    return ((a.float() - b.float()).norm() / b.float().norm()).item() <= 4 * 2.0**-11


def test_refused_requests_are_told_and_have_no_logits(gpu):
    """Too few pages, for a prompt that is new and for a request that runs."""
    rng = torch.Generator().manual_seed(11)
    model, _ = _model(SHAPE, 12, gpu)
    engine, ample = (Qwen2BatchDecoder(model, 3, num_pages=n, page_size=16) for n in (4, 20))
    a, b, c = _prompts(rng, SHAPE, [20, 10, 40])
    got, want = (_step(e, [a, b, c], gpu) for e in (engine, ample))
    assert engine.failed.tolist() == [0, 0, 1] and ample.failed.tolist() == [0, 0, 0]
    assert torch.isnan(got[2]).all() and engine.tables.lengths.tolist() == [20, 10, 0]
    assert _near(got[:2], want[:2])
    paged_release(ample.tables, _i32([20, 10, 0], gpu))
    a, b = _prompts(rng, SHAPE, [13, 7])                     # one page is left, and either needs one
    got, want = _step(engine, [a, b, None], gpu), _step(ample, [a, None, None], gpu)
    assert engine.failed.tolist() == [0, 1, 0] and engine.tables.lengths.tolist() == [33, 10, 0]
    assert torch.isnan(got[1]).all() and _near(got[0], want[0])
    for e in (engine, ample):                                # the first request ends: now the second has its page
        paged_release(e.tables, _i32([0, 10, 0], gpu))
    got, want = (_step(e, [None, b, None], gpu) for e in (engine, ample))
    assert engine.failed.tolist() == [0, 0, 0] and _near(got[1], want[1])


@pytest.mark.parametrize("limit,lens", [(100, [99, 90]), (130, [127, 128])])
def test_no_token_past_the_models_positions(gpu, limit, lens):
    """The last page reaches past max_seq_len; a request that would too is refused like one without pages."""
    rng = torch.Generator().manual_seed(limit)
    engine = Qwen2BatchDecoder(Qwen2AwqDecoder(SHAPE, limit, seed=3, device=gpu), 3, page_size=64)
    pages = lambda n: -(-n // 64)  # noqa: E731
    assert torch.isfinite(_step(engine, [*_prompts(rng, SHAPE, lens), None], gpu)[:2]).all()
    for add in ([1, 1], [limit - lens[0], 3], [0, 1], [2**30, 0], [1, limit - lens[1] - 1], [0, 1]):
        ids = torch.zeros(min(sum(add), 9), dtype=torch.int64, device=gpu)
        add.append(0)                                       # (behind rows that pass the batch, a request is refused too)
        fits = [(*lens, 0)[b] + add[b] <= limit and sum(add[:b + 1]) <= 9 for b in range(3)]
        logits = engine.step(ids, _i32(add, gpu), 9)
        lens = [n + m if ok else n for n, m, ok in zip(lens, add, fits)]
        assert engine.failed.tolist() == [0 if ok else 1 for ok in fits]
        assert engine.tables.lengths.tolist() == [*lens, 0]
        assert engine.tables.free_count.item() == engine.tables.free_pages.shape[0] - sum(map(pages, lens))
        for b in range(2):
            assert torch.isnan(logits[b]).all() if not fits[b] else add[b] == 0 or torch.isfinite(logits[b]).all()
    for bad in (_i32([1, 1], gpu), _i32([1, 1, 0], "cpu"), _i32([1, 1, 0], gpu).long()):
        with pytest.raises(ValueError):
            engine.step(ids, bad, 9)


def test_generate_leaves_running_requests_alone(gpu):
    """It refuses while a caller of step has requests, and takes back its own pages when it fails."""
    rng = torch.Generator().manual_seed(21)
    model, successor = _model(SHAPE, 22, gpu)
    engine = Qwen2BatchDecoder(model, 3, page_size=16)
    a, b = _prompts(rng, SHAPE, [20, 5])
    want = engine.generate([a, b], 4)
    _step(engine, [None, a, None], gpu)
    state = engine.tables.state.clone()
    with pytest.raises(RuntimeError, match="running"):
        engine.generate([a, b], 4)
    assert torch.equal(engine.tables.state, state)
    assert int(_step(engine, [None, successor[a[-1:]], None], gpu)[1].argmax()) == int(want[0, 1])
    paged_release(engine.tables, _i32([0, 0, 0], gpu))
    with pytest.raises(ValueError):                          # a mask of another vocabulary: found in the middle
        engine.generate([a, b], 4, mask=torch.zeros((2, 3), dtype=torch.int32, device=gpu))
    assert engine.tables.free_count.item() == engine.tables.free_pages.shape[0]
    assert torch.equal(engine.generate([a, b], 4), want)


def test_generate_takes_whole_penalties(gpu):
    """Penalties given as integers are the same numbers."""
    rng = torch.Generator().manual_seed(31)
    model, _ = _model(SHAPE, 32, gpu)
    engine = Qwen2BatchDecoder(model, 2, page_size=16)
    prompts = _prompts(rng, SHAPE, [9, 4])
    rules = {"repetition": 2, "presence": 3, "frequency": 1}
    assert torch.equal(engine.generate(prompts, 5, **rules), engine.generate(prompts, 5, **{k: float(v) for k, v in rules.items()}))


def test_generate_asks_for_no_page_that_it_does_not_use(gpu):
    """The last token is returned and never stored: 14 + 3 tokens are one page of 16."""
    rng = torch.Generator().manual_seed(41)
    model, _ = _model(SHAPE, 42, gpu)
    prompts = _prompts(rng, SHAPE, [14, 30])
    want = Qwen2BatchDecoder(model, 2, page_size=16).generate(prompts, 3)
    assert torch.equal(Qwen2BatchDecoder(model, 2, num_pages=3, page_size=16).generate(prompts, 3), want)
    with pytest.raises(ValueError, match="need 5 pages, the cache has 3"):
        Qwen2BatchDecoder(model, 2, num_pages=3, page_size=16).generate(prompts, 4)


def test_generate_refuses_ids_outside_the_vocabulary(gpu):
    """The embedding would look them up outside its table."""
    model, _ = _model(SHAPE, 52, gpu)
    engine = Qwen2BatchDecoder(model, 2, page_size=16)
    one = torch.zeros(3, dtype=torch.int64)
    for id_ in (-1, SHAPE.vocab_size, 2**40):
        for dev in ("cpu", gpu):
            bad = torch.tensor([5, id_], device=dev)
            with pytest.raises(ValueError, match="vocabulary"):
                engine.generate([one, bad], 2)
    assert engine.generate([one, torch.tensor([SHAPE.vocab_size - 1])], 2).shape == (2, 2)


def test_generate_refuses_biases_for_other_requests(gpu):
    model, _ = _model(SHAPE, 62, gpu)
    engine = Qwen2BatchDecoder(model, 2, page_size=16)
    one = torch.zeros(3, dtype=torch.int64)
    for biases in ([], [{5: 1.0}], [{}, {}, {5: 1.0}]):
        with pytest.raises(ValueError, match="biases"):
            engine.generate([one, one], 2, biases=biases)
    assert engine.generate([one, one], 2, biases=[{}, {}]).shape == (2, 2)
