"""The 16-bit cache's attention (``kernels/kv16.py``) where its plans are those of long prompts: many tiles an item, two groups
of waves that meet, no joining launch, more pages than a wave has lanes (``kv16_plans``), against 64 bits."""
import math

import kv16_cuts
import kv16_oracle as O
import pytest
import torch
from kv16_plans import PLANS
from test_gpu_kv16 import _batch, _call, _features, _gen, _i32

from kernels.kv16 import Kv16Cache, kv16_attention

pytestmark = pytest.mark.gpu


def _make(g, name, dtype, gain=1.0):
    nh, kvh, hd, page, requests, _ = PLANS[name]
    return _batch(g, requests, nh=nh, kvh=kvh, hd=hd, page=page, dtype=dtype, gain=gain)


@pytest.mark.parametrize("features", ["", "cap slopes window prefix first"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("name", PLANS)
def test_plan(gpu, name, dtype, features):
    g = _gen(gpu, 41)
    args = _make(g, name, dtype, 4.0 if features else 1.0)
    kw = _features(g, features.split(), PLANS[name][0], args[3], args[4])
    out = _call(*args, **kw)
    O.check(out, *O.attention(args[0], args[1].data, *args[2:], **kw))
    assert torch.equal(_call(*args, **kw), out)


@pytest.mark.parametrize("features", ["window", "prefix", "first", "slopes"])
@pytest.mark.parametrize("name", ["eight waves, odd", "whole", "eight waves behind a context"])
def test_plan_masks(gpu, name, features):
    g = _gen(gpu, 42)
    args = _make(g, name, "fp16")
    kw = _features(g, [features], PLANS[name][0], args[3], args[4])
    O.check(_call(*args, **kw), *O.attention(args[0], args[1].data, *args[2:], **kw))


@pytest.mark.parametrize("order", ["up", "down", "far up", "far down"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("name", ["eight waves", "eight waves, odd", "whole", "split", "eight waves, heads of 64"])
def test_scores_that_grow_along_the_tokens(gpu, name, dtype, order):
    """The running maximum is raised in tile after tile, or never again; far: past 2^8 powers of two, where exponents are
    differences first, from a late tile on or from the first to the last but no longer needed."""
    g = _gen(gpu, 43)
    q, cache, tables, lens, starts = args = _make(g, name, dtype, 24.0 if "far" in order else 4.0)
    page = cache.page_size
    for b, n in enumerate(lens):
        size = 0.05 + 2.0 * torch.arange(-(-n // page) * page, device=gpu) / n
        if "down" in order:
            size = size.flip(0)
        numbers = tables[b, :-(-n // page)].long()
        cache.k[numbers] = (cache.k[numbers].float() * size.view(-1, 1, page, 1)).to(cache.data.dtype)
    O.check(_call(*args), *O.attention(q, cache.data, *args[2:]))
    kw = {"slopes": torch.linspace(0.0, 0.02, PLANS[name][0], device=gpu)}
    O.check(_call(*args, **kw), *O.attention(q, cache.data, *args[2:], **kw))


def _seen(features, kw, n, rows, token, dev):
    """Which of one request's rows see the token."""
    p = torch.arange(n - rows, n, device=dev)
    sees = p >= token
    if features == "prefix":
        sees |= token < int(kw["prefix"][0])
    if features == "window":
        sees &= token > p - kw["window"]
    if features == "first":
        sees &= kw["first"] <= token
    return sees


@pytest.mark.parametrize("features", ["", "window", "first", "prefix"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("name", ["eight waves", "eight waves, odd", "whole", "eight waves, heads of 64"])
def test_what_a_row_does_not_see_may_hold_anything(gpu, name, dtype, features):
    """Values that are not finite and keys of NaN: exactly the rows that see one are not finite; pages outside the cache: NaN."""
    g = _gen(gpu, 44)
    q, cache, tables, lens, starts = args = _make(g, name, dtype)
    n, rows, page, hd = lens[0], starts[1], cache.page_size, cache.head_dim
    kw = _features(g, features.split(), PLANS[name][0], lens, starts)
    y, bound = O.attention(q, cache.data, *args[2:], **kw)
    for i, token in enumerate((0, 5, 64, 700, n // 2, n - 130, n - 2, n - 1)):
        sees = _seen(features, kw, n, rows, token, gpu)
        part, value = ((1, math.nan), (0, math.nan), (1, math.inf), (1, -math.inf))[i % 4]
        data = cache.data.clone()
        data[tables[0, token // page].long(), :, part, token % page, 7 * i] = value
        out = _call(q, Kv16Cache.of(data), tables, lens, starts, **kw)
        finite = torch.isfinite(out.view(rows, -1, hd)).all(2)
        assert not finite[sees].any() and sees.any(), (token, part, value)
        O.check(out[~sees], y[~sees], bound[~sees], f"part {part} token {token}")
    last = (n - 1) // page
    for i, at in enumerate((0, last // 3, last // 2, last - 1, last)):
        bad = tables.clone()
        bad[0, at] = (-1, cache.num_pages, 2**31 - 1)[i % 3]
        out = _call(q, cache, bad, lens, starts, **kw)
        sees = torch.stack([_seen(features, kw, n, rows, t, gpu) for t in range(at * page, min(n, (at + 1) * page))]).any(0)
        assert torch.isnan(out[sees]).all() and sees.any(), at
        O.check(out[~sees], y[~sees], bound[~sees], f"page {at}")


@pytest.mark.parametrize("name", ["eight waves", "whole", "eight waves, heads of 64", "whole, kv heads"])
def test_rows_that_see_nothing_and_rows_of_no_request(gpu, cuts, name):
    """One request with rows before its first token, rows behind a document's begin, rows of no request in front and behind, and
    rows past a max_query that is too small: zeros, and NaN for the last."""
    nh, kvh, hd, page, requests, want = PLANS[name]
    g = _gen(gpu, 45)
    q, cache, tables, lens, starts = _make(g, name, "fp16")
    rows = starts[1]
    n, most, total = rows - 2, rows - 3, rows + 8
    c = cuts([(n, rows)], nh // kvh, kvh, page=page, total=total, max_query=most).check()
    assert (c.parts, c.combine) == (want["parts"], 0)
    q = torch.cat((q[:5], q, q[:3]))
    first = torch.zeros(total, dtype=torch.int32, device=gpu)
    blind = [0, 1, 2, 3, 4, 5, 6, 5 + rows // 2, 6 + rows // 2, *range(5 + rows, total)]
    first[5 + rows // 2:7 + rows // 2] = 10**6
    out = kv16_attention(q, cache, tables, _i32([n], gpu), _i32([5, 5 + rows], gpu), most, first=first)
    y, bound = O.attention(q, cache.data, tables, [n], [5, 5 + rows], first=first)
    assert (out[blind] == 0).all() and torch.isnan(out[5 + most:5 + rows]).all()
    O.check(out[:5 + most], y[:5 + most], bound[:5 + most])
    # with every row blind, and without tokens
    none = kv16_attention(q, cache, tables, _i32([n], gpu), _i32([5, 5 + rows], gpu), rows, first=torch.full_like(first, 2**31 - 1))
    assert (none == 0).all()
    none = kv16_attention(q, cache, tables, _i32([0], gpu), _i32([5, 5 + rows], gpu), rows)
    assert (none == 0).all()


@pytest.fixture(scope="module")
def cuts(tmp_path_factory):
    return kv16_cuts.build(tmp_path_factory.mktemp("cuts16"))


@pytest.mark.parametrize("name", ["eight waves", "whole", "split"])
def test_in_a_graph(gpu, name):
    """Captured once, replayed with other lengths and starts; two of them at once on two streams."""
    g = _gen(gpu, 46)
    q, cache, tables, lens, starts = _make(g, name, "bf16")
    n, s = _i32(lens, gpu), _i32(starts, gpu)
    call = lambda: kv16_attention(q, cache, tables, n, s, starts[1], softcap=30.0)  # noqa: E731
    call()
    graphs, outs, sides = [], [], [torch.cuda.Stream() for _ in range(2)]
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(call())
        torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        now, used = [lens[0] - 500 * k], [13 * k, starts[1] - 201 * k]
        n.copy_(_i32(now, gpu))
        s.copy_(_i32(used, gpu))
        want = call()
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs), k
        O.check(want, *O.attention(q, cache.data, tables, now, used, softcap=30.0), f"replay {k}")
