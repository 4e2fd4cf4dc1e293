"""The 16-bit paged cache and its attention (``kernels/kv16.py``) against the definition in 64
bits (``kv16_oracle``, which derives the bound that every element is held to)."""
import math

import kv16_oracle as O
import pytest
import torch

from kernels import _native
from kernels.kv16 import Kv16Cache, kv16_append, kv16_attention
from kernels.paged import PagedTables, paged_step

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _batch(g, requests, *, nh=4, kvh=2, hd=64, page=16, dtype="fp16", spare=2, width=None, gain=1.0):
    """(q, cache, tables, lens, starts, keyword arguments of the calls) of [(length, rows)], pages in random order."""
    dev = g.device
    lens = [n for n, _ in requests]
    starts = [sum(m for _, m in requests[:b]) for b in range(len(requests) + 1)]
    held = [-(-n // page) for n in lens]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    tables = torch.full((len(requests), width or max(held) + 1), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, h in enumerate(held):
        tables[b, :h] = order[at:at + h]
        at += h
    data = torch.randn((pages, kvh, 2, page, hd), generator=g, device=dev)
    data[:, :, 0] *= 1.0 + 3.0 * torch.rand((kvh, 1, hd), generator=g, device=dev).pow(8)
    q = (torch.randn((starts[-1], nh * hd), generator=g, device=dev) * gain).to(DT[dtype])
    return q, Kv16Cache.of(data.to(DT[dtype])), tables, lens, starts


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _call(q, cache, tables, lens, starts, **kw):
    most = max([1] + [b - a for a, b in zip(starts, starts[1:])])
    return kv16_attention(q, cache, tables, _i32(lens, q.device), _i32(starts, q.device), most, **kw)


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _features(g, names, nh, lens, starts):
    """Keyword arguments of some of the masks and score rules."""
    dev, kw = g.device, {}
    if "cap" in names:
        kw["softcap"] = 20.0
    if "slopes" in names:
        kw["slopes"] = torch.exp2(-8.0 * torch.arange(1, nh + 1, device=dev) / nh)
    if "window" in names:
        kw["window"] = max(1, max(lens) // 3)
    if "prefix" in names:
        kw["prefix"] = _i32([(n * (b + 2)) // (b + 3) for b, n in enumerate(lens)], dev)
    if "first" in names:
        # a new document every 37 tokens
        pos = torch.cat([torch.arange(n - (b - a), n, device=dev) for n, a, b in zip(lens, starts, starts[1:])])
        kw["first"] = (pos.clamp(min=0) // 37 * 37).to(torch.int32)
    return kw


DECODE = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (31, 1), (33, 1), (129, 1), (700, 1)]
SHAPES = [
    (4, 2, 64, 16, "fp16", DECODE), (28, 4, 128, 64, "fp16", DECODE), (8, 8, 128, 32, "bf16", DECODE),
    (16, 1, 64, 128, "bf16", [(300, 1), (64, 1)]), (64, 1, 128, 256, "fp16", [(513, 1), (5, 1)]),
    # chunks: few rows, a block of columns and a little more, many
    (7, 1, 128, 16, "fp16", [(40, 18), (200, 19), (19, 19)]), (4, 4, 64, 32, "bf16", [(129, 129), (77, 5), (500, 131)]),
    (28, 4, 128, 64, "fp16", [(301, 301)]), (6, 2, 128, 16, "bf16", [(1, 1), (90, 64), (333, 333), (2, 2)]),
    (5, 5, 64, 256, "fp16", [(1000, 250)]), (1, 1, 128, 64, "fp16", [(2000, 1000)]),
]


@pytest.mark.parametrize("features", ["", "cap", "slopes", "window", "prefix", "first", "cap slopes window prefix first"])
@pytest.mark.parametrize("nh,kvh,hd,page,dtype,requests", SHAPES)
def test_attention(gpu, nh, kvh, hd, page, dtype, requests, features):
    g = _gen(gpu, 1)
    args = _batch(g, requests, nh=nh, kvh=kvh, hd=hd, page=page, dtype=dtype, gain=4.0 if "cap" in features else 1.0)
    kw = _features(g, features.split(), nh, args[3], args[4])
    O.check(_call(*args, **kw), *O.attention(args[0], args[1].data, *args[2:], **kw))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("features", ["", "cap slopes window prefix first"])
def test_a_chunk_beside_single_tokens(gpu, features, dtype):
    """One request is the tile kernel's, the others the decode kernel's; then chunks of which one is a single token's."""
    test_attention(gpu, 28, 4, 128, 64, dtype, [*DECODE[:5], (700, 300), *DECODE[5:]], features)
    test_attention(gpu, 14, 2, 64, 32, dtype, [(900, 120), (1500, 1), (333, 150)], features)


@pytest.mark.parametrize("features", ["", "cap slopes window prefix first"])
def test_many_requests(gpu, features):
    """More than a wave has lanes: single tokens, a few rows each with some that have none, and chunks alone."""
    test_attention(gpu, 4, 2, 64, 16, "fp16", [(1 + 37 * i % 300, 1) for i in range(150)], features)
    test_attention(gpu, 8, 2, 64, 32, "bf16", [(5 + 53 * i % 211, i % 4) for i in range(130)] + [(200, 90)], features)
    test_attention(gpu, 4, 1, 128, 64, "fp16", [(41 + 17 * i % 400, 40) for i in range(70)], features)


def test_split_along_the_tokens(gpu):
    """Few rows of long contexts are cut into items: decode and tiles, with a window that leaves out most of the context."""
    g = _gen(gpu, 2)
    for requests, window in (([(5000, 1), (9000, 1)], None), ([(9000, 1)], 700), ([(6000, 70)], None), ([(6000, 70)], 333)):
        args = _batch(g, requests, nh=14, kvh=2, hd=64, page=32)
        O.check(_call(*args, window=window), *O.attention(args[0], args[1].data, *args[2:], window=window), f"{requests} {window}")


@pytest.mark.parametrize("rows", [3, 300])
def test_rows_that_see_nothing(gpu, rows):
    """Positions before the first token, documents that begin past the row, requests without tokens, rows of no
    request: zeros.  (rows: the decode kernel's and the tile kernel's.)"""
    g = _gen(gpu, 3)
    q, cache, tables, lens, starts = _batch(g, [(rows + 50, rows), (2, 2), (rows, rows)], nh=2, kvh=1)
    lens = [rows + 50, 0, rows - 2]                     # two rows of the last stand before its first token
    q = torch.cat((q[:5], q))                           # five rows of no request at the front, and some at the end
    starts = [s + 5 for s in starts]
    q = torch.cat((q, q[:3]))
    first = torch.zeros(q.shape[0], dtype=torch.int32, device=gpu)
    first[5 + rows // 2:5 + rows // 2 + 2] = 10**6
    out = kv16_attention(q, cache, tables, _i32(lens, gpu), _i32(starts, gpu), rows, first=first)
    y, bound = O.attention(q, cache.data, tables, lens, starts, first=first)
    O.check(out, y, bound)
    empty = [*range(5), 5 + rows // 2, 6 + rows // 2, 5 + rows, 6 + rows, 7 + rows, 8 + rows, *range(7 + 2 * rows, 10 + 2 * rows)]
    assert (out[empty] == 0).all()
    # and with every row of a request blind
    out = kv16_attention(q, cache, tables, _i32(lens, gpu), _i32(starts, gpu), rows, first=torch.full_like(first, 2**31 - 1))
    assert (out == 0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,features", [(1, "window"), (5, ""), (5, "window"), (5, "first"), (200, ""), (200, "window"),
                                           (200, "first"), (200, "prefix")])
def test_what_a_row_does_not_see_may_hold_anything(gpu, rows, features, dtype, value):
    """Keys or values that are not finite at places that some rows see and others do not: exactly the rows that see one
    are not finite, the others as if it were not there."""
    g = _gen(gpu, 4)
    n, page = 260, 16
    args = _batch(g, [(n, rows), (n, rows)], nh=3, kvh=1, hd=128, page=page, dtype=dtype)
    q, cache, tables, lens, starts = args
    kw = _features(g, features.split(), 3, lens, starts)
    y, bound = O.attention(q, cache.data, tables, lens, starts, **kw)
    # the pages' ends past the length, and pages of nobody
    spare = sorted(set(range(cache.num_pages)) - set(tables[tables >= 0].tolist()))
    cache.data[spare] = value
    for b in range(2):
        cache.data[tables[b, n // page].long(), :, :, n % page:] = value
    O.check(_call(*args, **kw), y, bound, "past the length")
    for part in (0, 1):
        for token in (0, 5, n - rows, n - rows // 2 - 1, n - 2, n - 1):
            data = cache.data.clone()
            data[tables[0, token // page].long(), 0, part, token % page, 7] = value
            out = _call(q, Kv16Cache.of(data), tables, lens, starts, **kw)
            for i in range(rows):
                p = n - rows + i
                sees = token <= p or (features == "prefix" and token < int(kw["prefix"][0]))
                sees = sees and (features != "window" or token > p - kw["window"])
                sees = sees and (features != "first" or token >= int(kw["first"][i]))
                row = out[i].view(3, 128)
                if not sees:
                    O.check(out[i:i + 1], y[i:i + 1], bound[i:i + 1], f"part {part} token {token} row {i}")
                elif part == 1 or math.isnan(value):    # (an infinite key: a score of +-infinity by the sign of q)
                    assert not torch.isfinite(row).all(1).any(), (part, token, i)
            O.check(out[rows:], y[rows:], bound[rows:], "the other request")


@pytest.mark.parametrize("rows", [2, 150])
def test_pages_outside_the_cache_and_lengths_past_the_table(gpu, rows):
    """Only the rows that see such a token are NaN."""
    g = _gen(gpu, 5)
    page, n = 32, 400
    q, cache, tables, lens, starts = _batch(g, [(n, rows), (n, rows)], nh=2, kvh=1, page=page)
    y, bound = O.attention(q, cache.data, tables, lens, starts)
    for number in (-1, cache.num_pages, 2**31 - 1, -2**31):
        bad = tables.clone()
        at = (n - rows // 2) // page                   # a page that the first rows do not see
        bad[0, at] = number
        out = _call(q, cache, bad, lens, starts)
        blind = [i for i in range(rows) if n - rows + i < at * page]
        sees = [i for i in range(rows) if i not in blind]
        assert torch.isnan(out[sees]).all() and sees
        O.check(out[blind], y[blind], bound[blind], f"page {number}")
        O.check(out[rows:], y[rows:], bound[rows:], "the other request")
    # a window keeps the page out of sight of the last rows
    bad = tables.clone()
    bad[0, 0] = -1
    yw, bw = O.attention(q, cache.data, tables, lens, starts, window=100)
    O.check(_call(q, cache, bad, lens, starts, window=100), yw, bw, "behind the window")
    # a table that ends inside the rows' own tokens
    short = tables[:, :(n - rows // 2) // page].contiguous()
    limit = short.shape[1] * page
    out = _call(q, cache, short, lens, starts)
    inside = [b * rows + i for b in range(2) for i in range(rows) if n - rows + i < limit]
    outside = [i for i in range(2 * rows) if i not in inside]
    assert torch.isnan(out[outside]).all()
    O.check(out[inside], y[inside], bound[inside], "short table")
    # lengths far past the table, with and without a window that lies past it too
    far = kv16_attention(q, cache, tables, _i32([2**31 - 1, n], gpu), _i32(starts, gpu), rows, window=16)
    assert torch.isnan(far[:rows]).all()
    O.check(far[rows:], *(t[rows:] for t in O.attention(q, cache.data, tables, lens, starts, window=16)), "beside it")


@pytest.mark.parametrize("starts,lens,total,most", [([0, 3, 1, 9], [30, 30, 30], 9, 8), ([4, 4, 2, 300], [40, 9, 310], 300, 296)])
def test_starts_that_go_down_and_small_max_query(gpu, starts, lens, total, most):
    """A start below an earlier one counts as that one; rows past a max_query that is too small are NaN."""
    g = _gen(gpu, 6)
    _, cache, tables, _, _ = _batch(g, [(n, 1) for n in lens], nh=2, kvh=2)
    q = torch.randn((total, 128), generator=g, device=gpu).half()
    up = [max(starts[:b + 1]) for b in range(len(starts))]
    ends = [max(a, b) for a, b in zip(up, starts[1:])]
    out = kv16_attention(q, cache, tables, _i32(lens, gpu), _i32(starts, gpu), most)
    for b, (lo, hi) in enumerate(zip(up, ends)):
        if hi > lo:
            y, bound = O.attention(q[lo:hi], cache.data, tables[b:b + 1], lens[b:b + 1], [0, hi - lo])
            O.check(out[lo:hi], y, bound, f"request {b}")
    cut = kv16_attention(q, cache, tables, _i32(lens, gpu), _i32(starts, gpu), 2)
    for b, (lo, hi) in enumerate(zip(up, ends)):
        assert torch.isnan(cut[lo + 2:hi]).all() if hi > lo + 2 else True
        n = min(2, max(0, hi - lo))
        if n:
            y, bound = O.attention(q[lo:hi], cache.data, tables[b:b + 1], lens[b:b + 1], [0, hi - lo])
            O.check(cut[lo:lo + n], y[:n], bound[:n], f"request {b}, two rows")


@pytest.mark.parametrize("rows", [1, 200])
def test_extremes(gpu, rows):
    """Queries at fp16's largest value, bf16 near its own, scales from 1e-20 to 1e6, caps from 1e-3 to 1e6."""
    g = _gen(gpu, 7)
    q, cache, tables, lens, starts = args = _batch(g, [(300, rows), (1, 1)], nh=2, kvh=1, hd=128, page=64)
    for kw in ({"scale": 1e-20}, {"scale": 1e6}, {"softcap": 1e-3}, {"softcap": 1e6}, {"softcap": 3e4, "scale": 30.0}):
        O.check(_call(*args, **kw), *O.attention(q, cache.data, tables, lens, starts, **kw), str(kw))
    top = q.sign() * 65504
    out = _call(top, cache, tables, lens, starts)
    O.check(out, *O.attention(top, cache.data, tables, lens, starts), "65504")
    for scale in (1.0, 1e30):
        big = (q.float() * 2.0**125).to(torch.bfloat16)
        half = Kv16Cache.of(cache.data.to(torch.bfloat16))
        out = _call(big, half, tables, lens, starts, scale=scale)
        # one token has all of the weight
        y, _ = O.attention(big, half.data, tables, lens, starts, scale=scale)
        assert torch.isfinite(out).all()
        assert (out.double().view(y.shape) - y).abs().max() <= 2.0**-8 * y.abs().max()


@pytest.mark.parametrize("rows", [1, 200])
def test_products_near_fp32_s_smallest_and_caps_far_below(gpu, rows):
    """Scores that vanish beside 1, down to scales that no fp32 number but a subnormal holds, and a cap of 2^-100 over the
    largest scores and over scores of 0: all tokens weigh alike, masked ones nothing.  One tile, several, split."""
    g = _gen(gpu, 17)
    for tokens in (300, 5000):
        q, cache, tables, lens, starts = args = _batch(g, [(tokens, rows), (1, 1)], nh=2, kvh=1, hd=128, page=64)
        for kw in ({"scale": 1e-44}, {"scale": 1e-37, "softcap": 2.0**-100}):
            O.check(_call(*args, **kw), *O.attention(q, cache.data, tables, lens, starts, **kw), f"{tokens} {kw}")
        half = Kv16Cache.of(cache.data.to(torch.bfloat16))
        half.k[:, :, 5:9] = 0
        for power, kw in ((-100, {"scale": 1e-30}), (-100, {"scale": 1e-30, "softcap": 5.0}), (125, {"softcap": 2.0**-100})):
            far = (q.float() * 2.0**power).to(torch.bfloat16)
            O.check(_call(far, half, tables, lens, starts, **kw), *O.attention(far, half.data, tables, lens, starts, **kw),
                    f"{tokens} 2^{power} {kw}")


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("tokens", [300, 5000])
def test_values_near_bf16_s_largest_and_far_below(gpu, rows, tokens):
    """Their weighted mean is no larger than they are: no sum on the way may pass fp32."""
    g = _gen(gpu, 18)
    q, cache, tables, lens, starts = _batch(g, [(tokens, rows), (1, 1)], nh=2, kvh=1, hd=128, page=64, dtype="bf16")
    for size in (3.38e38, 1e-15):
        cache.v.copy_(torch.where(cache.v > 0, size, -size * 0.75))
        cache.v[..., 0] = size
        out = _call(q, cache, tables, lens, starts)
        O.check(out, *O.attention(q, cache.data, tables, lens, starts), f"{size}")
        # (of the small ones the bound's absolute term says nothing)
        y, _ = O.attention(q, cache.data, tables, lens, starts)
        assert ((out.double().view(y.shape) - y).abs() <= 2.0**-6 * size).all()


def test_strides_and_streams(gpu):
    """Rows of a wider tensor, an unaligned view, another stream than the tensors' own."""
    g = _gen(gpu, 8)
    q, cache, tables, lens, starts = args = _batch(g, [(200, 150), (70, 1)], nh=4, kvh=2)
    want = _call(*args)
    wide = torch.randn((q.shape[0], 3 * q.shape[1]), device=gpu).half()
    wide[:, 256:512] = q
    assert torch.equal(_call(wide[:, 256:512], *args[1:]), want)
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device=gpu)
    odd[1:] = q.reshape(-1)
    assert torch.equal(_call(odd[1:].view(q.shape), *args[1:]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_call(*args) for _ in range(4)]
    here = [_call(*args) for _ in range(4)]             # at the same time: each call has a workspace of its own
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got + here)


def test_in_a_graph(gpu):
    """Captured once for decode rows and once for a chunk, replayed with other lengths and eager work between."""
    g = _gen(gpu, 9)
    for rows in (1, 120):
        q, cache, tables, lens, starts = _batch(g, [(500, rows), (300, rows)], nh=4, kvh=1, width=40)
        n, s = _i32(lens, gpu), _i32(starts, gpu)
        slopes = torch.tensor([0.5, 0.25, 0.1, 0.0], device=gpu)
        call = lambda: kv16_attention(q, cache, tables, n, s, rows, slopes=slopes, softcap=30.0)  # noqa: E731
        call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call()
        torch.cuda.current_stream().wait_stream(side)
        for k in range(4):
            now = [500 - 90 * k, 300 - 5 * k]
            n.copy_(_i32(now, gpu))
            want = call()
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), k
            O.check(out, *O.attention(q, cache.data, tables, now, starts, slopes=slopes, softcap=30.0), f"replay {k}")


def test_repeats_bit_for_bit(gpu):
    g = _gen(gpu, 10)
    args = _batch(g, [(3000, 1), (3000, 400), (12, 12)], nh=8, kvh=2, dtype="bf16")
    want = _call(*args)
    assert all(torch.equal(_call(*args), want) for _ in range(5))


@pytest.mark.parametrize("rows", [1, 200])
def test_offsets_past_32_bits(gpu, rows):
    """A cache of 5 GB whose last pages are a request's."""
    pages, page, kvh, hd = 38000, 64, 4, 128           # 2.5e9 elements
    data = torch.zeros((pages, kvh, 2, page, hd), dtype=torch.float16, device=gpu)
    g = _gen(gpu, 11)
    n = 5 * page - 3
    tables = torch.arange(pages - 5, pages, dtype=torch.int32, device=gpu).flip(0).view(1, -1).contiguous()
    cos, sin = torch.ones((n, hd), device=gpu), torch.zeros((n, hd), device=gpu)
    qkv = torch.randn((n, 12 * hd), generator=g, device=gpu).half()
    pos = torch.arange(n, dtype=torch.int32, device=gpu)
    slots = tables[0, (pos // page).long()] * page + pos % page
    cache = Kv16Cache.of(data)
    q = kv16_append(qkv, cache, slots, pos, cos, sin, 4)
    assert torch.equal(q, qkv[:, :4 * hd])
    args = (q[-rows:].contiguous(), cache, tables, [n], [0, rows])
    O.check(_call(*args), *O.attention(args[0], data, *args[2:]))


# ---- the write ------------------------------------------------------------------------


def _rope(max_pos, hd, dev):
    f = torch.outer(torch.arange(max_pos, device=dev, dtype=torch.float32),
                    1.0 / 1e4 ** (torch.arange(0, hd, 2, device=dev, dtype=torch.float32) / hd))
    # halves that differ, as a caller's tables may
    return torch.cat((f, f * 1.5), -1).cos(), torch.cat((f, f * 1.5), -1).sin()


@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("nh,kvh,hd,page,dtype,n", [
    (4, 2, 64, 16, "fp16", 1), (28, 4, 128, 64, "fp16", 77), (3, 1, 128, 32, "bf16", 130), (12, 12, 64, 256, "bf16", 9),
    (1, 1, 64, 16, "fp16", 1000), (64, 1, 128, 128, "fp16", 33)])
def test_append(gpu, nh, kvh, hd, page, dtype, n, rotate):
    """q and k: three roundings of fp32 (2^-22 of the two products' sizes) and one of the type; v bit for bit; the
    other slots as they were."""
    g = _gen(gpu, 12)
    max_pos, pages = 900, -(-n // page) + 2
    qkv = torch.randn((n, (nh + 2 * kvh) * hd), generator=g, device=gpu).to(DT[dtype])
    slots = torch.randperm(pages * page, generator=g, device=gpu)[:n].to(torch.int32)
    positions = torch.randint(0, max_pos, (n,), generator=g, device=gpu, dtype=torch.int32)
    cos, sin = _rope(max_pos, hd, gpu) if rotate else (None, None)
    cache = Kv16Cache.of(torch.randn((pages, kvh, 2, page, hd), generator=g, device=gpu).to(DT[dtype]))
    before = cache.data.clone()
    q = kv16_append(qkv, cache, slots, positions, cos, sin, nh)
    x = qkv.double().view(n, nh + 2 * kvh, hd)
    turned, size = x.clone(), x.abs()
    if rotate:
        c, s = (t[positions.long()].double()[:, None] for t in (cos, sin))
        part = torch.cat((-x[..., hd // 2:], x[..., :hd // 2]), -1)
        turned, size = x * c + part * s, (x * c).abs() + (part * s).abs()
    off = torch.cat((q.view(n, nh, hd), cache.k[slots.long() // page, :, slots.long() % page]), 1).double() - turned[:, :nh + kvh]
    bound = size[:, :nh + kvh] * 2.0**-22 + turned[:, :nh + kvh].abs() * torch.finfo(DT[dtype]).eps / 2 * 1.01 + 2.0**-25
    assert (off.abs() <= (bound if rotate else 0.0)).all()
    v = qkv.view(n, nh + 2 * kvh, hd)[:, nh + kvh:]
    assert torch.equal(cache.v[slots.long() // page, :, slots.long() % page], v)
    held = torch.zeros(pages * page, dtype=torch.bool, device=gpu)
    held[slots.long()] = True
    untouched = (~held).view(pages, 1, 1, page, 1).expand_as(before)
    assert torch.equal(cache.data[untouched], before[untouched])


def test_append_what_is_not_stored(gpu):
    """Slots and positions outside: nothing is stored; q NaN only where the position is outside.  Values that are not
    finite are stored as they are."""
    g = _gen(gpu, 13)
    nh, kvh, hd, page, n = 4, 2, 64, 16, 8
    cos, sin = _rope(50, hd, gpu)
    qkv = torch.randn((n, (nh + 2 * kvh) * hd), generator=g, device=gpu).half()
    qkv[7, nh * hd:] = torch.tensor([math.nan, math.inf], device=gpu).half().repeat(2 * kvh * hd // 2)
    cache = Kv16Cache(3, kvh, hd, page, device=gpu)
    slots = _i32([-1, 48, 2**31 - 1, -2**31, 5, 6, 7, 47], gpu)
    positions = _i32([3, 4, 5, 6, -1, 50, 49, 0], gpu)
    q = kv16_append(qkv, cache, slots, positions, cos, sin, nh)
    assert torch.isnan(q[4:6]).all() and torch.isfinite(q[[0, 1, 2, 3, 6, 7]]).all()
    stored = torch.zeros(48, dtype=torch.bool, device=gpu)
    stored[[7, 47]] = True
    rows = cache.data.permute(0, 3, 1, 2, 4).reshape(48, -1)
    assert (rows[~stored] == 0).all() and (rows[7] != 0).any()
    assert torch.equal(torch.isnan(rows[47].view(kvh, 2, hd)[:, 1]), torch.isnan(qkv[7].view(-1, hd)[nh + kvh:]))
    assert torch.equal(torch.isinf(rows[47].view(kvh, 2, hd)[:, 1]), torch.isinf(qkv[7].view(-1, hd)[nh + kvh:]))


def test_append_row_stride_and_no_rows(gpu):
    g = _gen(gpu, 14)
    wide = torch.randn((9, 1000), generator=g, device=gpu).half()
    caches = [Kv16Cache(2, 2, 64, 16, device=gpu) for _ in range(3)]
    slots, positions = _i32(list(range(9)), gpu), _i32(list(range(9)), gpu)
    want = kv16_append(wide[:, 8:520].contiguous(), caches[0], slots, positions, None, None, 4)
    assert torch.equal(kv16_append(wide[:, 8:520], caches[1], slots, positions, None, None, 4), want)
    odd = wide[:, 3:515].contiguous()
    assert torch.equal(kv16_append(wide[:, 3:515], caches[2], slots, positions, None, None, 4), odd[:, :256])
    assert torch.equal(caches[0].data, caches[1].data)
    none = _i32([], gpu)
    assert kv16_append(wide[:0, 8:520], caches[0], none, none, None, None, 4).shape == (0, 256)
    assert kv16_attention(wide[:0, :256], caches[0], _i32([[0]], gpu), _i32([4], gpu), _i32([0, 0], gpu), 1).shape == (0, 256)


def test_steps_of_a_batch(gpu):
    """Prompts, then tokens one by one, through paged_step, kv16_append and kv16_attention: every step against the
    definition over what the steps before stored."""
    g = _gen(gpu, 15)
    nh, kvh, hd, page = 4, 2, 64, 16
    tables = PagedTables(3, 12, 30, page, gpu)
    cache = Kv16Cache(30, kvh, hd, page, device=gpu)
    cos, sin = _rope(200, hd, gpu)
    for new in ([40, 0, 7], [1, 33, 1], [1, 1, 1], [0, 1, 60], [1, 1, 1]):
        total = sum(new) + 2                            # two rows of no request
        qkv = torch.randn((total, (nh + 2 * kvh) * hd), generator=g, device=gpu).half()
        step = paged_step(tables, _i32(new, gpu), total)
        q = kv16_append(qkv, cache, step.slots, step.positions, cos, sin, nh)
        out = kv16_attention(q, cache, tables.block_tables, step.lengths, step.query_start, max(new), window=25)
        tables.commit(step)
        assert not step.failed.any()
        real = sum(new)
        y, bound = O.attention(q[:real], cache.data, tables.block_tables, step.lengths.tolist(), step.query_start.tolist(), window=25)
        O.check(out[:real], y, bound, str(new))
        assert (out[real:] == 0).all()


def test_refusals(gpu):
    g = _gen(gpu, 16)
    q, cache, tables, lens, starts = args = _batch(g, [(30, 2)], nh=4, kvh=2)
    n, s = _i32(lens, gpu), _i32(starts, gpu)
    ok = dict(q=q, cache=cache, block_tables=tables, seq_lens=n, query_start=s, max_query=2)
    kv16_attention(**ok)
    for change in ({"q": q.float()}, {"q": q.bfloat16()}, {"q": q[:, :192]}, {"q": q[0]}, {"q": q.cpu()}, {"block_tables": tables.long()},
                   {"block_tables": tables.cpu()}, {"block_tables": tables[0]}, {"seq_lens": n.long()}, {"seq_lens": _i32([1, 2], gpu)},
                   {"query_start": _i32([0], gpu)}, {"max_query": 0}, {"scale": 0.0}, {"scale": math.nan}, {"scale": math.inf},
                   {"scale": -1.0}, {"softcap": 0.0}, {"softcap": -3.0}, {"softcap": math.nan}, {"softcap": math.inf}, {"window": 0},
                   {"window": -1}, {"slopes": torch.zeros(3, device=gpu)}, {"slopes": torch.zeros(4, device=gpu).half()},
                   {"slopes": torch.zeros(4)}, {"prefix": _i32([1, 2], gpu)}, {"prefix": torch.tensor([1], device=gpu)},
                   {"first": _i32([0], gpu)}, {"first": torch.zeros(2, device=gpu)}):
        with pytest.raises(ValueError):
            kv16_attention(**{**ok, **change})
    for data in (cache.data.float(), cache.data[:, :, :1], cache.data[..., :32].contiguous(), cache.data[:, :, :, :8].contiguous(),
                 cache.data.transpose(0, 1), cache.data[0]):
        with pytest.raises(ValueError):
            Kv16Cache.of(data)
    qkv = torch.zeros((2, 512), dtype=torch.float16, device=gpu)
    cos = torch.zeros((5, 64), device=gpu)
    two = _i32([0, 1], gpu)
    ok = dict(qkv=qkv, cache=cache, slots=two, positions=two, cos=cos, sin=cos, num_heads=4)
    kv16_append(**ok)
    for change in ({"qkv": qkv.bfloat16()}, {"qkv": qkv[:, :500]}, {"num_heads": 3}, {"slots": two.long()}, {"positions": two[:1]},
                   {"cos": None}, {"sin": cos[:, :32]}, {"cos": cos.half()}, {"sin": cos[:4]}):
        with pytest.raises(ValueError):
            kv16_append(**{**ok, **change})
    assert _native.lib().awq_serve_kv16_attention_workspace(1, 1, 1, 4, 3, 64, 1, 16) == 0
