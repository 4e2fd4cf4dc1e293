"""``kv4_attention`` where its loops go round: items of many passes and tiles, more pages in an
item than a wave holds at once, more items of a row than a combining wave joins at once,
batches of more requests than a wave has lanes, and scores that rise along the tokens, so that
what was summed up is rescaled.  Which of these a case reaches is asserted from the kernels'
own arithmetic (``attention_items.cpp``).

The bound per element: one rounding of the result to its type (2^-11 of it for fp16, 2^-8
for bf16, or half of fp16's smallest step), and 2^-13 of the largest |v| for the fp32 work:
an error e of the scores moves the result by at most 2 e max|v|, e being five accumulations of
sums of up to 60 (after scaling), 5 * 60 * 2^-24 = 1.8e-5; up to 512 accumulations of the
probabilities' sums add 512 * 2^-24 = 3.1e-5; together 6.7e-5, doubled for the order of the
sums within a product.
"""
import math

import kv4_oracle as O
import numpy as np
import pytest
import torch
from test_attention_items import walk  # noqa: F401  (a fixture)
from test_gpu_kv4 import DT, _i32

from kernels.kv4 import Kv4Cache, kv4_attention

pytestmark = pytest.mark.gpu


def _pool(rng, pages, page, kvh, hd, group, rising):
    """(packed cache, k, v) of `pages` pages; rising: keys grow from page to page."""
    parts = []
    for key in (True, False):
        x = rng.standard_normal((pages, page, kvh, hd))
        if key and rising:
            x = 0.2 * x + np.linspace(0.0, 1.0, pages)[:, None, None, None]
        parts.append(O.quantise(x.reshape(pages * page, kvh, hd).astype(np.float32), group)[:3])
    return O.pack(*parts, pages, page, hd, group), O.values(parts[0], group), O.values(parts[1], group)


def _attend(q, k, v, slots, rows):
    """float64 [rows, heads, hd] of a request's last rows over its tokens."""
    heads, hd = q.shape[1:]
    each, n = heads // k.shape[1], len(slots)
    hidden = np.arange(n)[None] > np.arange(n - rows, n)[:, None]
    out = np.zeros(q.shape)
    for h in range(heads if n and rows else 0):
        s = q[:, h] @ k[slots, h // each].T / math.sqrt(hd)
        assert np.abs(s).max(initial=0.0) <= 60.0
        s[hidden] = -np.inf
        some = ~hidden.all(1)
        p = np.exp(s[some] - s[some].max(1, keepdims=True))
        out[some, h] = p @ v[slots, h // each] / p.sum(1, keepdims=True)
    return out


def _run(gpu, seed, heads, kvh, hd, page, group, dtype, requests, rising=False):
    rng = np.random.default_rng(seed)
    pages = 24
    data, k, v = _pool(rng, pages, page, kvh, hd, group, rising)
    cache = Kv4Cache.of(torch.from_numpy(data).to(gpu), hd, page, group)
    width = max(-(-n // page) for n, _ in requests) + 1
    table = np.full((len(requests), width), -1, np.int32)
    for b, (n, _) in enumerate(requests):
        held = rng.integers(0, pages, -(-n // page))           # pages of the pool again and again
        table[b, :len(held)] = np.sort(held) if rising else held
    starts = np.concatenate(([0], np.cumsum([m for _, m in requests]))).astype(np.int64)
    x = rng.standard_normal((int(starts[-1]), heads * hd))
    if rising:
        x = 0.5 * x + 1.0
    q = torch.from_numpy(x.astype(np.float32)).to(DT[dtype])
    y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32([n for n, _ in requests], gpu), _i32(starts, gpu),
                      max(m for _, m in requests))
    got = y.double().cpu().numpy().reshape(-1, heads, hd)
    assert np.isfinite(got).all()
    q = q.double().numpy().reshape(-1, heads, hd)
    unit, work = (2.0**-11 if dtype == "fp16" else 2.0**-8), 2.0**-13 * np.abs(v).max()
    for b, (n, m) in enumerate(requests):
        i = np.arange(n)
        lo, hi = starts[b], starts[b + 1]
        ref = _attend(q[lo:hi], k, v, table[b][i // page].astype(np.int64) * page + i % page, m)
        worst = (np.abs(got[lo:hi] - ref) / (np.abs(ref) * unit + 2.0**-25 + work)).max(initial=0.0)
        assert worst <= 1.0, f"request {b} of {n} tokens, {m} rows: {worst:.2f} of the bound"


DECODE = [
    # heads, kv heads, head size, page, group, dtype, requests, rising, passes of an item at least
    (8, 8, 64, 16, 64, "fp16", [(3000 + 7 * i, 1) for i in range(20)], False, 4),
    (16, 8, 64, 16, 32, "bf16", [(3500 + 11 * i, 1) for i in range(30)], False, 9),      # more than 64 pages in an item
    (16, 8, 128, 16, 64, "fp16", [(4100 - 13 * i, 1) for i in range(30)], True, 9),
    (8, 4, 128, 64, 128, "fp16", [(4000 + i, 1 + i % 3) for i in range(24)], True, 2),
    (8, 4, 128, 256, 32, "bf16", [(5000 - 17 * i, 1) for i in range(20)], False, 3),
    (28, 4, 128, 64, 64, "fp16", [(1000 + 190 * i, 1) for i in range(32)], True, 3),
    (14, 2, 64, 32, 64, "bf16", [(9000 + 31 * i, 2) for i in range(20)], True, 3),
]


@pytest.mark.parametrize("heads,kvh,hd,page,group,dtype,requests,rising,steps", DECODE)
def test_decode_items_of_many_passes(gpu, walk, heads, kvh, hd, page, group, dtype, requests, rising, steps):  # noqa: F811
    decode, tiles, _ = walk(requests, heads // kvh, kvh, page=page)
    assert decode.steps >= steps and tiles.items == 0
    _run(gpu, heads + hd, heads, kvh, hd, page, group, dtype, requests, rising)


TILES = [
    # heads, kv heads, head size, page, group, dtype, requests, rising, tiles of an item at least, places for sums
    (32, 8, 64, 16, 64, "fp16", [(600, 600)], False, 9, False),             # a whole prompt, not split
    (32, 8, 64, 16, 32, "bf16", [(1500, 530)], True, 20, False),            # ... with more than 64 pages
    (32, 8, 128, 64, 64, "fp16", [(777, 560)], True, 12, False),
    (32, 8, 128, 16, 128, "fp16", [(700, 520)], False, 10, False),
    (32, 8, 128, 256, 32, "bf16", [(641, 540)], True, 10, False),
    (28, 4, 128, 64, 64, "fp16", [(601, 601)], True, 9, False),
    (64, 8, 64, 64, 64, "fp16", [(4000, 40)], True, 2, True),               # split along the tokens
    (32, 32, 128, 16, 64, "fp16", [(8000, 150)], True, 10, True),
    (64, 32, 64, 16, 64, "bf16", [(20000, 70)], False, 17, True),           # ... with more than 64 pages in an item
    (16, 4, 128, 64, 32, "fp16", [(5000, 90), (3000, 70), (4000, 33)], True, 2, True),
]


@pytest.mark.parametrize("heads,kvh,hd,page,group,dtype,requests,rising,steps,places", TILES)
def test_tile_items_of_many_tiles(gpu, walk, heads, kvh, hd, page, group, dtype, requests, rising, steps, places):  # noqa: F811
    _, tiles, has_places = walk(requests, heads // kvh, kvh, page=page)
    assert tiles.steps >= steps and has_places == places
    _run(gpu, heads + hd, heads, kvh, hd, page, group, dtype, requests, rising)


@pytest.mark.parametrize("heads,kvh,hd,requests,splits", [
    (4, 1, 64, [(40000, 1)], 257),                          # four combining waves, each more than 64 items
    (7, 1, 128, [(35000, 2), (50, 1)], 257),
    (64, 1, 64, [(12000, 1)] + [(20, 1)] * 8, 65),          # one combining wave
])
def test_more_items_of_a_row_than_a_combining_wave_has_lanes(gpu, walk, heads, kvh, hd, requests, splits):  # noqa: F811
    decode, _, _ = walk(requests, heads // kvh, kvh)
    assert decode.splits >= splits
    _run(gpu, heads, heads, kvh, hd, 64, 64, "fp16", requests, rising=True)


@pytest.mark.parametrize("n", [64, 65, 130, 300])
@pytest.mark.parametrize("heads,kvh,hd,page", [(8, 2, 64, 16), (14, 2, 128, 64)])
def test_many_requests(gpu, n, heads, kvh, hd, page):
    """Single tokens, chunks of prompts and whole ones, requests without rows and without tokens, one after another."""
    rng = np.random.default_rng(n)
    requests = []
    for b in range(n):
        kind, length = rng.integers(0, 6), int(rng.integers(1, 400))
        requests.append([(length, 1), (length, 1), (length, 0), (0, 3), (length, min(length, 50)), (length, 2)][kind])
    requests[n - 1] = (333, 70)
    requests[n // 2] = (2000, 1)
    _run(gpu, n, heads, kvh, hd, page, 64, "fp16", requests)
