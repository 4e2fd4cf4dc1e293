"""The 4-bit paged cache and its attention (``kernels/kv4.py``) against plain
numpy in 64 bits (``kv4_oracle``).

Codes, scales and zeros are decided in fp32 by a fixed sequence of correctly
rounded steps: the stored bytes have to be equal.

Attention's bound per element: one rounding of the result to its type (2^-11 of
it for fp16, 2^-8 for bf16, or half of fp16's smallest step), and for the fp32
work before it 5e-5 of the largest value: a score is a sum of 128 terms and their
zeros' parts, each of magnitude up to about 50 here, so it errs by a few times
50 sqrt(128) 2^-24 = 3e-5 at most, and an error e of a score moves its
probability by e.
"""
import math

import kv4_oracle as O
import numpy as np
import pytest
import torch

from kernels import _native
from kernels.kv4 import Kv4Cache, kv4_append, kv4_attention, kv4_gather

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _cache(rng, pages, page, kvh, hd, group, dev, k_gain=3.0):
    """(cache on the device, k values, v values in 64 bits) of random content."""
    parts = []
    for gain in (k_gain, 0.0):
        x = rng.standard_normal((pages * page, kvh, hd)) * (1.0 + gain * rng.random((kvh, hd)) ** 8)
        parts.append(O.quantise(x.astype(np.float32), group)[:3])
    data = torch.from_numpy(O.pack(*parts, pages, page, hd, group)).to(dev)
    return Kv4Cache.of(data, hd, page, group), O.values(parts[0], group), O.values(parts[1], group)


def _batch(rng, requests, page, extra_pages=2, width=None):
    """Lengths, first rows and block tables (random pages) of [(length, rows)]."""
    lengths = [n for n, _ in requests]
    starts = np.concatenate(([0], np.cumsum([m for _, m in requests]))).astype(np.int32)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + extra_pages
    order = rng.permutation(pages).astype(np.int32)
    width = width or max(held) + 1
    table = np.full((len(requests), width), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return lengths, starts, table, pages


def _i32(a, dev):
    return torch.tensor(np.asarray(a, dtype=np.int32), device=dev)


def _close(y, ref, dtype, what):
    y = y.double().cpu().numpy().reshape(ref.shape)
    unit = 2.0**-11 if dtype == "fp16" else 2.0**-8
    bound = np.abs(ref) * unit + 2.0**-25 + 5e-5 * np.abs(ref).max()
    worst = (np.abs(y - ref) / bound).max() if ref.size else 0.0
    assert np.isfinite(y).all() and worst <= 1.0, f"{what}: {worst:.2f} of the bound"


CASES = [
    # heads, kv heads, head size, page, group, dtype, [(length, rows)]
    (28, 4, 128, 64, 64, "fp16", [(1, 1), (17, 1), (64, 1), (65, 1), (130, 1), (700, 1)]),
    (28, 4, 128, 16, 128, "bf16", [(127, 1), (128, 1), (129, 1), (15, 1)]),
    (8, 8, 128, 32, 32, "fp16", [(33, 1), (300, 1)]),
    (4, 2, 64, 16, 32, "bf16", [(5, 5), (33, 2), (0, 0), (100, 7), (1, 1)]),
    (18, 1, 64, 128, 64, "fp16", [(299, 1), (16, 3)]),           # more heads than a workgroup's columns
    (64, 1, 64, 16, 64, "fp16", [(90, 2), (31, 1)]),
    (14, 2, 64, 256, 64, "fp16", [(257, 1), (511, 4)]),
    (4, 2, 128, 16, 64, "fp16", [(150, 150)]),                   # a whole prompt
    (28, 4, 128, 64, 64, "fp16", [(190, 61), (77, 77), (203, 1), (2, 2)]),
    (6, 2, 64, 32, 64, "bf16", [(400, 129), (65, 64), (300, 33)]),
    (2, 2, 128, 16, 32, "fp16", [(70, 65)]),
    (2, 1, 64, 16, 64, "fp16", [(5000, 1), (3, 1)]),             # several items along the tokens
    (4, 1, 64, 64, 32, "fp16", [(2100, 40), (900, 1)]),
    (2, 2, 128, 64, 32, "fp16", [(200, 150)]),                   # more than 128 columns of a kv head
    (4, 2, 128, 16, 32, "bf16", [(190, 100), (40, 1), (66, 65)]),
    (8, 2, 128, 64, 128, "bf16", [(140, 70), (90, 33)]),
    (64, 1, 64, 64, 32, "fp16", [(70, 3), (65, 1)]),
    (12, 4, 64, 128, 64, "fp16", [(1500, 90)]),
]


@pytest.mark.parametrize("nh,kvh,hd,page,group,dtype,requests", CASES)
def test_attention(gpu, nh, kvh, hd, page, group, dtype, requests):
    rng = np.random.default_rng(nh * 1000 + hd + len(requests))
    lengths, starts, table, pages = _batch(rng, requests, page)
    cache, k, v = _cache(rng, pages, page, kvh, hd, group, gpu)
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]), nh * hd)).astype(np.float32)).to(DT[dtype])
    y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu),
                      max(m for _, m in requests))
    assert y.dtype == DT[dtype]
    ref = O.attend(q.double().numpy().reshape(-1, nh, hd), k, v, lengths, starts, table, page)
    _close(y, ref, dtype, "attention")


@pytest.mark.parametrize("rows", [1, 40, 70])
def test_attention_rows_that_see_nothing_and_rows_of_no_request(gpu, rows):
    """Three tokens under `rows` rows more than that: the first rows stand before the
    first token; a request without tokens; rows past the last request's."""
    rng = np.random.default_rng(3)
    requests = [(3, 3 + rows), (0, rows), (20, rows)]
    lengths, starts, table, pages = _batch(rng, requests, 16)
    cache, k, v = _cache(rng, pages, 16, 2, 64, 64, gpu)
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]) + 5, 4 * 64)).astype(np.float32)).half()
    y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), 3 + rows)
    ref = O.attend(q.double().numpy().reshape(-1, 4, 64), k, v, lengths, starts, table, 16)
    _close(y, ref, "fp16", "empty rows")
    y = y.cpu()
    assert (y[:rows] == 0).all() and (y[starts[1]:starts[2]] == 0).all() and (y[starts[-1]:] == 0).all()
    assert (y[rows] != 0).any()


@pytest.mark.parametrize("rows", [1, 33, 70])
def test_attention_reads_nothing_of_what_lies_past_the_length(gpu, rows):
    """Bytes that are NaN scales everywhere but in the request's tokens, and table
    entries outside the cache past its pages."""
    rng = np.random.default_rng(4)
    page, kvh, hd, group, n = 32, 2, 128, 64, 75
    lengths, starts, table, pages = _batch(rng, [(n, rows)], page, width=9)
    table[0, 3:] = [2**30, -2**31, 7777, -1, 5, 2**31 - 1]
    cache, k, v = _cache(rng, pages, page, kvh, hd, group, gpu)
    held = [table[0][i // page] * page + i % page for i in range(n)]
    mask = torch.from_numpy(O.bytes_of(held, pages, page, kvh, hd, group)).to(gpu)
    cache = Kv4Cache.of(cache.data | ~mask, hd, page, group)
    q = torch.from_numpy(rng.standard_normal((rows, 4 * hd)).astype(np.float32)).half()
    y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu),
                      _i32(starts, gpu), rows)
    _close(y, O.attend(q.double().numpy().reshape(-1, 4, hd), k, v, lengths, starts, table, page), "fp16", "past the length")


@pytest.mark.parametrize("rows", [4, 40, 70])
def test_a_token_that_is_not_finite_reaches_only_the_rows_that_see_it(gpu, rows):
    """k or v with a NaN or an infinity at the next to last position: the rows before it are as without it."""
    rng = np.random.default_rng(5)
    page, kvh, hd, nh, n = 16, 2, 64, 4, 60
    lengths, starts, table, pages = _batch(rng, [(n, rows)], page)
    for part, bad in ((1, math.nan), (2, math.inf), (2, math.nan)):
        cache, k, v = _cache(rng, pages, page, kvh, hd, 64, gpu)
        qkv = torch.zeros((1, (nh + 2 * kvh) * hd), dtype=torch.float16)
        qkv[0, nh * hd + (part - 1) * kvh * hd + 3] = bad                # kv head 0
        at = n - 2
        slot = table[0][at // page] * page + at % page
        kv4_append(qkv.to(gpu), cache, _i32([slot], gpu), _i32([0], gpu), None, None, nh)
        q = torch.from_numpy(rng.standard_normal((rows, nh * hd)).astype(np.float32)).half()
        y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), rows).cpu()
        y = y.view(rows, nh, hd)
        assert torch.isnan(y[-2:, :2]).all(), "rows that see it, query heads of kv head 0"
        k[slot, 1], v[slot, 1] = 0.0, 0.0
        ref = O.attend(q.double().numpy().reshape(-1, nh, hd), k, v, lengths, starts, table, page)
        _close(y[:-2], ref[:-2], "fp16", "rows before it")
        _close(y[-2:, 2:], ref[-2:, 2:], "fp16", "the other kv head")


def test_attention_pages_outside_the_cache_and_lengths_past_the_table_give_nan(gpu):
    rng = np.random.default_rng(6)
    requests = [(40, 1), (40, 1), (40, 1), (40, 2)]
    lengths, starts, table, pages = _batch(rng, requests, 16, width=3)
    cache, k, v = _cache(rng, pages, 16, 1, 64, 64, gpu)
    q = torch.from_numpy(rng.standard_normal((5, 64)).astype(np.float32)).half()
    broken = table.copy()
    broken[0, 1] = -1
    broken[1, 2] = pages
    y = kv4_attention(q.to(gpu), cache, _i32(broken, gpu), _i32([40, 40, 40, 2**31 - 1], gpu), _i32(starts, gpu), 2).cpu()
    assert torch.isnan(y[:2]).all() and torch.isnan(y[3:]).all()
    ref = O.attend(q.double().numpy().reshape(-1, 1, 64), k, v, lengths, starts, table, 16)
    _close(y[2:3], ref[2:3], "fp16", "the request beside them")


def test_attention_extremes(gpu):
    """Groups over nearly the whole of fp16, groups of one value, tiny groups; large and tiny queries."""
    rng = np.random.default_rng(7)
    page, hd, n = 16, 64, 40
    for gain, q_gain in ((30000.0, 1e-6), (1e-7, 60000.0), (0.0, 1.0)):
        lengths, starts, table, pages = _batch(rng, [(n, 1)], page)
        parts = []
        for _ in range(2):
            x = (rng.random((pages * page, 1, hd)) * 2 - 1) * gain
            parts.append(O.quantise((x + (gain == 0.0)).astype(np.float32), 32)[:3])
        cache = Kv4Cache.of(torch.from_numpy(O.pack(*parts, pages, page, hd, 32)).to(gpu), hd, page, 32)
        q = torch.from_numpy((rng.standard_normal((1, hd)) * q_gain).clip(-65504, 65504).astype(np.float32)).half()
        y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), 1)
        ref = O.attend(q.double().numpy().reshape(1, 1, hd), O.values(parts[0], 32), O.values(parts[1], 32), lengths,
                       starts, table, page)
        _close(y, ref, "fp16", f"values of {gain}")


def test_attention_strides_scale_and_streams(gpu):
    rng = np.random.default_rng(8)
    requests = [(100, 3), (41, 1)]
    lengths, starts, table, pages = _batch(rng, requests, 16)
    cache, k, v = _cache(rng, pages, 16, 2, 64, 32, gpu)
    wide = torch.from_numpy(rng.standard_normal((4, 7 * 64 + 8)).astype(np.float32)).half().to(gpu)
    args = (cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), 3)
    ref = O.attend(wide[:, 8:8 + 256].double().cpu().numpy().reshape(-1, 4, 64), k, v, lengths, starts, table, 16, 0.3)
    inside = wide[:, 8:8 + 256]                             # rows of a wider tensor
    _close(kv4_attention(inside, *args, scale=0.3), ref, "fp16", "row stride")
    odd = torch.empty(4 * 256 + 1, dtype=torch.float16, device=gpu)[1:].view(4, 256).copy_(inside)
    _close(kv4_attention(odd, *args, scale=0.3), ref, "fp16", "odd offset")
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        y = kv4_attention(inside, *args, scale=0.3)
    torch.cuda.current_stream(gpu).wait_stream(side)
    _close(y, ref, "fp16", "another stream")


def test_attention_in_a_graph(gpu):
    """Captured once; lengths and queries change under it, every replay as the eager call."""
    rng = np.random.default_rng(9)
    requests = [(90, 1), (33, 1), (200, 1)]
    lengths, starts, table, pages = _batch(rng, requests, 16, width=16)
    cache, _, _ = _cache(rng, pages, 16, 2, 64, 64, gpu)
    q = torch.randn((3, 8 * 64), device=gpu).half()
    table, lengths, starts = _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu)
    kv4_attention(q, cache, table, lengths, starts, 1)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = kv4_attention(q, cache, table, lengths, starts, 1)
    torch.cuda.current_stream(gpu).wait_stream(side)
    for step in range(4):
        q.copy_(torch.randn_like(q))
        lengths.copy_(_i32([90 - step, 33 - 8 * step, 200 - step], gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, kv4_attention(q, cache, table, lengths, starts, 1)), f"replay {step}"


def test_attention_repeats_bit_for_bit(gpu):
    rng = np.random.default_rng(10)
    lengths, starts, table, pages = _batch(rng, [(3000, 1), (70, 40)], 64)
    cache, _, _ = _cache(rng, pages, 64, 1, 64, 64, gpu)
    q = torch.randn((41, 4 * 64), device=gpu).half()
    args = (cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), 40)
    y = kv4_attention(q, *args)
    for _ in range(3):
        assert torch.equal(y, kv4_attention(q, *args))


# ---- append and gather -------------------------------------------------------------


def _append_reference(qkv, data, slots, positions, cos, sin, nh, kvh, hd, page, group):
    """q (float32) and the cache's bytes after the rows, one by one."""
    n = qkv.shape[0]
    x = qkv.reshape(n, nh + 2 * kvh, hd).astype(np.float32)
    on = np.ones(n, bool) if cos is None else (positions >= 0) & (positions < cos.shape[0])
    qk = x[:, :nh + kvh]
    if cos is not None:
        at = np.where(on, positions, 0)
        qk = O.rope(qk, cos[at], sin[at])
    k, v = O.quantise(qk[:, nh:], group), O.quantise(x[:, nh + kvh:], group)
    pages, groups = data.shape[0], hd // group
    out = data.copy()
    for i in range(n):
        if not on[i] or not 0 <= slots[i] < pages * page:
            continue
        held = k[3][i] & v[3][i]                             # [kvh]
        full = []
        for part, nan in ((k, True), (v, False)):
            codes, scale, zero = (np.zeros((pages * page, kvh, hd), np.uint8),
                                  *(np.zeros((pages * page, kvh, groups), np.float16) for _ in range(2)))
            codes[slots[i]] = np.where(held[:, None], part[0][i], 0)
            fill = np.float16(np.nan if nan else 0.0)
            scale[slots[i]] = np.where(held[:, None], part[1][i], fill)
            zero[slots[i]] = np.where(held[:, None], part[2][i], fill)
            full.append((codes, scale, zero))
        mask = O.bytes_of([slots[i]], pages, page, kvh, hd, group)
        out = (out & ~mask) | (O.pack(*full, pages, page, hd, group) & mask)
    q = np.where(on[:, None, None], qk[:, :nh], np.nan)
    return q.reshape(n, nh * hd), out


def _same_cache(got, want, kvh, hd, page, group):
    """Equal bytes, a NaN being as good as another."""
    got, want = got.cpu().numpy(), want
    codes = page * hd
    assert np.array_equal(got[..., :codes], want[..., :codes]), "codes"
    a, b = (np.ascontiguousarray(x[..., codes:]).view(np.float16) for x in (got, want))
    assert np.array_equal(np.isnan(a), np.isnan(b)), "tokens that are not finite"
    assert np.array_equal(np.nan_to_num(a), np.nan_to_num(b)), "scales and zeros"


@pytest.mark.parametrize("nh,kvh,hd,page,group,dtype,n,rotate", [
    (28, 4, 128, 64, 64, "fp16", 5, True),
    (28, 4, 128, 16, 32, "bf16", 3, True),
    (2, 2, 128, 32, 128, "fp16", 7, True),
    (3, 1, 64, 16, 32, "fp16", 9, True),
    (14, 2, 64, 16, 64, "bf16", 1, True),
    (5, 5, 64, 32, 64, "fp16", 4, False),
])
def test_append(gpu, nh, kvh, hd, page, group, dtype, n, rotate):
    rng = np.random.default_rng(nh + n)
    pages, max_pos = 2, 50
    x = (rng.standard_normal((n, (nh + 2 * kvh) * hd)) * 3).astype(np.float32)
    x[0, nh * hd:nh * hd + group] = 2.5                       # a group of one value
    qkv = torch.from_numpy(x).to(DT[dtype])
    slots = rng.permutation(pages * page)[:n].astype(np.int32)
    positions = rng.integers(0, max_pos, n).astype(np.int32)
    angle = rng.random((max_pos, hd)).astype(np.float32) * 6
    cos, sin = (np.cos(angle), np.sin(angle)) if rotate else (None, None)
    before = rng.integers(0, 256, (pages, kvh, O.block_bytes(hd, page, group))).astype(np.uint8)
    before.view(np.float16)[..., page * hd // 2:] = 1.0       # (scales that compare)
    cache = Kv4Cache.of(torch.from_numpy(before.copy()).to(gpu), hd, page, group)
    dev = lambda a: None if a is None else torch.from_numpy(a).to(gpu)  # noqa: E731
    q = kv4_append(qkv.to(gpu), cache, dev(slots), dev(positions), dev(cos), dev(sin), nh)
    q_ref, data = _append_reference(qkv.float().numpy(), before, slots, positions, cos, sin, nh, kvh, hd, page, group)
    assert torch.equal(q.cpu(), torch.from_numpy(q_ref.astype(np.float32)).to(DT[dtype]))
    _same_cache(cache.data, data, kvh, hd, page, group)
    # and read back: code * scale + zero, rounded once
    k, v = kv4_gather(cache, dev(slots), dtype=DT[dtype])
    xs = qkv.float().numpy().reshape(n, -1, hd)
    kr = xs[:, nh:nh + kvh]
    if rotate:
        kr = O.rope(kr, cos[positions], sin[positions])
    for got, part in ((k, O.quantise(kr, group)), (v, O.quantise(xs[:, nh + kvh:], group))):
        want = torch.from_numpy(O.values(part[:3], group)).float().to(DT[dtype])
        assert torch.equal(got.cpu(), want)


def test_append_what_cannot_be_stored(gpu):
    """Slots and positions outside; values that are not finite, or that fp16 cannot hold."""
    rng = np.random.default_rng(12)
    nh, kvh, hd, page, group, n, max_pos = 2, 2, 64, 16, 32, 9, 8
    x = rng.standard_normal((n, (nh + 2 * kvh) * hd)).astype(np.float32)
    x[5, nh * hd + 7] = np.nan
    x[6, (nh + kvh) * hd + 70] = -np.inf
    x[7, nh * hd:nh * hd + 2] = [65504, 60000]               # rotated past 65504, or a range too wide
    x[8, (nh + kvh) * hd:(nh + kvh) * hd + 2] = [-40000, 40000]
    qkv = torch.from_numpy(x).half()
    slots = np.array([0, -1, 32, 3, 4, 5, 6, 7, 8], np.int32)
    positions = np.array([0, 1, 2, -1, max_pos, 5, 6, 7, 1], np.int32)
    angle = rng.random((max_pos, hd)).astype(np.float32) * 6
    cos, sin = np.cos(angle), np.sin(angle)
    before = np.zeros((2, kvh, O.block_bytes(hd, page, group)), np.uint8)
    cache = Kv4Cache.of(torch.from_numpy(before.copy()).to(gpu), hd, page, group)
    dev = lambda a: torch.from_numpy(a).to(gpu)  # noqa: E731
    q = kv4_append(qkv.to(gpu), cache, dev(slots), dev(positions), dev(cos), dev(sin), nh).cpu()
    q_ref, data = _append_reference(qkv.float().numpy(), before, slots, positions, cos, sin, nh, kvh, hd, page, group)
    assert torch.isnan(q[3:5]).all() and torch.isfinite(q[[0, 1, 2, 5]]).all()
    assert torch.equal(q[:3], torch.from_numpy(q_ref.astype(np.float32)).half()[:3])
    _same_cache(cache.data, data, kvh, hd, page, group)
    k, v = kv4_gather(cache, dev(np.array([5, 6, 8, 0, -1, 32], np.int32)))
    assert torch.isnan(k[0, 0]).all() and (v[0, 0] == 0).all() and torch.isfinite(k[0, 1]).all()
    assert torch.isnan(k[1, 1]).all() and torch.isfinite(k[1, 0]).all()
    assert torch.isnan(k[2, 0]).all() and torch.isfinite(k[3]).all()
    assert torch.isnan(k[4:]).all() and torch.isnan(v[4:]).all()


def test_append_row_stride_and_no_rows(gpu):
    rng = np.random.default_rng(13)
    nh, kvh, hd = 4, 2, 64
    n = (nh + 2 * kvh) * hd
    wide = torch.from_numpy(rng.standard_normal((6, n + 24)).astype(np.float32)).half().to(gpu)
    slots, positions = _i32(range(6), gpu), _i32([0] * 6, gpu)
    results = []
    for qkv in (wide[:, 8:8 + n], wide[:, 8:8 + n].contiguous(), wide[:, 8:8 + n].t().contiguous().t()):
        cache = Kv4Cache(1, kvh, hd, 16, 64, gpu)
        results.append((kv4_append(qkv, cache, slots, positions, None, None, nh), cache.data))
    for q, data in results[1:]:
        assert torch.equal(q, results[0][0]) and torch.equal(data, results[0][1])
    assert torch.equal(results[0][0], wide[:, 8:8 + nh * hd])
    empty = kv4_append(wide[:0, :n], Kv4Cache(1, kvh, hd, 16, 64, gpu), slots[:0], positions[:0], None, None, nh)
    assert empty.shape == (0, nh * hd)
    k, v = kv4_gather(Kv4Cache(1, kvh, hd, 16, 64, gpu), slots[:0])
    assert k.shape == v.shape == (0, kvh, hd)
    y = kv4_attention(empty, Kv4Cache(1, kvh, hd, 16, 64, gpu), _i32([[0]], gpu), _i32([0], gpu), _i32([0, 0], gpu), 1)
    assert y.shape == (0, nh * hd)


def test_offsets_past_32_bits(gpu):
    """A cache of more than 4 GiB: its last page holds what was stored there."""
    kvh, hd, page, group = 4, 128, 256, 128
    pages = (2**32 + 2**28) // (kvh * Kv4Cache.block_bytes(hd, page, group))
    cache = Kv4Cache.of(torch.zeros((pages, kvh, Kv4Cache.block_bytes(hd, page, group)), dtype=torch.uint8, device=gpu),
                        hd, page, group)
    n = 40
    qkv = torch.randn((n, (8 + 2 * kvh) * hd), device=gpu).half()
    first = (pages - 1) * page
    small = Kv4Cache(1, kvh, hd, page, group, gpu)
    q = kv4_append(qkv, cache, _i32(range(first, first + n), gpu), _i32([0] * n, gpu), None, None, 8)
    kv4_append(qkv, small, _i32(range(n), gpu), _i32([0] * n, gpu), None, None, 8)
    assert torch.equal(cache.data[-1], small.data[0]) and not cache.data[:-1].any()
    rest = (_i32([n], gpu), _i32([0, n], gpu), n)
    assert torch.equal(kv4_attention(q, cache, _i32([[pages - 1]], gpu), *rest),
                       kv4_attention(q, small, _i32([[0]], gpu), *rest))
    a, b = kv4_gather(cache, _i32([first + 3], gpu)), kv4_gather(small, _i32([3], gpu))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals(gpu):
    cache = Kv4Cache(2, 2, 64, 16, 64, gpu)
    q = torch.zeros((1, 4 * 64), dtype=torch.float16, device=gpu)
    qkv = torch.zeros((1, 8 * 64), dtype=torch.float16, device=gpu)
    one, table, starts = _i32([0], gpu), _i32([[0]], gpu), _i32([0, 1], gpu)
    cos = torch.zeros((4, 64), device=gpu)
    for bad in (lambda: kv4_append(qkv.float(), cache, one, one, cos, cos, 4),
                lambda: kv4_append(qkv, cache, one, one, cos, cos, 3),
                lambda: kv4_append(qkv, cache, one.long(), one, cos, cos, 4),
                lambda: kv4_append(qkv, cache, one, _i32([0, 1], gpu), cos, cos, 4),
                lambda: kv4_append(qkv, cache, one, one, cos, None, 4),
                lambda: kv4_append(qkv, cache, one, one, cos[:, :32], cos, 4),
                lambda: kv4_append(qkv, cache, one.cpu(), one, cos, cos, 4),
                lambda: kv4_gather(cache, one, dtype=torch.float32),
                lambda: kv4_gather(cache, one.long()),
                lambda: kv4_attention(q.float(), cache, table, one, starts, 1),
                lambda: kv4_attention(q[:, :192], cache, table, one, starts, 1),
                lambda: kv4_attention(q, cache, table.long(), one, starts, 1),
                lambda: kv4_attention(q, cache, table, one, one, 1),
                lambda: kv4_attention(q, cache, table, one, starts, 0),
                lambda: kv4_attention(q, cache, table, one, starts, 1, scale=0.0),
                lambda: kv4_attention(q, cache, table, one, starts, 1, scale=math.nan),
                lambda: kv4_attention(torch.zeros((1, 130 * 64), dtype=torch.float16, device=gpu), cache, table, one, starts, 1)):
        with pytest.raises(ValueError):
            bad()
    # the C entry's own checks, with statuses
    L = _native.lib()
    assert L.awq_serve_kv4_attention(q.data_ptr(), 256, cache.data.data_ptr(), table.data_ptr(), one.data_ptr(),
                                     starts.data_ptr(), q.data_ptr(), 1, 1, 1, 4, 2, 64, 1, 2, 16, 64, 0.1, 0,
                                     q.data_ptr(), 16, 0) == _native.AWQ_ERR_WORKSPACE
