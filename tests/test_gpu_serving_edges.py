"""The serving operators where a caller's numbers are out of the ordinary: values on
the device that no host check sees, bounds that are too small, and batches so long that
the kernels' loops go round more than once."""
import kv4_oracle as O
import numpy as np
import pytest
import torch
from test_gpu_kv4 import DT, _batch, _cache, _close, _i32

from test_gpu_logits import _check

from kernels.kv4 import Kv4Cache, kv4_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts,total,rows", [
    ([0, 3, 1, 4, 4, 2, 9], 12, 3),
    ([5, 2, 9, -7, 2**31 - 1, 30, -2**31], 33, 40),
    ([0, 70, 0, 70, 10, 140], 140, 70),                       # tiles
    ([0, 2] * 70 + [150], 150, 20),                           # the largest start so far passes from 64 requests on to the next
    ([0, 40] * 50 + [1000], 1000, 960),                       # ... also where prompts are not split
])
def test_starts_that_go_down(gpu, starts, total, rows):
    """A start below an earlier one counts as that one."""
    rng = np.random.default_rng(len(starts))
    lengths, _, table, pages = _batch(rng, [(int(rng.integers(0, 90)), 0) for _ in starts[1:]], 16)
    cache, k, v = _cache(rng, pages, 16, 2, 64, 64, gpu)
    q = torch.from_numpy(rng.standard_normal((total, 8 * 64)).astype(np.float32)).half()
    args = (q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu))
    meant = np.maximum.accumulate(np.clip(starts, 0, total))
    rows = max(rows, int(np.diff(meant).max()))
    y = kv4_attention(*args, _i32(starts, gpu), rows)
    _close(y, O.attend(q.double().numpy().reshape(-1, 8, 64), k, v, lengths, meant, table, 16), "fp16", "starts that go down")
    assert torch.equal(y, kv4_attention(*args, _i32(meant, gpu), rows))


@pytest.mark.parametrize("start", [
    [2**31 - 1, 2**31 - 1, 2**31 - 1], [2**31 - 100, 2**31 - 1, 3], [9, 2**31 - 1, 2**31 - 500], [-2**31, -5, 2**31 - 1],
    [2**31 - 2, -2**31, 5]])
def test_bias_starts_outside_the_entries(gpu, start):
    """Only entries that there are count: 0 .. 8."""
    ids = torch.tensor([5, 5, 4, 99, 7, 5, 2, 9, 5], dtype=torch.int32)
    _check(gpu, torch.zeros((2, 100)), bias=(torch.tensor(start, dtype=torch.int32), ids, torch.arange(9, dtype=torch.float32) + 1))


@pytest.mark.parametrize("n", [511, 512, 513, 2000])
def test_many_biases_in_a_row(gpu, n):
    """More entries than a workgroup has threads, most tokens several times: the last one counts."""
    g = torch.Generator().manual_seed(n)
    start = torch.tensor([0, n, n + 3], dtype=torch.int32)
    ids = torch.randint(0, 300, (n + 3,), generator=g, dtype=torch.int32) * 17
    _check(gpu, torch.randn((2, 5100), generator=g).half(), bias=(start, ids, torch.randn(n + 3, generator=g) * 4))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("most", [1, 3, 40])
def test_rows_past_max_query_are_nan(gpu, most, dtype):
    """A bound that is too small: the rows within it are right, the others say that they are not."""
    rng = np.random.default_rng(most)
    requests = [(50, 45), (9, 1), (0, 60), (300, 41)]
    lengths, starts, table, pages = _batch(rng, requests, 16)
    cache, k, v = _cache(rng, pages, 16, 2, 64, 64, gpu)
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]), 4 * 64)).astype(np.float32)).to(DT[dtype])
    for _ in range(2):                                        # (memory that held a result before)
        y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), most)
    ref = O.attend(q.double().numpy().reshape(-1, 4, 64), k, v, lengths, starts, table, 16)
    for b, (n, m) in enumerate(requests):
        seen = m if n == 0 else min(m, most)                  # (rows of a request without tokens are zeros)
        lo = int(starts[b])
        _close(y[lo:lo + seen], ref[lo:lo + seen], dtype, f"request {b}")
        assert torch.isnan(y[lo + seen:lo + m]).all()


@pytest.mark.parametrize("rows", [1, 6, 75])
def test_only_rows_that_see_past_the_table_are_nan(gpu, rows):
    """Five pages of 16 tokens under a length of 82: the rows at 80 and 81."""
    rng = np.random.default_rng(rows)
    lengths, starts, table, pages = _batch(rng, [(80, rows)], 16, width=5)
    cache, k, v = _cache(rng, pages, 16, 2, 64, 64, gpu)
    q = torch.from_numpy(rng.standard_normal((rows, 4 * 64)).astype(np.float32)).half()
    y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32([82], gpu), _i32(starts, gpu), rows)
    past = min(rows, 2)
    assert torch.isnan(y[rows - past:]).all()
    seen = rows - past                                       # positions up to 79
    ref = O.attend(q[:seen].double().numpy().reshape(-1, 4, 64), k, v, lengths, [0, seen], table, 16)
    if seen:
        _close(y[:seen], ref, "fp16", "rows within the table")


@pytest.mark.parametrize("rows", [1, 70])
def test_queries_near_the_largest_bf16_under_a_large_scale(gpu, rows):
    """Finite scores of 1e37 and more: the largest takes all, none is NaN."""
    rng = np.random.default_rng(rows + 5)
    lengths, starts, table, pages = _batch(rng, [(100, rows)], 16)
    parts = [O.quantise((rng.standard_normal((pages * 16, 1, 64)) * gain).astype(np.float32), 64)[:3] for gain in (1e-4, 1.0)]
    k, v = (O.values(p, 64) for p in parts)
    cache = Kv4Cache.of(torch.from_numpy(O.pack(*parts, pages, 16, 64, 64)).to(gpu), 64, 16, 64)
    q = torch.from_numpy((rng.choice([-1.0, 1.0], (rows, 64)) * rng.uniform(1e38, 3.3e38, (rows, 64))).astype(np.float32)).bfloat16()
    y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), rows, scale=300.0)
    ref = O.attend(q.double().numpy().reshape(-1, 1, 64), k, v, lengths, starts, table, 16, 300.0)
    _close(y, ref, "bf16", "queries of 1e38")


def test_rows_past_max_query_of_one_prompt_are_nan(gpu):
    """The tile kernel by itself, which then fills them; rows of no request behind them."""
    rng = np.random.default_rng(17)
    lengths, starts, table, pages = _batch(rng, [(300, 90)], 16)
    cache, k, v = _cache(rng, pages, 16, 2, 64, 64, gpu)
    q = torch.from_numpy(rng.standard_normal((95, 8 * 64)).astype(np.float32)).half()
    y = kv4_attention(q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu), _i32(starts, gpu), 40)
    ref = O.attend(q.double().numpy().reshape(-1, 8, 64), k, v, lengths, starts, table, 16)
    _close(y[:40], ref[:40], "fp16", "rows within the bound")
    assert torch.isnan(y[40:90]).all() and (y[90:] == 0).all()
