"""The 16-bit cache and the log-probabilities without a GPU: which statuses the checks before any device work give, and
how attention cuts its work into items (``attention16_items.cpp``)."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from kernels import _native
from kernels.kv16 import Kv16Cache, kv16_append, kv16_attention
from kernels.logprobs import token_logprobs

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "qwen2-7b-triton_engine_amd", "csrc")


def _attention(**kw):
    """Arguments that pass every check but the workspace's size."""
    a = {"q": 16, "q_stride": 256, "cache": 16, "tables": 16, "lens": 16, "starts": 16, "slopes": 0, "prefix": 0, "first": 0,
         "out": 16, "requests": 1, "total": 1, "max_query": 1, "heads": 4, "kv_heads": 2, "hd": 64, "width": 1, "pages": 2,
         "page": 16, "window": 0, "scale": 0.1, "softcap": 0.0, "dtype": 0, "ws": 16, "ws_bytes": 0, "stream": 0}
    return _native.lib().awq_serve_kv16_attention(*{**a, **kw}.values())


@pytest.mark.parametrize("change,status", [
    ({}, _native.AWQ_ERR_WORKSPACE), ({"ws": 0}, _native.AWQ_ERR_WORKSPACE), ({"total": 0}, _native.AWQ_OK),
    *[({k: 0}, _native.AWQ_ERR_NULL_POINTER) for k in ("q", "cache", "tables", "lens", "starts", "out")],
    *[({k: 8}, _native.AWQ_ERR_MISALIGNED) for k in ("q", "cache", "out", "ws")],
    *[({k: 2}, _native.AWQ_ERR_MISALIGNED) for k in ("tables", "lens", "starts", "slopes", "prefix", "first")],
    ({"q_stride": 260}, _native.AWQ_ERR_MISALIGNED), ({"q_stride": 255}, _native.AWQ_ERR_BAD_DIMS),
    ({"heads": 3}, _native.AWQ_ERR_BAD_DIMS), ({"requests": 0}, _native.AWQ_ERR_BAD_DIMS), ({"pages": 0}, _native.AWQ_ERR_BAD_DIMS),
    ({"max_query": 0}, _native.AWQ_ERR_BAD_DIMS), ({"window": -1}, _native.AWQ_ERR_BAD_DIMS),
    *[({"scale": v}, _native.AWQ_ERR_BAD_DIMS) for v in (0.0, -1.0, float("nan"), float("inf"))],
    *[({"softcap": v}, _native.AWQ_ERR_BAD_DIMS) for v in (-1.0, 1e-38, float("nan"), float("inf"))],
    ({"hd": 96}, _native.AWQ_ERR_PATH), ({"page": 48}, _native.AWQ_ERR_PATH), ({"dtype": 2}, _native.AWQ_ERR_PATH),
    ({"heads": 256, "kv_heads": 2, "q_stride": 16384}, _native.AWQ_ERR_PATH),
    ({"requests": 4097}, _native.AWQ_ERR_TOO_LARGE), ({"pages": 2**31}, _native.AWQ_ERR_TOO_LARGE),
    ({"width": 2**27}, _native.AWQ_ERR_TOO_LARGE),
    # more workgroups than a launch holds
    ({"heads": 4096, "kv_heads": 4096, "q_stride": 4096 * 64, "total": 2**19 - 1, "max_query": 2**19 - 1}, _native.AWQ_ERR_TOO_LARGE),
])
def test_attention_statuses(change, status):
    assert _attention(**change) == status


def test_workspaces():
    L = _native.lib()
    assert L.awq_serve_kv16_attention_workspace(1, 1, 1, 4, 2, 64, 1, 16) > 0
    assert L.awq_serve_kv16_attention_workspace(1, 1, 1, 4, 2, 96, 1, 16) == 0
    assert L.awq_serve_kv16_attention_workspace(1, 2**19 - 1, 2**19 - 1, 4096, 4096, 64, 1, 16) == 0
    assert L.awq_serve_logprobs_workspace(3, 1000) > 0
    assert L.awq_serve_logprobs_workspace(2**24, 2**24) == 0 and L.awq_serve_logprobs_workspace(-1, 5) == 0


def _append(**kw):
    a = {"qkv": 16, "stride": 512, "cache": 16, "slots": 16, "positions": 16, "cos": 16, "sin": 16, "q": 16, "tokens": 1, "heads": 4,
         "kv_heads": 2, "hd": 64, "pages": 2, "page": 16, "max_pos": 9, "dtype": 0, "stream": 0}
    return _native.lib().awq_serve_kv16_append(*{**a, **kw}.values())


@pytest.mark.parametrize("change,status", [
    ({"tokens": 0}, _native.AWQ_OK), ({"cos": 0}, _native.AWQ_ERR_NULL_POINTER), ({"qkv": 0}, _native.AWQ_ERR_NULL_POINTER),
    ({"q": 0}, _native.AWQ_ERR_NULL_POINTER), ({"cache": 8}, _native.AWQ_ERR_MISALIGNED), ({"stride": 516}, _native.AWQ_ERR_MISALIGNED),
    ({"stride": 504}, _native.AWQ_ERR_BAD_DIMS), ({"tokens": -1}, _native.AWQ_ERR_BAD_DIMS), ({"heads": 0}, _native.AWQ_ERR_BAD_DIMS),
    ({"max_pos": 0}, _native.AWQ_ERR_BAD_DIMS), ({"hd": 32}, _native.AWQ_ERR_PATH), ({"dtype": 2}, _native.AWQ_ERR_PATH),
    ({"tokens": 2**31}, _native.AWQ_ERR_TOO_LARGE), ({"pages": 2**30}, _native.AWQ_ERR_TOO_LARGE)])
def test_append_statuses(change, status):
    assert _append(**change) == status


def _logprobs(**kw):
    a = {"hidden": 16, "stride": 64, "weight": 16, "targets": 16, "bytes": 8, "logprobs": 16, "lse": 16, "tokens": 1, "vocab": 5,
         "k": 64, "dtype": 0, "ws": 16, "ws_bytes": 0, "stream": 0}
    return _native.lib().awq_serve_logprobs(*{**a, **kw}.values())


@pytest.mark.parametrize("change,status", [
    ({}, _native.AWQ_ERR_WORKSPACE), ({"tokens": 0}, _native.AWQ_OK),
    *[({k: 0}, _native.AWQ_ERR_NULL_POINTER) for k in ("hidden", "weight", "targets", "logprobs", "lse")],
    *[({k: 8}, _native.AWQ_ERR_MISALIGNED) for k in ("hidden", "weight")], ({"targets": 4}, _native.AWQ_ERR_MISALIGNED),
    ({"stride": 68}, _native.AWQ_ERR_MISALIGNED), ({"ws": 4}, _native.AWQ_ERR_MISALIGNED),
    ({"k": 96}, _native.AWQ_ERR_BAD_DIMS), ({"stride": 56}, _native.AWQ_ERR_BAD_DIMS), ({"vocab": 0}, _native.AWQ_ERR_BAD_DIMS),
    ({"tokens": -1}, _native.AWQ_ERR_BAD_DIMS), ({"bytes": 2}, _native.AWQ_ERR_PATH), ({"dtype": 2}, _native.AWQ_ERR_PATH),
    ({"k": 2**21, "stride": 2**21}, _native.AWQ_ERR_TOO_LARGE), ({"stride": 2**23}, _native.AWQ_ERR_TOO_LARGE),
    ({"vocab": 2**25}, _native.AWQ_ERR_TOO_LARGE), ({"tokens": 2**24, "vocab": 2**24}, _native.AWQ_ERR_TOO_LARGE)])
def test_logprobs_statuses(change, status):
    assert _logprobs(**change) == status


def test_tensors_on_the_host_are_refused():
    cache = Kv16Cache(2, 2, 64, 16, device="cpu")
    assert cache.k.shape == cache.v.shape == (2, 2, 16, 64) and cache.num_pages == 2 and cache.head_dim == 64
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        kv16_append(torch.zeros((1, 512), dtype=torch.float16), cache, i, i, None, None, 4)
    with pytest.raises(ValueError):
        kv16_attention(torch.zeros((1, 256), dtype=torch.float16), cache, i[None], i, torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros((1, 64), dtype=torch.float16), torch.zeros((3, 64), dtype=torch.float16), i)
    for bad in (dict(head_dim=32), dict(page_size=24), dict(dtype=torch.float32), dict(num_pages=0)):
        with pytest.raises(ValueError):
            Kv16Cache(**{**dict(num_pages=2, num_kv_heads=2, head_dim=64, page_size=16, device="cpu"), **bad})


@pytest.fixture(scope="session")
def walk(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("items16") / "libitems16.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{CSRC}",
                    os.path.join(HERE, "attention16_items.cpp"), "-o", lib], check=True)
    fn = ctypes.CDLL(lib).attention16_items

    def run(requests, group, kvh, *, window=0, total=None, max_query=None, width=None, page=64):
        """[(length, rows)]: every item has a workgroup of its grid less one, and several of a request places for sums."""
        lens = [n for n, _ in requests]
        starts = [sum(m for _, m in requests[:b]) for b in range(len(requests) + 1)]
        total = starts[-1] if total is None else total
        max_query = max(1, max(m for _, m in requests)) if max_query is None else max_query
        width = -(-max(max(lens), 1) // page) if width is None else width
        out = (ctypes.c_longlong * 9)()
        ints = lambda v: (ctypes.c_int * len(v))(*v)  # noqa: E731
        fn(len(requests), ints(starts), ints(lens), total, max_query, group, kvh, width, page.bit_length() - 1, window, out)
        for items, grid, _, wrong in (out[:4], out[4:8]):
            assert wrong == 0 and items <= max(0, grid - 1), list(out)
        assert out[8] or out[6] <= 1
        return list(out)

    return run


@pytest.mark.parametrize("window", [0, 1, 100, 4096, 2**31 - 2])
@pytest.mark.parametrize("requests,group,kvh", [
    ([(2**30, 1)], 7, 4), ([(2**30, 4096)], 7, 4), ([(2**31 - 1, 1)], 8, 8), ([(2**30 - 1, 1)] * 4096, 1, 768),
    ([(2**29 + 65, 70), (1, 1), (2**29 + 1, 9), (3, 5)], 64, 1), ([(1, 1)], 1, 1), ([(0, 0), (0, 3)], 4, 2)])
def test_items_under_windows(walk, requests, group, kvh, window):
    walk(requests, group, kvh, window=window, page=256, width=min(2**22, -(-max(n for n, _ in requests) // 256) or 1))


def test_items_of_many_shapes(walk):
    rng = random.Random(1)
    for _ in range(400):
        longest, most = rng.choice([1, 100, 5000, 200000]), rng.choice([1, 4, 60, 700])
        requests = [(rng.choice([0, rng.randint(1, longest)]), rng.choice([0, 1, 1, rng.randint(1, most)]))
                    for _ in range(rng.choice([1, 1, 2, 5, 64, 65, 300]))]
        kw = {"total": max(0, sum(m for _, m in requests) + rng.choice([0, 0, 9, -3])), "page": rng.choice([16, 64, 256]),
              "window": rng.choice([0, rng.randint(1, longest + 5)])}
        if rng.random() < 0.2:
            kw["max_query"] = rng.randint(1, most)
        if rng.random() < 0.2:
            kw["width"] = rng.randint(1, 20)
        walk(requests, rng.choice([1, 4, 7, 8, 64]), rng.choice([1, 4, 8, 40]), **kw)
