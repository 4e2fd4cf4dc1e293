"""The serving operators without a GPU: the library exports what
include/awq_serving.h declares, and the checks that come before any device work."""
import os
import re

import pytest
import torch

from kernels import _native
from kernels.kv4 import Kv4Cache, kv4_append, kv4_attention, kv4_gather
from kernels.logits import process_logits
from kernels.paged import PagedTables, paged_release, paged_step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _header():
    return open(os.path.join(ROOT, "include", "awq_serving.h")).read()


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", _header(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(awq_serve_[a-z0-9_]+)\s*\(", text)))
    assert declared == sorted(_native.SERVING_SIGNATURES)
    for name in declared:
        assert hasattr(_native.lib(), name)
        arguments = re.search(name + r"\s*\(([^)]*)\)", text).group(1).count(",") + 1
        assert len(_native.SERVING_SIGNATURES[name][1]) == arguments, name


def test_constants_match_the_header():
    text = _header()
    for name, value in (("FP16", _native.SERVE_FP16), ("BF16", _native.SERVE_BF16), ("FP32", _native.SERVE_FP32),
                        ("MAX_REQUESTS", _native.SERVE_MAX_REQUESTS), ("MAX_GROUP", _native.SERVE_MAX_GROUP)):
        assert int(re.search(rf"#define AWQ_SERVE_{name} (\d+)", text).group(1)) == value


def _attention(**kw):
    """Arguments of awq_serve_kv4_attention that pass every check but the null pointers."""
    a = {"q": 16, "q_stride": 256, "cache": 16, "tables": 16, "lens": 16, "starts": 16, "out": 16, "requests": 1,
         "total": 1, "max_query": 1, "heads": 4, "kv_heads": 2, "hd": 64, "width": 1, "pages": 2, "page": 16,
         "group": 64, "scale": 0.1, "dtype": 0, "ws": 16, "ws_bytes": 0, "stream": 0}
    return _native.lib().awq_serve_kv4_attention(*{**a, **kw}.values())


@pytest.mark.parametrize("change,status", [
    ({"q": 0}, _native.AWQ_ERR_NULL_POINTER), ({"out": 0}, _native.AWQ_ERR_NULL_POINTER),
    ({"q": 8}, _native.AWQ_ERR_MISALIGNED), ({"q_stride": 260}, _native.AWQ_ERR_MISALIGNED),
    ({"q_stride": 255}, _native.AWQ_ERR_BAD_DIMS), ({"heads": 3}, _native.AWQ_ERR_BAD_DIMS),
    ({"scale": 0.0}, _native.AWQ_ERR_BAD_DIMS), ({"scale": float("nan")}, _native.AWQ_ERR_BAD_DIMS),
    ({"scale": float("inf")}, _native.AWQ_ERR_BAD_DIMS), ({"requests": 0}, _native.AWQ_ERR_BAD_DIMS),
    ({"max_query": 0}, _native.AWQ_ERR_BAD_DIMS), ({"hd": 96}, _native.AWQ_ERR_PATH), ({"page": 24}, _native.AWQ_ERR_PATH),
    ({"page": 8}, _native.AWQ_ERR_PATH), ({"dtype": 2}, _native.AWQ_ERR_PATH), ({"heads": 130, "q_stride": 8320}, _native.AWQ_ERR_PATH),
    ({"group": 128}, _native.AWQ_ERR_GROUP_SIZE), ({"group": 16}, _native.AWQ_ERR_GROUP_SIZE),
    ({"requests": 4097}, _native.AWQ_ERR_TOO_LARGE), ({"pages": 2**31}, _native.AWQ_ERR_TOO_LARGE),
    ({"width": 2**28}, _native.AWQ_ERR_TOO_LARGE), ({}, _native.AWQ_ERR_WORKSPACE), ({"total": 0}, _native.AWQ_OK)])
def test_attention_statuses(change, status):
    assert _attention(**change) == status


def test_other_statuses():
    L = _native.lib()
    step = lambda **kw: L.awq_serve_page_step(*{**dict(zip("abcdefghi", [16] * 9)), "B": 2, "T": 3, "W": 4, "N": 5,  # noqa: E731
                                                "P": 16, "s": 0, **kw}.values())
    assert step(a=0) == step(i=0) == _native.AWQ_ERR_NULL_POINTER and step(B=0) == step(T=-1) == _native.AWQ_ERR_BAD_DIMS
    assert step(P=20) == step(P=512) == _native.AWQ_ERR_PATH and step(B=4097) == step(N=2**28) == _native.AWQ_ERR_TOO_LARGE
    assert step(g=18) == _native.AWQ_ERR_MISALIGNED
    append = lambda **kw: L.awq_serve_kv4_append(*{  # noqa: E731
        "qkv": 16, "ld": 512, "cache": 16, "slots": 16, "pos": 16, "cos": 16, "sin": 16, "q": 16, "T": 1, "nh": 4, "kvh": 2,
        "hd": 64, "pages": 2, "page": 16, "group": 64, "max_pos": 9, "dtype": 0, "s": 0, **kw}.values())
    assert append(sin=0) == append(q=0) == _native.AWQ_ERR_NULL_POINTER and append(T=0) == _native.AWQ_OK
    assert append(ld=511) == append(max_pos=0) == _native.AWQ_ERR_BAD_DIMS and append(ld=513) == _native.AWQ_ERR_MISALIGNED
    assert append(hd=32) == _native.AWQ_ERR_PATH and append(T=2**30) == _native.AWQ_ERR_TOO_LARGE
    gather = lambda **kw: L.awq_serve_kv4_gather(*{  # noqa: E731
        "c": 16, "slots": 16, "k": 16, "v": 16, "T": 1, "kvh": 2, "hd": 64, "pages": 2, "page": 16, "group": 64, "dt": 1,
        "s": 0, **kw}.values())
    assert gather(k=0) == _native.AWQ_ERR_NULL_POINTER and gather(T=0) == _native.AWQ_OK
    assert gather(v=8) == _native.AWQ_ERR_MISALIGNED and gather(dt=2) == _native.AWQ_ERR_PATH
    logits = lambda **kw: L.awq_serve_logits(*{  # noqa: E731
        "x": 16, "ld": 100, "out": 16, "next": 16, "B": 2, "V": 100, "dt": 0, "tokens": 0, "size": 8, "L": 0, "len": 0,
        "prompt": 0, "rep": 0, "pres": 0, "freq": 0, "start": 0, "ids": 0, "values": 0, "n": 0, "mask": 0, "ws": 16,
        "bytes": 0, "s": 0, **kw}.values())
    assert logits(x=0) == logits(tokens=16) == logits(rep=16) == logits(start=16) == _native.AWQ_ERR_NULL_POINTER
    assert logits(V=0) == logits(ld=99) == _native.AWQ_ERR_BAD_DIMS and logits(dt=3) == _native.AWQ_ERR_PATH
    assert logits(B=65536) == _native.AWQ_ERR_TOO_LARGE and logits(x=17) == _native.AWQ_ERR_MISALIGNED
    assert logits() == _native.AWQ_ERR_WORKSPACE and logits(B=0) == _native.AWQ_OK
    assert L.awq_serve_kv4_attention_workspace(1, 1, 1, 4, 2, 96, 1, 16) == 0 and L.awq_serve_logits_workspace(0, 5) == 0


def test_tensors_on_the_host_are_refused():
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    tables = PagedTables(2, 3, 4, 16, "cpu")
    assert tables.lengths.tolist() == [0, 0] and tables.free_count.tolist() == [4]
    cache = Kv4Cache(2, 2, 64, 16, 32, "cpu")
    assert cache.data.shape == (2, 2, 16 * (64 + 16)) and cache.num_pages == 2 and cache.num_kv_heads == 2
    for bad in (lambda: paged_step(tables, i32(2), 2), lambda: paged_release(tables, i32(2)),
                lambda: kv4_append(torch.zeros((1, 512)).half(), cache, i32(1), i32(1), None, None, 4),
                lambda: kv4_gather(cache, i32(1)), lambda: process_logits(torch.zeros((1, 8))),
                lambda: kv4_attention(torch.zeros((1, 256)).half(), cache, i32(1, 1), i32(1), i32(2), 1),
                lambda: Kv4Cache(2, 2, 96, 16, 32, "cpu"), lambda: Kv4Cache(2, 2, 64, 16, 128, "cpu"),
                lambda: Kv4Cache.of(cache.data[:, :, :-4], 64, 16, 32), lambda: Kv4Cache.of(cache.data, 64, 32, 32)):
        with pytest.raises(ValueError):
            bad()
