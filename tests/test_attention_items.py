"""How ``kv4_attention`` cuts its work into items, on the host: the arithmetic that the
kernels, their grids and the workspace share (``csrc/awq_serve_items.h``), compiled into a
walk over a call's requests (``attention_items.cpp``).  Every item needs a workgroup
of its launch's grid (less one, which clears rows of no request), and an item that is one of
several of its request a place for its sums."""
import ctypes
import os
import random
import subprocess
from dataclasses import dataclass

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "qwen2-7b-triton_engine_amd", "csrc")


@dataclass
class Items:
    items: int
    grid: int
    splits: int        # the most of a request
    steps: int         # the most of an item
    wrong: int         # items that do not meet, or do not end where the tokens do


@pytest.fixture(scope="session")
def walk(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("items") / "libitems.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{CSRC}",
                    os.path.join(HERE, "attention_items.cpp"), "-o", lib], check=True)
    fn = ctypes.CDLL(lib).attention_items

    def run(requests, group, kvh, *, starts=None, total=None, max_query=None, width=None, page=64):
        """Items of [(length, rows)]; (decode's, tiles', whether tiles have places for sums)."""
        lens = [n for n, _ in requests]
        if starts is None:
            starts = [sum(m for _, m in requests[:b]) for b in range(len(requests) + 1)]
        total = max(0, max(starts)) if total is None else total
        max_query = max(1, max(m for _, m in requests)) if max_query is None else max_query
        width = -(-max(max(lens), 1) // page) if width is None else width
        out = (ctypes.c_longlong * 11)()
        ints = lambda v: (ctypes.c_int * len(v))(*v)  # noqa: E731
        fn(len(requests), ints(starts), ints(lens), total, max_query, group, kvh, width, page.bit_length() - 1, out)
        return Items(*out[:5]), Items(*out[5:10]), bool(out[10])

    return run


def _fits(decode, tiles, places):
    assert decode.wrong == tiles.wrong == 0
    for k in (decode, tiles):
        assert k.items <= max(0, k.grid - 1), k
    assert places or tiles.splits <= 1, tiles


@pytest.mark.parametrize("requests,group,kvh", [
    ([(2**29 + 4096, 4096)], 7, 4),              # a prompt behind 2^29 tokens: not split, one item a block
    ([(2**30, 4096)], 7, 4),
    ([(2**30, 1)], 7, 4),
    ([(2**30, 20)], 8, 1),
    ([(2**30, 1)] * 200, 8, 8),                  # more work than items of 2^29 tokens have room for
    ([(2**30 - 1, 1)] * 4096, 1, 768),
    ([(2**30, 40), (2**30, 3)] * 30, 8, 32),
    ([(2**29 + 65, 70), (1, 1), (2**29 + 1, 9)], 64, 1),
])
def test_lengths_up_to_the_limit(walk, requests, group, kvh):
    _fits(*walk(requests, group, kvh, page=256))


@pytest.mark.parametrize("starts,lens,total,group,kvh", [
    ([0, 32] * 32 + [64], [4096] * 64, 64, 4, 8),
    ([0, 16] * 32 + [16], [4096] * 64, 16, 8, 8),
    ([0, 400] * 100 + [0], [2000] * 200, 400, 4, 4),           # tiles
    ([9, 2, 30, -7, 2**31 - 1, 5, -2**31, 40, 12], [300] * 8, 33, 8, 2),
])
def test_starts_that_go_down(walk, starts, lens, total, group, kvh):
    """No row is two requests': a start below an earlier one counts as that one."""
    requests = list(zip(lens, [0] * len(lens)))
    max_query = min(total, max(max(0, b - a) for a, b in zip(starts, starts[1:])))
    _fits(*walk(requests, group, kvh, starts=starts, total=total, max_query=max_query))
    _fits(*walk(requests, group, kvh, starts=starts, total=total, max_query=1))


def test_many_shapes(walk):
    """Random batches: single tokens, chunks and prompts, empty requests, bounds that are too small."""
    rng = random.Random(0)
    for _ in range(300):
        n = rng.choice([1, 1, 2, 5, 64, 65, 300])
        longest = rng.choice([1, 100, 5000, 200000])
        most = rng.choice([1, 4, 60, 700])
        requests = [(rng.choice([0, rng.randint(1, longest)]), rng.choice([0, 1, 1, rng.randint(1, most)])) for _ in range(n)]
        total = sum(m for _, m in requests)
        kw = {"total": max(0, total + rng.choice([0, 0, 9, -3])), "page": rng.choice([16, 64, 256])}
        if rng.random() < 0.2:
            kw["max_query"] = rng.randint(1, most)
        if rng.random() < 0.2:
            kw["width"] = rng.randint(1, 20)
        _fits(*walk(requests, rng.choice([1, 4, 7, 8, 64]), rng.choice([1, 4, 8, 40]), **kw))
