"""Tables and caches whose parts were set after they were made: every call checks what it is
given, before anything else, so this needs no GPU."""
import pytest
import torch

from kernels.kv4 import Kv4Cache, kv4_append, kv4_attention, kv4_gather
from kernels.paged import PagedStep, PagedTables, paged_release, paged_step


def _i32(*n):
    return torch.zeros(n, dtype=torch.int32)


@pytest.mark.parametrize("name,value,says", [
    ("state", _i32(2), "state must be"), ("state", _i32(3).long(), "state must be"), ("state", _i32(6)[::2], "state must be"),
    ("block_tables", _i32(2, 6)[:, ::2], "block_tables must be"), ("block_tables", _i32(6), "block_tables must be"),
    ("block_tables", _i32(3, 3), "state must be"), ("free_pages", _i32(4).short(), "free_pages must be"),
    ("free_pages", _i32(2, 2), "free_pages"), ("page_size", 24, "page_size 24"), ("page_size", 2**20, "page_size")])
def test_tables(name, value, says):
    tables = PagedTables(2, 3, 4, 16, "cpu")
    setattr(tables, name, value)
    for call in (lambda: paged_step(tables, _i32(2), 2), lambda: paged_release(tables, _i32(2))):
        with pytest.raises(ValueError, match=says):
            call()


def test_a_step_of_another_type_is_not_committed():
    """Its state has the tables' shape: the next call refuses it."""
    tables = PagedTables(2, 3, 4, 16, "cpu")
    parts = vars(PagedStep.empty(2, 2, torch.device("cpu")))
    tables.commit(PagedStep(**{**parts, "state": parts["state"].float()}))
    with pytest.raises(ValueError, match="state must be"):
        paged_step(tables, _i32(2), 2)


@pytest.mark.parametrize("name,value,says", [
    ("data", torch.zeros((2, 2, 1264), dtype=torch.uint8), "data must be"), ("data", torch.zeros((2, 2, 1280)), "data must be"),
    ("data", torch.zeros((2, 2, 2560), dtype=torch.uint8)[:, :, ::2], "data must be"), ("head_dim", 128, "data must be"),
    ("data", torch.zeros(1280, dtype=torch.uint8), "data must be"), ("page_size", 32, "data must be"),
    ("group_size", 64, "data must be"), ("group_size", 48, "group_size 48"), ("head_dim", 0, "head_dim 0")])
def test_caches(name, value, says):
    cache = Kv4Cache(2, 2, 64, 16, 32, "cpu")
    assert cache.data.shape[2] == 1280
    setattr(cache, name, value)
    for call in (lambda: kv4_append(torch.zeros((1, 512)).half(), cache, _i32(1), _i32(1), None, None, 4),
                 lambda: kv4_gather(cache, _i32(1)),
                 lambda: kv4_attention(torch.zeros((1, 256)).half(), cache, _i32(1, 1), _i32(1), _i32(2), 1)):
        with pytest.raises(ValueError, match=says):
            call()
