"""``Kv16Cache`` without a GPU: its sizes."""
import pytest
import torch

from kernels.kv16 import HEAD_DIMS, PAGE_SIZES, Kv16Cache


@pytest.mark.parametrize("head_dim", HEAD_DIMS)
@pytest.mark.parametrize("page_size", PAGE_SIZES)
def test_block_bytes(head_dim, page_size):
    """What a program reckons its pages with is what the cache takes."""
    for dtype in (torch.float16, torch.bfloat16):
        cache = Kv16Cache(3, 2, head_dim, page_size, dtype, device="cpu")
        assert cache.data.nbytes == 3 * 2 * Kv16Cache.block_bytes(head_dim, page_size)
