"""A KV cache held in 4 bits, in pages that many requests share, and the
attention over it (``awq_serve_kv4_append``, ``_gather``, ``_attention``; the
format is written out in ``include/awq_serving.h``).

``kv4_append`` takes the rows of a fused QKV projection: RoPE of q and k
(``kernels/rope.py:41-57``), k and v quantised by groups of columns and stored by a
step's slots (``kernels.paged``).  ``kv4_attention`` is softmax(scale q K^T) V for all
rows of a batch, one token of each request or chunks of prompts, each row seeing
the tokens up to its own position (``model/qwen2.py:104-163``).  A token takes
``head_dim + 8 head_dim / group_size`` bytes for k and v of a head: 144 instead of
512 for heads of 128 in groups of 64.  Attention adds no rounding to the cache's
values: scores, softmax and sums are fp32, the values exact, q held to 2^-32 of its
row's largest value, the probabilities to 23 bits.
"""
from __future__ import annotations

import torch

from . import _native

__all__ = ["Kv4Cache", "kv4_append", "kv4_gather", "kv4_attention", "GROUP_SIZES", "HEAD_DIMS", "PAGE_SIZES"]

GROUP_SIZES = (32, 64, 128)
HEAD_DIMS = (64, 128)
PAGE_SIZES = (16, 32, 64, 128, 256)


class Kv4Cache:
    """One layer's cache: ``data`` uint8 ``[num_pages, num_kv_heads, block_bytes]``."""

    __slots__ = ("data", "head_dim", "page_size", "group_size")

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, group_size: int = 64,
                 device: torch.device | str = "cuda:0"):
        if group_size not in GROUP_SIZES:
            raise ValueError(f"group_size {group_size} must be one of {GROUP_SIZES}")
        data = torch.zeros((num_pages, num_kv_heads, self.block_bytes(head_dim, page_size, group_size)),
                           dtype=torch.uint8, device=device)
        self._set(data, head_dim, page_size, group_size)

    @classmethod
    def of(cls, data: torch.Tensor, head_dim: int, page_size: int = 64, group_size: int = 64) -> "Kv4Cache":
        """A cache over a tensor that exists (a layer's part of a larger one, say)."""
        cache = cls.__new__(cls)
        cache._set(data, head_dim, page_size, group_size)
        return cache

    def _set(self, data, head_dim, page_size, group_size):
        _native.binding().check_cache(data, head_dim, page_size, group_size)
        self.data, self.head_dim, self.page_size, self.group_size = data, head_dim, page_size, group_size

    @staticmethod
    def block_bytes(head_dim: int, page_size: int, group_size: int) -> int:
        """Bytes of one page of one kv head, k and v."""
        return page_size * (head_dim + 8 * (head_dim // group_size))

    @property
    def num_pages(self) -> int:
        return self.data.shape[0]

    @property
    def num_kv_heads(self) -> int:
        return self.data.shape[1]


def kv4_append(qkv: torch.Tensor, cache: Kv4Cache, slots: torch.Tensor, positions: torch.Tensor,
               cos: torch.Tensor | None, sin: torch.Tensor | None, num_heads: int) -> torch.Tensor:
    """q after RoPE, ``[T, num_heads * head_dim]`` in ``qkv``'s type, of the rows ``qkv``
    fp16 or bf16 ``[T, (num_heads + 2 kv heads) * head_dim]`` (any row stride); their k
    (after RoPE) and v go into the cache's ``slots`` (int32 ``[T]``; one outside the cache,
    -1 say: not stored; a slot that two rows have holds a mixture of theirs).  ``cos`` / ``sin`` fp32 ``[max_pos, head_dim]`` at ``positions`` (int32
    ``[T]``; one outside: q NaN, nothing stored), both None: no rotation.  A token
    whose k or v of a head is not finite is stored so that every query that sees
    it gives NaN."""
    return _native.binding().kv4_append(qkv, cache.data, cache.head_dim, cache.page_size, cache.group_size, slots, positions,
                                        cos, sin, num_heads)


def kv4_gather(cache: Kv4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
    """``(k, v)`` ``[T, kv heads, head_dim]`` in fp16 or bf16: the values that the cache
    holds in ``slots`` (int32 ``[T]``), rounded once; NaN for a slot outside."""
    return _native.binding().kv4_gather(cache.data, cache.head_dim, cache.page_size, cache.group_size, slots, dtype)


def kv4_attention(q: torch.Tensor, cache: Kv4Cache, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  query_start: torch.Tensor, max_query: int, scale: float | None = None) -> torch.Tensor:
    """softmax(scale q K^T) V, ``[T, num_heads * head_dim]`` in q's type.

    ``q`` fp16 or bf16 ``[T, num_heads * head_dim]`` (any row stride), ``block_tables`` int32
    ``[requests, width]``, ``seq_lens`` int32 ``[requests]`` the tokens of each request with
    its rows among them, ``query_start`` int32 ``[requests + 1]`` its first row (an entry below
    an earlier one counts as that one), ``max_query``
    at least the most rows of a request (rows past it are NaN).  The i-th
    of a request's n rows stands at position ``seq_lens - n + i`` and sees the tokens up to
    it; a row before the first token, and a row of no request, gives zeros.
    ``scale``: 1 / sqrt(head_dim) unless given.  A row that sees a token in a page outside the
    cache, or past the table, gives NaN."""
    return _native.binding().kv4_attention(q, cache.data, cache.head_dim, cache.page_size, cache.group_size, block_tables,
                                           seq_lens, query_start, max_query, scale)
