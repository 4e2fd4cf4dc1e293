"""A KV cache of 16-bit values, in pages that many requests share, and the attention
over it (``awq_serve_kv16_append``, ``_attention``; ``include/awq_serving.h``).

The cache of ``kernels.kv4`` quantises; this one holds what the projection gave, at
3.6 times the bytes for heads of 128 in groups of 64.  ``kv16_append`` takes the rows of a fused QKV projection:
RoPE of q and k (``kernels/rope.py:41-57``), k and v stored by a step's slots
(``kernels.paged``).  ``kv16_attention`` is softmax(score) V for all rows of a batch, one token of
each request or chunks of prompts (``model/qwen2.py:104-163``), and serves scores that the
reference's model has no use for: capped by a tanh, with a bias for the distance; and rows that see a
sliding window, a document of a packed text, or a prefix as a whole.  Neither is differentiable: results
carry no gradient.
"""
from __future__ import annotations

import torch

from . import _native

__all__ = ["Kv16Cache", "kv16_append", "kv16_attention", "HEAD_DIMS", "PAGE_SIZES"]

HEAD_DIMS = (64, 128)
PAGE_SIZES = (16, 32, 64, 128, 256)


class Kv16Cache:
    """One layer's cache: ``data`` fp16 or bf16 ``[num_pages, num_kv_heads, 2, page_size, head_dim]``, K and V
    of a page and head; ``k`` and ``v`` are views of it, slot s is token ``s % page_size`` of page ``s // page_size``."""

    __slots__ = ("data",)

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float16, device: torch.device | str = "cuda:0"):
        self._set(torch.zeros((num_pages, num_kv_heads, 2, page_size, head_dim), dtype=dtype, device=device))

    @classmethod
    def of(cls, data: torch.Tensor) -> "Kv16Cache":
        """A cache over a tensor that exists (a layer's part of a larger one, say)."""
        cache = cls.__new__(cls)
        cache._set(data)
        return cache

    def _set(self, data):
        _native.binding().check_cache16(data)
        self.data = data

    @staticmethod
    def block_bytes(head_dim: int, page_size: int) -> int:
        """Bytes of one page of one kv head, k and v."""
        return 4 * page_size * head_dim

    @property
    def num_pages(self) -> int:
        return self.data.shape[0]

    @property
    def num_kv_heads(self) -> int:
        return self.data.shape[1]

    @property
    def page_size(self) -> int:
        return self.data.shape[3]

    @property
    def head_dim(self) -> int:
        return self.data.shape[4]

    @property
    def k(self) -> torch.Tensor:
        return self.data[:, :, 0]

    @property
    def v(self) -> torch.Tensor:
        return self.data[:, :, 1]


def kv16_append(qkv: torch.Tensor, cache: Kv16Cache, slots: torch.Tensor, positions: torch.Tensor,
                cos: torch.Tensor | None, sin: torch.Tensor | None, num_heads: int) -> torch.Tensor:
    """q after RoPE, ``[T, num_heads * head_dim]``, of the rows ``qkv`` ``[T, (num_heads + 2 kv heads) * head_dim]`` (the
    cache's type, any row stride); their k (after RoPE) and v go into the cache's ``slots`` (int32 ``[T]``; one outside
    the cache, -1 say: not stored; a slot that two rows have holds a mixture of theirs).  ``cos`` / ``sin`` fp32
    ``[max_pos, head_dim]`` at ``positions`` (int32 ``[T]``; one outside: q NaN, nothing stored), both None: no
    rotation.  RoPE is computed in fp32 and rounded once (past 65504, fp16 gives an infinity)."""
    return _native.binding().kv16_append(qkv, cache.data, slots, positions, cos, sin, num_heads)


def kv16_attention(q: torch.Tensor, cache: Kv16Cache, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                   query_start: torch.Tensor, max_query: int, scale: float | None = None, *, softcap: float | None = None,
                   slopes: torch.Tensor | None = None, window: int | None = None, prefix: torch.Tensor | None = None,
                   first: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(score) V, ``[T, num_heads * head_dim]`` in q's type, the cache's.

    ``q`` ``[T, num_heads * head_dim]`` (any row stride), ``block_tables`` int32 ``[requests, width]``, ``seq_lens``
    int32 ``[requests]`` the tokens of each request with its rows among them, ``query_start`` int32
    ``[requests + 1]`` its first row (an entry below an earlier one counts as that one), ``max_query`` at least the most
    rows of a request (rows past it are NaN).  The i-th of a request's n rows stands at position p =
    ``seq_lens - n + i``.  Its score with token j is ``scale`` q.k (1 / sqrt(head_dim) unless given), then
    ``softcap * tanh(x / softcap)``, then ``x - slopes[head] * |p - j|`` (fp32 ``[num_heads]``).  It sees the tokens
    j <= p, with ``prefix`` (int32 ``[requests]``) also those j < prefix of its request; of these only j > p -
    ``window``, and j >= ``first`` (int32 ``[T]``: where the row's document begins, say).

    A row that sees no token, and a row of no request, gives zeros; one that sees a page outside the cache or a token
    past the table NaN; one that sees a key of NaN or a value that is not finite is not finite, in the columns that the
    arithmetic says or in all; so is one whose scores before the distance's part pass 2^127 (fp32 holds them) where ``slopes``
    are given without a cap.  What a row does not see may hold anything.

    Scores and sums are fp32; of requests with many rows each probability is rounded to the cache's type before its product
    with V (half a step, as the result's own rounding), of the others it is held in two such parts."""
    return _native.binding().kv16_attention(q, cache.data, block_tables, seq_lens, query_start, max_query, scale, softcap, slopes,
                                            window, prefix, first)
