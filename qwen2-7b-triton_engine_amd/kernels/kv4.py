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
values: scores, softmax and sums are fp32, q and the values exact, the
probabilities held to 23 bits.
"""
from __future__ import annotations

import math

import torch

from . import _native
from .awq_gemm import _OnDevice, _aligned16, _stream_handle

__all__ = ["Kv4Cache", "kv4_append", "kv4_gather", "kv4_attention", "GROUP_SIZES", "HEAD_DIMS"]

GROUP_SIZES = (32, 64, 128)
HEAD_DIMS = (64, 128)
_PAGE_SIZES = (16, 32, 64, 128, 256)
_DTYPES = {torch.float16: _native.SERVE_FP16, torch.bfloat16: _native.SERVE_BF16}


class Kv4Cache:
    """One layer's cache: ``data`` uint8 ``[num_pages, num_kv_heads, block_bytes]``."""

    __slots__ = ("data", "head_dim", "page_size", "group_size")

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, group_size: int = 64,
                 device: torch.device | str = "cuda:0"):
        self._check(head_dim, page_size, group_size)
        data = torch.zeros((num_pages, num_kv_heads, self.block_bytes(head_dim, page_size, group_size)),
                           dtype=torch.uint8, device=device)
        self._set(data, head_dim, page_size, group_size)

    @classmethod
    def of(cls, data: torch.Tensor, head_dim: int, page_size: int = 64, group_size: int = 64) -> "Kv4Cache":
        """A cache over a tensor that exists (a layer's part of a larger one, say)."""
        cls._check(head_dim, page_size, group_size)
        cache = cls.__new__(cls)
        cache._set(data, head_dim, page_size, group_size)
        return cache

    @staticmethod
    def _check(head_dim, page_size, group_size):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim {head_dim} must be one of {HEAD_DIMS}")
        if page_size not in _PAGE_SIZES:
            raise ValueError(f"page_size {page_size} must be one of {_PAGE_SIZES}")
        if group_size not in GROUP_SIZES or group_size > head_dim:
            raise ValueError(f"group_size {group_size} must be one of {GROUP_SIZES} and at most head_dim {head_dim}")

    def _set(self, data, head_dim, page_size, group_size):
        block = self.block_bytes(head_dim, page_size, group_size)
        if data.dtype is not torch.uint8 or data.dim() != 3 or data.shape[2] != block or not data.is_contiguous():
            raise ValueError(f"data must be a contiguous uint8 tensor [pages, kv heads, {block}], got {data.dtype} "
                             f"{tuple(data.shape)}")
        if data.shape[0] < 1 or data.shape[1] < 1 or data.data_ptr() % 16 != 0:
            raise ValueError("data must hold a page and a head and start on 16 bytes")
        if data.shape[0] > (2**31 - 1) // page_size:
            raise ValueError("slot numbers pass 32 bits")
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


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``t`` [rows, columns] itself where its rows are dense and start on 16 bytes, else a copy."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return _aligned16(t.contiguous())


def _check_index(t: torch.Tensor, what: str, n: int, dev: torch.device) -> None:
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{what} must be a contiguous int32 tensor {(n,)} on {dev}")


def kv4_append(qkv: torch.Tensor, cache: Kv4Cache, slots: torch.Tensor, positions: torch.Tensor,
               cos: torch.Tensor | None, sin: torch.Tensor | None, num_heads: int) -> torch.Tensor:
    """q after RoPE, ``[T, num_heads * head_dim]`` in ``qkv``'s type, of the rows ``qkv``
    fp16 or bf16 ``[T, (num_heads + 2 kv heads) * head_dim]`` (any row stride); their k
    (after RoPE) and v go into the cache's ``slots`` (int32 ``[T]``; one outside the cache,
    -1 say: not stored).  ``cos`` / ``sin`` fp32 ``[max_pos, head_dim]`` at ``positions`` (int32
    ``[T]``; one outside: q NaN, nothing stored), both None: no rotation.  A token
    whose k or v of a head is not finite is stored so that every query that sees
    it gives NaN."""
    dev, hd, kvh = qkv.device, cache.head_dim, cache.num_kv_heads
    if qkv.dtype not in _DTYPES or qkv.dim() != 2 or qkv.shape[1] != (num_heads + 2 * kvh) * hd or num_heads < 1:
        raise ValueError(f"qkv must be an fp16 or bf16 tensor [T, {(num_heads + 2 * kvh) * hd}], got {qkv.dtype} "
                         f"{tuple(qkv.shape)}")
    if dev.type != "cuda" or cache.data.device != dev:
        raise ValueError(f"qkv and the cache must be on one ROCm device, got {dev} and {cache.data.device}")
    T = qkv.shape[0]
    _check_index(slots, "slots", T, dev)
    _check_index(positions, "positions", T, dev)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    max_pos = 2**31 - 1
    if cos is not None:
        max_pos = cos.shape[0]
        for t, what in ((cos, "cos"), (sin, "sin")):
            if t.dtype is not torch.float32 or t.shape != (max_pos, hd) or not t.is_contiguous() or t.device != dev \
                    or max_pos < 1:
                raise ValueError(f"{what} must be a contiguous float32 tensor [max_pos, {hd}] on {dev}")
        cos, sin = _aligned16(cos), _aligned16(sin)
    qkv = _rows16(qkv)
    q = torch.empty((T, num_heads * hd), dtype=qkv.dtype, device=dev)
    with _OnDevice(dev):
        st = _native.lib().awq_serve_kv4_append(
            qkv.data_ptr(), qkv.stride(0) if T > 1 else qkv.shape[1], cache.data.data_ptr(), slots.data_ptr(),
            positions.data_ptr(), 0 if cos is None else cos.data_ptr(), 0 if sin is None else sin.data_ptr(),
            q.data_ptr(), T, num_heads, kvh, hd, cache.num_pages, cache.page_size, cache.group_size, max_pos,
            _DTYPES[qkv.dtype], _stream_handle(dev))
    _native.check(st, "awq_serve_kv4_append")
    return q


def kv4_gather(cache: Kv4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
    """``(k, v)`` ``[T, kv heads, head_dim]`` in fp16 or bf16: the values that the cache
    holds in ``slots`` (int32 ``[T]``), rounded once; NaN for a slot outside."""
    dev = cache.data.device
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
    if dev.type != "cuda" or slots.dim() != 1:
        raise ValueError("the cache must be on a ROCm device and slots 1-D")
    T = slots.shape[0]
    _check_index(slots, "slots", T, dev)
    k, v = torch.empty((2, T, cache.num_kv_heads, cache.head_dim), dtype=dtype, device=dev)
    with _OnDevice(dev):
        st = _native.lib().awq_serve_kv4_gather(
            cache.data.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), T, cache.num_kv_heads, cache.head_dim,
            cache.num_pages, cache.page_size, cache.group_size, _DTYPES[dtype], _stream_handle(dev))
    _native.check(st, "awq_serve_kv4_gather")
    return k, v


def kv4_attention(q: torch.Tensor, cache: Kv4Cache, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  query_start: torch.Tensor, max_query: int, scale: float | None = None) -> torch.Tensor:
    """softmax(scale q K^T) V, ``[T, num_heads * head_dim]`` in q's type.

    ``q`` fp16 or bf16 ``[T, num_heads * head_dim]`` (any row stride), ``block_tables`` int32
    ``[requests, width]``, ``seq_lens`` int32 ``[requests]`` the tokens of each request with
    its rows among them, ``query_start`` int32 ``[requests + 1]`` its first row, ``max_query``
    at least the most rows of a request (rows past it are not computed).  The i-th
    of a request's n rows stands at position ``seq_lens - n + i`` and sees the tokens up to
    it; a row before the first token, and a row of no request, gives zeros.
    ``scale``: 1 / sqrt(head_dim) unless given.  A page outside the cache, or a length
    past the table, gives NaN."""
    dev, hd, kvh = q.device, cache.head_dim, cache.num_kv_heads
    if q.dtype not in _DTYPES or q.dim() != 2 or q.shape[1] == 0 or q.shape[1] % (hd * kvh) != 0:
        raise ValueError(f"q must be an fp16 or bf16 tensor [T, heads * {hd}] with heads a multiple of {kvh}, got "
                         f"{q.dtype} {tuple(q.shape)}")
    num_heads = q.shape[1] // hd
    if num_heads // kvh > _native.SERVE_MAX_GROUP:
        raise ValueError(f"{num_heads // kvh} heads share a kv head: at most {_native.SERVE_MAX_GROUP} are served")
    if dev.type != "cuda" or cache.data.device != dev:
        raise ValueError(f"q and the cache must be on one ROCm device, got {dev} and {cache.data.device}")
    if block_tables.dim() != 2 or block_tables.dtype is not torch.int32 or not block_tables.is_contiguous() \
            or block_tables.device != dev:
        raise ValueError(f"block_tables must be a contiguous int32 tensor [requests, width] on {dev}")
    requests, width = block_tables.shape
    if not 0 < requests <= _native.SERVE_MAX_REQUESTS or width < 1:
        raise ValueError(f"block_tables {tuple(block_tables.shape)}: need 1 to {_native.SERVE_MAX_REQUESTS} requests")
    if width > 2**30 // cache.page_size:
        raise ValueError("a request's tokens pass 2^30")
    _check_index(seq_lens, "seq_lens", requests, dev)
    _check_index(query_start, "query_start", requests + 1, dev)
    if max_query < 1:
        raise ValueError(f"max_query {max_query} must be positive")
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale {scale} must be positive and finite")
    T = q.shape[0]
    max_query = min(max_query, max(T, 1))
    q = _rows16(q)
    out = torch.empty((T, num_heads * hd), dtype=q.dtype, device=dev)
    if T == 0:
        return out
    L = _native.lib()
    ws = torch.empty(L.awq_serve_kv4_attention_workspace(requests, T, max_query, num_heads, kvh, hd, width,
                                                         cache.page_size), dtype=torch.uint8, device=dev)
    with _OnDevice(dev):
        st = L.awq_serve_kv4_attention(
            q.data_ptr(), q.stride(0) if T > 1 else q.shape[1], cache.data.data_ptr(), block_tables.data_ptr(),
            seq_lens.data_ptr(), query_start.data_ptr(), out.data_ptr(), requests, T, max_query, num_heads, kvh, hd,
            width, cache.num_pages, cache.page_size, cache.group_size, scale, _DTYPES[q.dtype], ws.data_ptr(),
            ws.numel(), _stream_handle(dev))
    _native.check(st, "awq_serve_kv4_attention")
    return out
