"""A decode step's logits under penalties for repeated tokens, biases and a
grammar's mask, and the greedy token of the result (``awq_serve_logits``).

The reference takes its tokens from the logits as they are
(``inference/engine.py:93,127``); the rules here are what a server adds before a
token is chosen.  In this order, in fp32, rounded once to the logits' type:

* repetition: ``x / r`` where ``x > 0``, else ``x * r``, of every token of the history;
* frequency: ``x - f * n``, n how often the request generated the token;
* presence: ``x - p`` where n > 0;
* bias: ``x + b`` of the tokens listed for the request (the last entry of a token);
* mask: -inf where the grammar's bit is 0.

The history is what the request holds anyway, its token ids: no counters are
kept from step to step.
"""
from __future__ import annotations

import torch

from . import _native
from .awq_gemm import _OnDevice, _stream_handle

__all__ = ["process_logits", "MAX_ROWS"]

MAX_ROWS = 65535
_DTYPES = {torch.float16: _native.SERVE_FP16, torch.bfloat16: _native.SERVE_BF16, torch.float32: _native.SERVE_FP32}


def _vector(t: torch.Tensor, what: str, dtype: torch.dtype, n: int, dev: torch.device) -> torch.Tensor:
    if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{what} must be a contiguous {dtype} tensor {(n,)} on {dev}")
    return t


def process_logits(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                   prompt_lens: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                   presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                   bias: tuple | None = None, mask: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """``(logits, next_token)``: the processed logits ``[B, V]`` in the type of ``logits`` (fp16,
    bf16 or fp32, any row stride) and the int64 ``[B]`` lowest index of each row's
    largest (a NaN counts as the largest; -1 where every logit is -inf).

    ``tokens`` int64 or int32 ``[B, L]`` with ``lengths`` and ``prompt_lens`` int32 ``[B]``: the
    request's history, the prompt first (ids outside the vocabulary are ignored).
    ``repetition``, ``presence``, ``frequency`` fp32 ``[B]``: any of them, with a history.  ``bias``:
    ``(start int32 [B + 1], tokens int32 [n], values fp32 [n])``, row b's entries
    ``start[b] .. start[b + 1] - 1``.  ``mask`` int32 ``[B, ceil(V / 32)]``, bit v % 32 of word
    v / 32 set where token v is allowed.  ``out``: a contiguous tensor for the result, which
    may be ``logits`` itself."""
    if logits.dtype not in _DTYPES or logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be an fp16, bf16 or fp32 tensor [B, V], got {logits.dtype} {tuple(logits.shape)}")
    dev, (B, V) = logits.device, logits.shape
    if dev.type != "cuda":
        raise ValueError(f"logits must be on a ROCm device, got {dev}")
    if B > MAX_ROWS or V > (2**31 - 1) // 2:
        raise ValueError(f"logits {tuple(logits.shape)}: at most {MAX_ROWS} rows and 2^30 - 1 tokens are served")
    if logits.stride(1) != 1 or (B > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    ptr = {"tokens": 0, "lengths": 0, "prompt_lens": 0, "repetition": 0, "presence": 0, "frequency": 0, "mask": 0}
    width, token_bytes = 0, 8
    if tokens is not None:
        if tokens.dtype not in (torch.int64, torch.int32) or tokens.dim() != 2 or tokens.shape[0] != B \
                or not tokens.is_contiguous() or tokens.device != dev:
            raise ValueError(f"tokens must be a contiguous int64 or int32 tensor [{B}, L] on {dev}")
        if lengths is None or prompt_lens is None:
            raise ValueError("tokens, lengths and prompt_lens come together")
        width, token_bytes = tokens.shape[1], tokens.element_size()
        ptr["lengths"] = _vector(lengths, "lengths", torch.int32, B, dev).data_ptr()
        ptr["prompt_lens"] = _vector(prompt_lens, "prompt_lens", torch.int32, B, dev).data_ptr()
        # (an empty tensor has no address: without tokens there is no history)
        ptr["tokens"] = tokens.data_ptr()
        if width == 0:
            ptr["tokens"] = ptr["lengths"] = ptr["prompt_lens"] = 0
    elif not (lengths is None and prompt_lens is None and repetition is None and presence is None and frequency is None):
        raise ValueError("penalties need the history: tokens, lengths and prompt_lens")
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            _vector(t, name, torch.float32, B, dev)
            ptr[name] = t.data_ptr() if ptr["tokens"] else 0
    start = ids = values = 0
    count = 0
    if bias is not None:
        if len(bias) != 3 or bias[1].dim() != 1:
            raise ValueError("bias must be (start, tokens, values)")
        count = bias[1].shape[0]
        _vector(bias[0], "bias start", torch.int32, B + 1, dev)
        _vector(bias[1], "bias tokens", torch.int32, count, dev)
        _vector(bias[2], "bias values", torch.float32, count, dev)
        if count:
            start, ids, values = (t.data_ptr() for t in bias)
    if mask is not None:
        if mask.dtype is not torch.int32 or mask.shape != (B, (V + 31) // 32) or not mask.is_contiguous() \
                or mask.device != dev:
            raise ValueError(f"mask must be a contiguous int32 tensor {(B, (V + 31) // 32)} on {dev}")
        ptr["mask"] = mask.data_ptr()
    if out is None:
        out = torch.empty((B, V), dtype=logits.dtype, device=dev)
    elif out.dtype is not logits.dtype or out.shape != (B, V) or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out must be a contiguous {logits.dtype} tensor {(B, V)} on {dev}")
    token = torch.empty(B, dtype=torch.int64, device=dev)
    if B == 0:
        return out, token
    L = _native.lib()
    ws = torch.empty(L.awq_serve_logits_workspace(B, V), dtype=torch.uint8, device=dev)
    with _OnDevice(dev):
        st = L.awq_serve_logits(logits.data_ptr(), logits.stride(0) if B > 1 else V, out.data_ptr(), token.data_ptr(),
                                B, V, _DTYPES[logits.dtype], ptr["tokens"], token_bytes, width, ptr["lengths"],
                                ptr["prompt_lens"], ptr["repetition"], ptr["presence"], ptr["frequency"], start, ids,
                                values, count, ptr["mask"], ws.data_ptr(), ws.numel(), _stream_handle(dev))
    _native.check(st, "awq_serve_logits")
    return out, token
