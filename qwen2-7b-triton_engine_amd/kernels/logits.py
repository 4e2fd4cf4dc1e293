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

__all__ = ["process_logits", "MAX_ROWS"]

MAX_ROWS = 65535

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
    return _native.binding().process_logits(logits, tokens, lengths, prompt_lens, repetition, presence, frequency, bias,
                                            mask, out)
