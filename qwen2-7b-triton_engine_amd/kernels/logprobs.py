"""Log-probabilities of given tokens under the output projection, without its logits
(``awq_serve_logprobs``).

What scoring a text needs -- its perplexity, the likelihood of an answer: the reference
computes all logits of all positions (``model/qwen2.py:280``) and keeps the last position's;
for a text of 2047 tokens and 152064 of vocabulary they are 1.2 GB in fp32.  Here a tile of
them leaves only its maximum, its sum of exponentials and the target's logit.
"""
from __future__ import annotations

import torch

from . import _native

__all__ = ["token_logprobs"]


def token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor):
    """``(logprobs, lse)``, both fp32 ``[T]``: with the logits ``z = hidden @ weight.T``, ``lse`` is log sum exp z and
    ``logprobs`` is z[target] - lse.

    ``hidden`` fp16 or bf16 ``[T, K]`` (any row stride), ``weight`` ``[V, K]`` of the same type (``nn.Linear.weight``), K a
    multiple of 64, ``targets`` int64 or int32 ``[T]``: a negative one (no target) gives 0, one of V or more NaN.
    Products are exact and summed in fp32.  Not differentiable: the results carry no gradient, whatever the inputs.  A
    ``weight`` that is not contiguous, or does not begin on 16 bytes, is copied whole in each call."""
    return _native.binding().token_logprobs(hidden, weight, targets)
