"""Greedy decoding and scoring of many requests at once over one paged cache, in 4 bits or in 16.

``Qwen2AwqDecoder`` (``engine/qwen2_decode.py``) has one sequence and a static
fp16 cache, as the reference has (``inference/engine.py:64-147``,
``inference/kv_cache.py:31-67``).  ``Qwen2BatchDecoder`` runs the same weights for a
batch: the prompts of all requests in one pass, then one token of each per step.  A
step is

* ``paged_step``: where the step's tokens are stored, which positions they stand at;
* per layer, the AWQ projections and norms of the single decoder, and between them
  ``kv4_append`` (RoPE, the cache's new rows) and ``kv4_attention``, or ``kv16_append`` and ``kv16_attention``;
* the output projection of each request's last row;
* ``process_logits``: penalties, biases, a grammar's mask, and the greedy token.

A token takes ``head_dim + 8 head_dim / group_size`` bytes of a kv head in a layer in 4 bits, 144 for heads of
128 in groups of 64, and 512 in 16.

``score`` gives the log-probabilities of texts' tokens (perplexity, the likelihood of an answer): the same passes
over chunks of the texts, and ``token_logprobs`` in the place of the logits.
"""
from __future__ import annotations

import torch

from engine.qwen2_decode import Qwen2AwqDecoder
from kernels.awq_gemm import awq_gemm_forward_ex
from kernels.kv16 import Kv16Cache, kv16_append, kv16_attention
from kernels.kv4 import HEAD_DIMS, Kv4Cache, kv4_append, kv4_attention
from kernels.lm_head import MAX_ROWS, lm_head_forward
from kernels.logits import process_logits
from kernels.logprobs import token_logprobs
from kernels.paged import PagedStep, PagedTables, paged_release, paged_step
from kernels.rmsnorm import rmsnorm
from kernels.silu_mul import silu_mul_gate_up

__all__ = ["Qwen2BatchDecoder"]


class Qwen2BatchDecoder:
    """``model``'s weights and RoPE tables for up to ``max_requests`` requests that
    share ``num_pages`` pages of ``page_size`` tokens (unless given: enough for all of them
    at the model's ``max_seq_len``).  ``cache_bits``: 4, with scales for groups of ``group_size`` columns, or 16,
    keys and values as the model gives them."""

    def __init__(self, model: Qwen2AwqDecoder, max_requests: int, num_pages: int | None = None, page_size: int = 64,
                 group_size: int = 64, cache_bits: int = 4):
        s = model.s
        if s.head_dim not in HEAD_DIMS:
            raise ValueError(f"heads of {s.head_dim} columns are not served (only {HEAD_DIMS})")
        if cache_bits not in (4, 16):
            raise ValueError(f"cache_bits {cache_bits} must be 4 or 16")
        self.model, self.s, self.dev = model, s, model.dev
        width = -(-model.max_seq_len // page_size)
        num_pages = max_requests * width if num_pages is None else num_pages
        self.tables = PagedTables(max_requests, width, num_pages, page_size, self.dev)
        if cache_bits == 16:
            self._data = torch.zeros((s.num_layers, num_pages, s.num_kv_heads, 2, page_size, s.head_dim), dtype=torch.float16,
                                     device=self.dev)
            self.caches = [Kv16Cache.of(d) for d in self._data]
        else:
            self._data = torch.zeros((s.num_layers, num_pages, s.num_kv_heads,
                                      Kv4Cache.block_bytes(s.head_dim, page_size, group_size)), dtype=torch.uint8,
                                     device=self.dev)
            self.caches = [Kv4Cache.of(d, s.head_dim, page_size, group_size) for d in self._data]
        self.failed = torch.zeros(max_requests, dtype=torch.int32, device=self.dev)   # of the last step

    # ---- one pass over a step's rows ---------------------------------------------
    def _place(self, new_tokens: torch.Tensor, total: int) -> PagedStep:
        """``paged_step`` under the model's ``max_seq_len``, which the tables know as whole pages
        only.  A request that would pass it inside its last page is shown to the step with
        a length that the step refuses, and keeps its own."""
        t, limit = self.tables, self.model.max_seq_len
        if limit % t.page_size == 0 or new_tokens.shape != t.lengths.shape or new_tokens.device != t.state.device:
            return paged_step(t, new_tokens, total)      # (which refuses what is no int32 tensor of the tables')
        over = t.lengths + new_tokens > limit
        state = torch.cat((t.lengths.masked_fill(over, -1), t.free_count))
        step = paged_step(PagedTables.of(t.block_tables, state, t.free_pages, t.page_size), new_tokens, total)
        step.lengths.copy_(torch.where(over, t.lengths, step.lengths))
        return step

    def _attention(self, li: int, qkv: torch.Tensor, step: PagedStep, max_query: int) -> torch.Tensor:
        m, cache = self.model, self.caches[li]
        append, attention = (kv16_append, kv16_attention) if isinstance(cache, Kv16Cache) else (kv4_append, kv4_attention)
        q = append(qkv, cache, step.slots, step.positions, m.cos, m.sin, self.s.num_heads)
        return attention(q, cache, self.tables.block_tables, step.lengths, step.query_start, max_query)

    def _rows(self, ids: torch.Tensor, step: PagedStep, max_query: int) -> torch.Tensor:
        """Hidden states of the rows ``ids`` after the last layer."""
        eps = self.s.rms_norm_eps
        h = torch.nn.functional.embedding(ids, self.model.embed)
        for li, p in enumerate(self.model.layers):
            qkv = awq_gemm_forward_ex(rmsnorm(h, p["ln1"], eps), *p["qkv"], bias=p["qkv_bias"])
            h = awq_gemm_forward_ex(self._attention(li, qkv, step, max_query), *p["o"], residual=h)
            inter = silu_mul_gate_up(awq_gemm_forward_ex(rmsnorm(h, p["ln2"], eps), *p["gate_up"]))
            h = awq_gemm_forward_ex(inter, *p["down"], residual=h)
        return h

    def _pass(self, ids: torch.Tensor, new_tokens: torch.Tensor, max_query: int):
        """(hidden states of the rows, the step), which is committed."""
        step = self._place(new_tokens, ids.shape[0])
        h = self._rows(ids, step, max_query)
        self.tables.commit(step)
        self.failed = step.failed
        return h, step

    def _logits(self, h: torch.Tensor) -> torch.Tensor:
        """fp16 [rows, vocab] of hidden states [rows, hidden]."""
        last = rmsnorm(h.contiguous(), self.model.final_norm, self.s.rms_norm_eps)
        out = torch.empty((h.shape[0], self.s.vocab_size), dtype=torch.float16, device=self.dev)
        for at in range(0, h.shape[0], MAX_ROWS):       # the kernel serves eight rows
            lm_head_forward(last[at:at + MAX_ROWS], self.model.lm_head, out=out[at:at + MAX_ROWS])
        return out

    # ---- public API ---------------------------------------------------------------
    @torch.no_grad()
    def step(self, ids: torch.Tensor, new_tokens: torch.Tensor, max_query: int, requests: int | None = None) -> torch.Tensor:
        """Logits fp16 ``[requests, vocab]`` of each request's last row after one pass:
        ``ids`` int64 the rows of all requests (within the vocabulary), ``new_tokens`` int32 ``[max_requests]`` how many
        of them each has, ``max_query`` at least the most of one, ``requests`` the first so many
        whose logits are wanted (all).  A request that adds no row has no logits of its own: its row
        is another request's.

        Nothing here waits for the device, so what it refuses -- a request whose pages or
        rows do not suffice (``paged_step``), or whose tokens would pass ``max_seq_len`` -- is told in ``failed``, int32 ``[max_requests]``, 1
        where this step refused a request: it keeps its length, nothing of it is stored, and its
        logits are NaN.  The other requests' tokens count."""
        h, step = self._pass(ids, new_tokens, max_query)
        ends = (step.query_start[1:].long() - 1).clamp(min=0)[:requests]
        refused = step.failed[:requests].bool().unsqueeze(1)
        return self._logits(h.index_select(0, ends).masked_fill(refused, float("nan")))

    def _check(self, prompts, new_tokens):
        """Texts and tokens after them (none: the texts' own), all but the last of which are stored."""
        requests, page = len(prompts), self.tables.page_size
        if not 0 < requests <= self.tables.block_tables.shape[0]:
            raise ValueError(f"{requests} prompts for a decoder of {self.tables.block_tables.shape[0]} requests")
        if new_tokens < 0 or any(p.dim() != 1 or p.shape[0] < 1 for p in prompts):
            raise ValueError("each prompt must be a 1-D tensor of at least one token, and new_tokens positive")
        ends = [p.shape[0] + new_tokens for p in prompts]
        if max(ends) > self.model.max_seq_len:
            raise ValueError(f"prompt + new tokens ({max(ends)}) exceed max_seq_len {self.model.max_seq_len}")
        pages = sum(-(-(n - 1) // page) for n in ends)   # the last token is returned and not stored
        if pages > self.tables.free_pages.shape[0]:
            raise ValueError(f"the requests need {pages} pages, the cache has {self.tables.free_pages.shape[0]}")
        if self.tables.lengths.any():
            raise RuntimeError("requests of earlier steps are running: release their pages (paged_release) first")

    @torch.no_grad()
    def generate(self, prompts: list, new_tokens: int, repetition: float = 1.0, presence: float = 0.0,
                 frequency: float = 0.0, biases: list | None = None, mask: torch.Tensor | None = None) -> torch.Tensor:
        """``new_tokens`` greedy tokens of each prompt (a list of 1-D id tensors): int64
        ``[requests, new_tokens]`` on the host.  Penalties as in ``process_logits``, the same for all
        requests; ``biases`` a dict {token: value} per request; ``mask`` int32
        ``[requests, ceil(vocab / 32)]``, the tokens that a request's grammar allows.  All
        requests' pages are returned at the end.  Raises if a mask left a request no token, and if
        requests that a caller of ``step`` began are still running (it has all pages to itself)."""
        self._check(prompts, new_tokens if new_tokens > 0 else -1)
        B, slots, dev = len(prompts), self.tables.block_tables.shape[0], self.dev
        lens = [p.shape[0] for p in prompts]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        history = torch.zeros((B, max(lens) + new_tokens), dtype=torch.int64, device=dev)
        for b, p in enumerate(prompts):
            history[b, :lens[b]] = p.to(dev)
        ids, most = torch.cat([p.to(dev) for p in prompts]), max(lens)
        if ((ids < 0) | (ids >= self.s.vocab_size)).any():
            raise ValueError(f"a prompt has a token outside the vocabulary [0, {self.s.vocab_size})")
        prompt_lens = i32(lens)
        each = lambda v: torch.full((B,), v, dtype=torch.float32, device=dev)  # noqa: E731
        rules = {"repetition": each(repetition), "presence": each(presence), "frequency": each(frequency), "mask": mask,
                 "prompt_lens": prompt_lens}
        if biases is not None:
            if len(biases) != B:
                raise ValueError(f"biases of {len(biases)} requests for {B} prompts")
            counts = [len(d) for d in biases]
            rules["bias"] = (i32([sum(counts[:b]) for b in range(B + 1)]), i32([t for d in biases for t in d]),
                             torch.tensor([float(v) for d in biases for v in d.values()], dtype=torch.float32, device=dev))
        new = i32(lens + [0] * (slots - B))
        rows = torch.arange(B, device=dev)
        out = []
        try:
            for i in range(new_tokens):
                logits = self.step(ids, new, most, B)
                lengths = prompt_lens + i
                _, token = process_logits(logits, tokens=history, lengths=lengths, out=logits, **rules)
                out.append(token)
                # a token that does not exist (-1) must not reach the embedding; reported below
                ids, most = token.clamp(min=0), 1
                history[rows, lengths.long()] = ids
                if i == 0:
                    new = i32([1] * B + [0] * (slots - B))
        finally:                                        # also of a call that fails or is interrupted
            paged_release(self.tables, torch.zeros(slots, dtype=torch.int32, device=dev))
        tokens = torch.stack(out, 1).cpu()
        if (tokens < 0).any():
            raise RuntimeError("the mask left a request no token to take")
        return tokens

    @torch.no_grad()
    def score(self, texts: list, chunk: int = 2048) -> list:
        """The log-probabilities of texts' tokens, each given those before it: for each text (a 1-D id tensor of n tokens)
        fp32 ``[n - 1]`` on the host, of its tokens 1 .. n - 1.  Their mean's negative is the logarithm of the text's
        perplexity.  ``chunk``: the most rows of a pass; texts go through in order, as many at a time as fit.  All
        pages are returned at the end.  Raises if requests that a caller of ``step`` began are still running."""
        if chunk < 1:
            raise ValueError(f"chunk {chunk} must be positive")
        self._check(texts, 0)
        slots, dev = self.tables.block_tables.shape[0], self.dev
        texts = [t.to(dev) for t in texts]
        every = torch.cat(texts)
        if ((every < 0) | (every >= self.s.vocab_size)).any():
            raise ValueError(f"a text has a token outside the vocabulary [0, {self.s.vocab_size})")
        left = [t.shape[0] - 1 for t in texts]           # the last token is scored and not stored
        parts = [[] for _ in texts]
        try:
            while any(left):
                room, new = chunk, [0] * slots
                ids, targets = [], []
                for b, text in enumerate(texts):
                    new[b] = min(left[b], room)
                    if new[b]:
                        at = text.shape[0] - 1 - left[b]
                        ids.append(text[at:at + new[b]])
                        targets.append(text[at + 1:at + 1 + new[b]])
                    left[b] -= new[b]
                    room -= new[b]
                h, _ = self._pass(torch.cat(ids), torch.tensor(new, dtype=torch.int32, device=dev), max(new))
                last = rmsnorm(h, self.model.final_norm, self.s.rms_norm_eps)
                scores, _ = token_logprobs(last, self.model.lm_head, torch.cat(targets))
                for b, s in enumerate(scores.split(new[:len(texts)])):
                    parts[b].append(s)
        finally:                                         # also of a call that fails or is interrupted
            paged_release(self.tables, torch.zeros(slots, dtype=torch.int32, device=dev))
        return [torch.cat(p).cpu() if p else torch.zeros(0) for p in parts]
