"""Block tables, slots and positions of a serving step, built on the GPU from
the requests' lengths (``awq_serve_page_step``, ``awq_serve_page_release``).

A cache of pages is shared by up to ``MAX_REQUESTS`` requests (``PagedTables``):
which pages a request has, how many tokens it holds, and which pages are free.
``paged_step`` adds a step's new tokens -- one each while decoding, a prompt or a
chunk of one before -- and returns a ``PagedStep``: where each row of the batch is
stored and which position it stands at, and the state after the step.  It
changes neither lengths nor free pages until ``PagedTables.commit``, so a step in
which a request was refused (``PagedStep.failed``) can be given up or made smaller.
The reference has one static cache and one sequence
(``inference/kv_cache.py:31-67``); these have no counterpart there.
"""
from __future__ import annotations

import dataclasses

import torch

from . import _native

__all__ = ["PagedTables", "PagedStep", "paged_step", "paged_release", "MAX_REQUESTS", "PAGE_SIZES"]

MAX_REQUESTS = _native.SERVE_MAX_REQUESTS
PAGE_SIZES = (16, 32, 64, 128, 256)


@dataclasses.dataclass
class PagedTables:
    """``block_tables`` int32 ``[requests, width]``: the pages of each request in
    order; ``state`` int32 ``[requests + 1]``: the requests' lengths, then the
    number of free pages; ``free_pages`` int32 ``[capacity]``, as many as can be free
    at once, the first ``state[-1]`` of them free, taken from the end."""

    block_tables: torch.Tensor
    state: torch.Tensor
    free_pages: torch.Tensor
    page_size: int

    def __init__(self, requests: int, width: int, num_pages: int, page_size: int = 64,
                 device: torch.device | str = "cuda:0"):
        dev = torch.device(device)
        self._set(torch.full((requests, width), -1, dtype=torch.int32, device=dev),
                  torch.zeros(requests + 1, dtype=torch.int32, device=dev),
                  # from the end: page 0 is taken first
                  torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=dev), page_size)
        self.state[-1] = num_pages

    @classmethod
    def of(cls, block_tables: torch.Tensor, state: torch.Tensor, free_pages: torch.Tensor,
           page_size: int = 64) -> "PagedTables":
        """Tables over tensors that exist; they are used in place."""
        t = cls.__new__(cls)
        t._set(block_tables, state, free_pages, page_size)
        return t

    def _set(self, block_tables, state, free_pages, page_size):
        _native.binding().check_tables(block_tables, state, free_pages, page_size)
        self.block_tables, self.state, self.free_pages, self.page_size = block_tables, state, free_pages, page_size

    @property
    def lengths(self) -> torch.Tensor:
        return self.state[:-1]

    @property
    def free_count(self) -> torch.Tensor:
        return self.state[-1:]

    def commit(self, step: "PagedStep") -> None:
        """The step's lengths and free pages become the tables' (the tensor itself: no copy).  A step
        goes with the state that it was made from: not after a release or another step's commit."""
        if step.state.shape != self.state.shape or step.state.device != self.state.device:
            raise ValueError("the step belongs to other tables")
        self.state = step.state


@dataclasses.dataclass
class PagedStep:
    """``slots`` and ``positions`` int32 ``[total]`` of the batch's rows (-1: no token),
    ``query_start`` int32 ``[requests + 1]`` the requests' first rows, ``state`` as the
    tables' after the step (``lengths`` of it: with the new tokens), ``failed`` int32
    ``[requests]``, 1 where a request was refused."""

    state: torch.Tensor
    query_start: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    failed: torch.Tensor

    @property
    def lengths(self) -> torch.Tensor:
        return self.state[:-1]

    @classmethod
    def empty(cls, requests: int, total: int, device: torch.device) -> "PagedStep":
        # one allocation: an allocator call costs about as much as the launch
        sizes = (requests + 1, requests + 1, total, total, requests)
        flat = torch.empty(sum(sizes), dtype=torch.int32, device=device)
        return cls(*flat.split(sizes))


def paged_step(tables: PagedTables, new_tokens: torch.Tensor, total: int, out: PagedStep | None = None) -> PagedStep:
    """The rows of ``new_tokens`` (int32 ``[requests]``) more tokens of each request in a
    batch of ``total`` rows, the first request's first.  New pages are entered into
    ``tables.block_tables``; lengths and free pages change with ``tables.commit``.

    A request is refused -- ``failed`` 1, slots and positions -1, nothing taken -- whose
    rows pass ``total``, whose tokens pass its table's width, or for which and all
    before it the free pages do not suffice.  ``out``: a step of the same sizes
    whose tensors are reused (not the one whose ``state`` the tables hold)."""
    r = _native.binding().paged_step(
        tables.state, new_tokens, tables.block_tables, tables.free_pages, tables.page_size, total,
        None if out is None else [out.state, out.query_start, out.slots, out.positions, out.failed])
    return PagedStep(*r) if out is None else out


def paged_release(tables: PagedTables, keep: torch.Tensor) -> None:
    """Request b keeps its first ``keep[b]`` tokens (int32 ``[requests]``; 0: the request
    ended) and returns the pages past them."""
    tables.state = _native.binding().paged_release(tables.state, keep, tables.block_tables, tables.free_pages,
                                                   tables.page_size)
