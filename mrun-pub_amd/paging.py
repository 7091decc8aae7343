"""Paging metadata of a serving step, built on the GPU from request lengths.

A pool of pages is a ring of free page numbers (int32) and a state of three int64 on the device:
``(head, tail, missing)``, where the free pages are ring entries ``head .. tail - 1`` modulo the
ring's size and ``missing`` counts the pages that the last plan asked for and did not get.
``plan_step`` takes pages from the head, ``release_pages`` returns them at the tail.  Both leave the
old state as it is and give the new one, so that a step can be planned again or captured into a
graph, and nothing waits for the GPU.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat


def free_pages(pages: int, device, *, first: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """``(ring, state)`` of a pool whose pages ``first .. pages - 1`` are all free."""
    if not 0 <= first < pages:
        raise ValueError("a pool needs at least one free page")
    ring = torch.arange(first, pages, dtype=torch.int32, device=device)
    return ring, torch.tensor([0, pages - first, 0], dtype=torch.int64, device=device)


class StepPlan(NamedTuple):
    """One step's metadata; every tensor is on the device, all six in one allocation, which the last of
    them that is held keeps.

    ``slots [tokens] int64`` (page * page_size + offset; -1 for a row of padding or one whose page
    was missing), ``positions [tokens] int32``, ``requests [tokens] int32`` (-1 for padding),
    ``query_starts [B + 1] int32``, ``context_lens [B] int32``, ``free_state [3] int64``.
    """

    slots: torch.Tensor
    positions: torch.Tensor
    requests: torch.Tensor
    query_starts: torch.Tensor
    context_lens: torch.Tensor
    free_state: torch.Tensor


def _pool(ring: torch.Tensor, state: torch.Tensor) -> None:
    if ring.ndim != 1 or ring.dtype != torch.int32 or not ring.numel() or not ring.is_contiguous():
        raise ValueError("the ring of free pages must be a contiguous int32 vector")
    if state.shape != (3,) or state.dtype != torch.int64 or not state.is_contiguous():
        raise ValueError("the pool's state must be three int64")


def _tables(block_tables: torch.Tensor, requests: int) -> None:
    if block_tables.ndim != 2 or block_tables.dtype != torch.int32 or int(block_tables.shape[0]) != requests:
        raise ValueError("block tables must be int32 [requests, columns]")
    if block_tables.numel() and block_tables.shape[1] > 1 and block_tables.stride(1) != 1:
        raise ValueError("block table rows must be contiguous")


def _lengths(name: str, lens: torch.Tensor, requests: int) -> torch.Tensor:
    if lens.ndim != 1 or int(lens.numel()) != requests or lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 vector of one length per request")
    return lens.to(torch.int32).contiguous()


def plan_step(
    ring: torch.Tensor, free_state: torch.Tensor, block_tables: torch.Tensor, past_lens: torch.Tensor,
    new_lens: torch.Tensor, *, page_size: int, tokens: int,
) -> StepPlan:
    """Where each of a step's tokens goes: request b has ``past_lens[b]`` tokens in the cache and
    brings ``new_lens[b]`` (0 included; negative lengths count as 0).

    New pages are taken from the pool in request order and entered into ``block_tables`` in place;
    columns that a request already holds are read.  ``tokens`` is the number of rows to describe, at
    least the sum of the new lengths: rows after them are padding, and if it is less, the rest of
    the new tokens are left out, their pages and context too.  Columns past the table's width take
    no pages.
    """
    return StepPlan._make(
        nat.fast().plan_step(ring, free_state, block_tables, past_lens, new_lens, page_size, tokens)
    )


@nat.inference
def release_pages(
    ring: torch.Tensor, free_state: torch.Tensor, block_tables: torch.Tensor, lens: torch.Tensor,
    done: torch.Tensor, *, page_size: int,
) -> torch.Tensor:
    """The pool's new state after the pages of requests with ``done[b]`` (bool), which hold
    ``lens[b]`` tokens, went back to the ring, in request order.  Table entries of -1 are passed
    over; the tables keep their entries.  The ring has room for the pages that were taken from it and
    is not checked for more: a page given back twice overwrites a free one's entry."""
    _pool(ring, free_state)
    B = int(lens.numel())
    held = _lengths("lens", lens, B)
    _tables(block_tables, B)
    if done.dtype != torch.bool or done.shape != (B,):
        raise ValueError("done must be a bool vector of one value per request")
    device = nat.require_device(ring, free_state, block_tables, held, done)
    state = torch.empty(3, dtype=torch.int64, device=device)
    with torch.cuda.device(device):  # the default stream's handle means the current device's
        nat.call(
            "qs_release_pages", nat.ptr(ring), int(ring.numel()), nat.ptr(free_state), nat.ptr(state),
            nat.ptr(block_tables), block_tables.stride(0), int(block_tables.shape[1]), nat.ptr(held),
            nat.ptr(done.contiguous()), B, int(page_size), nat.stream_of(device),
        )
    return state
