"""The paged 4-bit KV cache and attention over it, on gfx950.

``KV4Cache`` holds, for every layer, ``pages`` pages of ``page_size`` tokens: each key and value of a
head in groups of 64 values with ``lo = fp16(min)``, ``s = fp16((max - min) / 15)`` and 4-bit codes
``clamp(rint((x - lo) / s), 0, 15)``; a code stands for ``code * s + lo``.  That is 72 bytes for a
token's key of 128 values, against 256 in 16 bits.  NaN is stored as 0 and values are held to
+-60000.

* ``append`` codes a step's keys and values into their slots (``paging.plan_step`` gives them) and
  turns queries and keys by their rotary positions on the way;
* ``attend`` is attention of the step's queries over the cache, the step's own tokens included;
* ``read`` gives back what slots hold.

They are for serving: results are inference tensors, and no gradient goes through them.
"""

from __future__ import annotations

import torch

from . import _native as nat
from .rotary import RotarySpec

HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)
GROUP = 64


class KV4Cache:
    """Storage of ``layers`` layers: uint8 ``[layers, pages, kv_heads, block bytes]``, zeroed."""

    def __init__(self, *, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int, device):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if layers < 1 or kv_heads < 1 or pages < 1:
            raise ValueError("a cache needs at least one layer, head and page")
        self.layers, self.kv_heads, self.head_dim = int(layers), int(kv_heads), int(head_dim)
        self.pages, self.page_size = int(pages), int(page_size)
        block = int(nat.load().qs_kv4_block_bytes(head_dim, page_size))
        self.storage = torch.zeros((layers, pages, kv_heads, block), dtype=torch.uint8, device=device)
        bases = tuple(int(self.storage[i].data_ptr()) for i in range(self.layers))
        # as the binding takes a cache
        self.native = (self.storage, bases, self.kv_heads, self.head_dim, self.pages, self.page_size)

    @property
    def nbytes(self) -> int:
        return int(self.storage.numel())


def append(
    cache: KV4Cache, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
    q: torch.Tensor | None = None, positions: torch.Tensor | None = None, rotary: RotarySpec | None = None,
) -> torch.Tensor | None:
    """Code ``k`` and ``v`` ``[tokens, kv_heads, head_dim]`` (fp32, bf16 or fp16) into ``slots``.

    With ``rotary`` (and ``positions``), keys are turned first, rounded to their type, and so are
    the queries ``q [tokens, heads, head_dim]``, which are returned (contiguous).  Slots outside the
    cache (-1: padding) are passed over, their queries are still turned.  A slot is given at most
    once.  k, v and q may be views of one fused projection.
    """
    turn, freq = None, None
    if rotary is not None:
        turn, freq = rotary.native, rotary.on(k.device) if k.is_cuda else None
    return nat.fast().append(cache.native, layer, k, v, slots, q, positions, turn, freq)


def read(cache: KV4Cache, layer: int, slots: torch.Tensor, *,
         dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[n, kv_heads, head_dim]`` that ``slots [n]`` stand for (zeros for a slot
    outside the cache), computed in fp32 and rounded once to ``dtype``."""
    return nat.fast().read(cache.native, layer, slots, nat.dtype_code(dtype))


def attend(
    q: torch.Tensor, cache: KV4Cache, layer: int, block_tables: torch.Tensor, query_starts: torch.Tensor,
    context_lens: torch.Tensor, *, max_query: int | None = None, max_context: int | None = None,
    scale: float | None = None, window: int | None = None, out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of new tokens over the cache, ``[tokens, heads, head_dim]`` in q's type.

    Request b's queries are rows ``query_starts[b] .. query_starts[b + 1] - 1`` of ``q`` (fp32, bf16
    or fp16) and stand at the end of its ``context_lens[b]`` tokens, which ``append`` put into the
    pages of ``block_tables[b]`` (the step's own tokens too): one token (decode), a few (drafts to
    verify) or a whole prompt, ragged, in one call.  A query sees the tokens up to its own, with
    ``window`` the last ``window`` of them; query heads share KV heads in equal groups.  Tokens
    whose table entry is no page of the cache are not seen; a query that sees nothing (a row of
    padding after the last request, a context of 0) gives zeros.  ``scale`` defaults to
    ``head_dim ** -0.5``.

    ``max_query`` and ``max_context`` bound the requests' new tokens and contexts; they choose how
    the work is split, never what is computed, and default to the largest that the shapes allow.
    ``query_starts`` must not decrease.
    """
    return nat.fast().attend(
        q, cache.native, layer, block_tables, query_starts, context_lens, max_query, max_context, scale, window, out
    )
