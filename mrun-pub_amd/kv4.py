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
"""

from __future__ import annotations

import functools
import math

import torch

from . import _native as nat
from .rotary import RotarySpec, check_positions

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
        self._bases = [int(self.storage[i].data_ptr()) for i in range(self.layers)]

    @property
    def nbytes(self) -> int:
        return int(self.storage.numel())

    def layer_ptr(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of a cache of {self.layers}")
        return self._bases[layer]


def _heads(name: str, x: torch.Tensor, tokens: int, heads: int | None, head_dim: int, values: int) -> torch.Tensor:
    """``x [tokens, heads, head_dim]`` with heads aligned to ``values`` values (copied if it is not)."""
    if x.ndim != 3 or int(x.shape[0]) != tokens or int(x.shape[2]) != head_dim:
        raise ValueError(f"{name} must have shape [{tokens}, heads, {head_dim}]")
    if heads is not None and int(x.shape[1]) != heads:
        raise ValueError(f"{name} must have {heads} heads")
    t, h, one = x.stride()
    size = x.element_size() * values
    if one != 1 or t % values or h % values or x.data_ptr() % size:
        x = x.contiguous()
        if x.data_ptr() % size:  # a contiguous view that starts off the grid
            x = x.clone()
    return x


def _slots(slots: torch.Tensor, tokens: int) -> torch.Tensor:
    if slots.ndim != 1 or int(slots.numel()) != tokens or slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("slots must be an int32 or int64 vector of one slot per token")
    return slots.to(torch.int64).contiguous()


@nat.inference
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
    code = nat.dtype_code(k.dtype)
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError("queries, keys and values must share one type")
    if k.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError("keys and values must be float32, bfloat16 or float16")
    T, D = int(k.shape[0]), cache.head_dim
    k = _heads("keys", k, T, cache.kv_heads, D, 4)
    v = _heads("values", v, T, cache.kv_heads, D, 4)
    slot = _slots(slots, T)
    base = cache.layer_ptr(layer)
    device = nat.require_device(k, v, slot, cache.storage, q, positions)
    if (rotary is None) != (positions is None):
        raise ValueError("rotary positions need both a spec and positions")
    if q is not None and rotary is None:
        raise ValueError("queries are only turned: without rotary positions there is nothing to do for them")
    rot, freq, pos, interleaved, magnitude = 0, None, None, 0, 1.0
    if rotary is not None:
        if rotary.dim > D or rotary.dim % 8:
            raise ValueError(f"the rotated size must be a multiple of 8 up to {D}")
        pos = check_positions(positions, T)
        rot, freq, magnitude = rotary.dim, rotary.on(device), rotary.magnitude
        interleaved = int(rotary.layout == "interleaved")
    q_out, Hq, q_strides = None, 0, (0, 0)
    if q is not None:
        q = _heads("queries", q, T, None, D, 4)
        Hq, q_strides = int(q.shape[1]), (q.stride(0), q.stride(1))
        q_out = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    nat.call(
        "qs_kv4_append", nat.ptr(k), k.stride(0), k.stride(1), nat.ptr(v), v.stride(0), v.stride(1), code,
        nat.ptr(slot), base, cache.pages, cache.page_size, cache.kv_heads, D, T, nat.ptr(q), *q_strides, Hq,
        nat.ptr(q_out), nat.ptr(pos), nat.ptr(freq), rot, interleaved, magnitude, nat.stream_of(device),
    )
    return q_out


@nat.inference
def read(cache: KV4Cache, layer: int, slots: torch.Tensor, *,
         dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[n, kv_heads, head_dim]`` that ``slots [n]`` stand for (zeros for a slot
    outside the cache), computed in fp32 and rounded once to ``dtype``."""
    if dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError("cache values are read as float32, bfloat16 or float16")
    n = int(slots.numel())
    slot = _slots(slots, n)
    base = cache.layer_ptr(layer)
    device = nat.require_device(slot, cache.storage)
    k, v = (torch.empty((n, cache.kv_heads, cache.head_dim), dtype=dtype, device=device) for _ in range(2))
    nat.call(
        "qs_kv4_read", base, cache.pages, cache.page_size, cache.kv_heads, cache.head_dim, nat.ptr(slot), n,
        nat.ptr(k), nat.ptr(v), nat.dtype_code(dtype), nat.stream_of(device),
    )
    return k, v


@functools.lru_cache(maxsize=512)
def _attend_space(*sizes: int) -> int:
    return int(nat.load().qs_kv4_attend_workspace_bytes(*sizes))


@nat.inference
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
    if q.ndim != 3 or q.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError("queries must be float32, bfloat16 or float16 [tokens, heads, head_dim]")
    T, Hq, D = map(int, q.shape)
    if D != cache.head_dim or Hq < 1 or Hq % cache.kv_heads:
        raise ValueError("query heads must be a multiple of the cache's KV heads, of its head size")
    B = int(context_lens.numel())
    if block_tables.ndim != 2 or block_tables.dtype != torch.int32 or int(block_tables.shape[0]) != B:
        raise ValueError("block tables must be int32 [requests, columns]")
    if block_tables.numel() and block_tables.stride(1) != 1:
        raise ValueError("block table rows must be contiguous")
    if query_starts.ndim != 1 or int(query_starts.numel()) != B + 1 or query_starts.dtype != torch.int32:
        raise ValueError("query_starts must be int32, one more than requests")
    if context_lens.ndim != 1 or context_lens.dtype != torch.int32:
        raise ValueError("context_lens must be an int32 vector")
    width = int(block_tables.shape[1])
    most = width * cache.page_size
    mq = T if max_query is None else int(max_query)
    mc = most if max_context is None else min(int(max_context), most)
    mc = -(-mc // 512) * 512  # so that a step's plan serves the next steps
    win = int(window or 0)
    if mq < 0 or mc < 0 or (window is not None and window < 1):
        raise ValueError("bounds must not be negative and a window holds at least one token")
    s = 1.0 / math.sqrt(D) if scale is None else float(scale)
    q = _heads("queries", q, T, None, D, 4 if q.dtype == torch.float32 else 8)
    starts, ctx = query_starts.contiguous(), context_lens.contiguous()
    base = cache.layer_ptr(layer)
    device = nat.require_device(q, cache.storage, block_tables, starts, ctx, out)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("attention output must be contiguous, 16-byte aligned, of the queries' shape and type")
    stream = nat.stream_of(device)
    need = _attend_space(T, B, cache.kv_heads, Hq, D, cache.page_size, mq, mc, win)
    workspace = nat.kept_workspace(device, stream, need) if need else None
    nat.call(
        "qs_kv4_attend", nat.ptr(q), nat.dtype_code(q.dtype), q.stride(0), q.stride(1), base, cache.pages,
        cache.page_size, cache.kv_heads, Hq, D, nat.ptr(block_tables), block_tables.stride(0), width, nat.ptr(starts),
        nat.ptr(ctx), B, T, mq, mc, s, win, nat.ptr(out), nat.ptr(workspace), need, stream,
    )
    return out
