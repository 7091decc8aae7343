"""Attention, its cache, rotary positions and paging at the edges of what their calls allow, on the GPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mrun_pub_amd import kv4, paging
from oracle import attention as oa
from test_gpu_attention import Setup, f64, i32

pytestmark = pytest.mark.gpu


def narrow(s, columns):
    """The first columns of a setup's table: tokens past them are not seen."""
    s.tables = s.tables[:, :columns]
    most = columns * s.cache.page_size
    for x in s.keys:
        x[most:] = np.nan
    for x in s.values:
        x[most:] = 0


def check_unseen(s, out, window):
    """Queries that see nothing give zeros, the others what the plain form gives."""
    _, weight, _ = oa.attend(f64(s.q), s.keys, s.values, s.starts, s.ctx, s.d**-0.5, window)
    none = torch.tensor(weight.sum(-1) == 0, device=out.device)
    assert not out[none].any()
    s.check(out, window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("columns,window", [(0, 5), (1, 1), (1, 40), (7, 100), (9, 33), (100, 1500)])
def test_windows_over_a_table_narrower_than_the_context(dev, dtype, new, columns, window):
    """A window that begins past the table's last column, and one that ends past it: single tokens and
    prompts, whole and in parts, contexts just past the table and far past it."""
    room = 16 * columns
    for ctx in (room + 1, room + window - 1, room + window, room + window + 1, room + window + new, room + window + new + 17,
                room + 5000, 1 << 30):
        s = Setup(dev, [max(room, new) + 40, 90], [new, 1], 8, 2, 64, 16, dtype, seed=columns)
        s.ctx = [max(ctx, new), 90]
        narrow(s, columns)
        check_unseen(s, s.attend(window=window), window)


def test_a_plan_that_outgrew_its_table(dev):
    """The plan gives contexts past a narrow table; attention sees the tokens that the table has."""
    s = Setup(dev, [48, 20], [1, 1], 4, 2, 64, 16, torch.bfloat16)
    narrow(s, 2)
    ring, state = paging.free_pages(8, dev)
    s.tables = s.tables.contiguous()
    p = paging.plan_step(ring, state, s.tables, i32([47, 19], dev), i32([1, 1], dev), page_size=16, tokens=2)
    assert p.context_lens.tolist() == [48, 20] and p.slots[0] == -1
    out = kv4.attend(s.q, s.cache, 0, s.tables, p.query_starts, p.context_lens, window=10)
    check_unseen(s, out, 10)
    assert not out[0].any() and out[1].any()
