"""How attention over the 4-bit cache shares its work out: many requests, prompts beside long
contexts, parts of one tile's tokens and their joins, streams and graphs; and the example that runs
plan, rotary, cache and attention together.  Bounds as in ``test_gpu_attention``."""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from mrun_pub_amd import kv4
from test_gpu_attention import DTYPES, Setup, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,most,hq,hkv,d", [(63, 500, 4, 2, 64), (64, 500, 4, 2, 64), (70, 900, 6, 1, 128), (300, 200, 2, 1, 64),
                                             (1030, 40, 1, 1, 64)])
def test_many_requests(dev, B, most, hq, hkv, d):
    """Up to 63 requests are planned by single waves, more by blocks, thousands not at all."""
    rng = np.random.default_rng(B)
    ctx = rng.integers(1, most + 1, B).tolist()
    ctx[B // 2] = 3 * most  # one that is much longer
    s = Setup(dev, ctx, [1] * B, hq, hkv, d, 16, torch.bfloat16, seed=B)
    s.check(s.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 8, 64), (5, 1, 64), (4, 2, 256)])
@pytest.mark.parametrize("window", [None, 700])
def test_prompts_beside_long_contexts(dev, dtype, hq, hkv, d, window):
    ctx, new = [3000, 90, 2500, 17, 0, 1400], [1, 90, 60, 2, 0, 9]
    s = Setup(dev, ctx, new, hq, hkv, d, 32, dtype, seed=hq + d)
    s.check(s.attend(window=window), window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,P", [(64, 16), (128, 64), (256, 128)])
def test_a_chunk_at_the_end_of_a_long_context(dev, dtype, d, P):
    """One or two tiles of rows whose tokens are cut into parts; pages that end inside a tile."""
    s = Setup(dev, [6007], [21], 16, 2, d, P, dtype, seed=d)
    s.check(s.attend())
    s.check(s.attend(window=2500), window=2500)


def test_parts_with_missing_pages(dev):
    s = Setup(dev, [4000, 2000], [40, 1], 8, 1, 128, 16, torch.bfloat16, seed=3)
    for b, cols in ((0, range(3, 200, 7)), (0, range(120, 140)), (1, range(0, 60))):
        for col in cols:
            s.tables[b, col] = -1
            for x in (s.keys, s.values):
                x[b][16 * col: 16 * col + 16] = np.nan
    out = s.attend()
    for x in s.values:
        x[np.isnan(x)] = 0
    s.check(out)


@pytest.mark.parametrize("B", [1, 2])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_padding_after_prompts(dev, B, dtype):
    s = Setup(dev, [200, 90][:B], [150, 40][:B], 4, 1, 64, 16, dtype, seed=B)
    q = torch.cat([s.q, torch.full((77, 4, 64), float("nan"), device=dev, dtype=dtype)])
    n = s.q.shape[0]
    out = s.attend(q)
    assert torch.equal(out[:n], s.attend()) and not out[n:].any()
    s.check(out[:n])


def test_wrong_bounds_of_long_contexts(dev):
    s = Setup(dev, [3000, 40, 900], [70, 1, 33], 4, 1, 128, 16, torch.float16, seed=5)
    for kw in ({"max_query": 1, "max_context": 1}, {"max_query": 1, "max_context": 10**6}, {"max_query": None, "max_context": 1},
               {"max_query": 0, "max_context": 0}):
        s.check(s.attend(**kw))


def test_calls_on_two_streams_at_once(dev):
    """Each stream joins its parts in a workspace of its own."""
    a = Setup(dev, [9000, 5000], [1, 1], 8, 2, 128, 16, torch.bfloat16, seed=6)
    b = Setup(dev, [7000, 300], [40, 2], 8, 2, 128, 16, torch.bfloat16, seed=7)
    want_a, want_b = a.attend(), b.attend()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(one):
            got.append((a.attend(), want_a))
            got.append((b.attend(), want_b))
        with torch.cuda.stream(two):
            got.append((b.attend(), want_b))
            got.append((a.attend(), want_a))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)


def test_parts_in_a_graph_beside_eager_calls(dev):
    s = Setup(dev, [9000, 5000, 33], [1, 70, 1], 8, 2, 128, 16, torch.bfloat16, seed=8)
    other = Setup(dev, [4000], [3], 8, 2, 128, 16, torch.bfloat16, seed=9)
    want, want_other = s.attend(), other.attend()
    starts, ctx = i32(s.starts, dev), i32(s.ctx, dev)
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(s.q)
    with torch.cuda.graph(graph):
        kv4.attend(s.q, s.cache, 0, s.tables, starts, ctx, max_query=70, max_context=9000, out=out)
    for _ in range(5):
        out.zero_()
        graph.replay()
        assert torch.equal(other.attend(), want_other)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(s.attend(), want)


def test_unequal_values_and_one_token(dev):
    """A row that sees one token gives its value: exactly in fp32 but for one rounding of code * s + lo."""
    s = Setup(dev, [1, 300], [1, 300], 8, 2, 128, 16, torch.float32, seed=10)
    out = s.attend(window=1).cpu().numpy()
    for b in range(2):
        for i in range(s.new[b]):
            want = np.repeat(s.values[b][s.ctx[b] - s.new[b] + i], 4, 0)
            assert (abs(out[s.starts[b] + i] - want) <= 2.0**-23 * abs(want)).all()


def test_the_example(dev):
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import attention_step

    prompts, steps = [70, 16, 1], 5
    outputs, batch, cache = attention_step.run(prompts, steps)
    assert [list(o.shape) for o in outputs] == [[87, attention_step.HIDDEN]] + [[3, attention_step.HIDDEN]] * steps
    assert all(torch.isfinite(o).all() for o in outputs)
    assert batch.lens.tolist() == [75, 21, 6]
    taken = 5 + 2 + 1
    assert batch.pool.tolist() == [taken, batch.pages, 0]
    batch.finish()
    assert batch.pool.tolist() == [taken, batch.pages + taken, 0]
    again, _, cache2 = attention_step.run(prompts, steps)
    assert all(torch.equal(a, b) for a, b in zip(outputs, again)) and torch.equal(cache.storage, cache2.storage)
