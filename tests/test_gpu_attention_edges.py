"""Attention, its cache, rotary positions and paging at the edges of what their calls allow, on the GPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mrun_pub_amd import kv4, paging, rotary
from oracle import attention as oa
from test_gpu_attention import HALF, TINY, Setup, f64, i32

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


@pytest.mark.parametrize("hq,hkv,d,ctx,new", [(8, 4, 64, 1300, 200), (8, 4, 64, 4000, 70), (4, 2, 128, 2200, 100), (4, 2, 128, 300, 300), (4, 2, 64, 700, 700),
                                              (8, 2, 64, 5000, 1), (8, 2, 128, 9000, 3), (4, 1, 256, 3000, 9)])
def test_fp32_attention_is_as_exact_as_the_plain_form(dev, hq, hkv, d, ctx, new):
    """Against 64 bits, in the 2-norm: twice what the plain form in fp32 is off, and what n / 16 roundings
    of a sum that runs over n tokens, 16 at a time, add to it: each at most 2^-24 of the sum, of no
    common sign, so sqrt(n / 16) of them.  Codes and lowest values, whose sums cancel, add nothing."""
    s = Setup(dev, [ctx], [new], hq, hkv, d, 16, torch.float32, seed=ctx)
    out = f64(s.attend())
    q, k, v = f64(s.q), s.keys[0], s.values[0]
    want, _, _ = oa.attend(q, s.keys, s.values, s.starts, s.ctx, d**-0.5)
    plain = np.zeros_like(want)
    for i in range(new):
        n = ctx - new + i + 1
        for h in range(hq):
            kh, vh = (x[:n, h // (hq // hkv)].astype(np.float32) for x in (k, v))
            x = kh @ q[i, h].astype(np.float32) * np.float32(d**-0.5)
            w = np.exp(x - x.max())
            plain[i, h] = (w @ vh) / w.sum()
    size = np.linalg.norm(want)
    off, plain_off = np.linalg.norm(out - want) / size, np.linalg.norm(plain - want) / size
    print(f"off by {off:.2e}, the plain form by {plain_off:.2e}")
    assert off <= 2 * plain_off + (ctx / 16) ** 0.5 * 2.0**-24


def test_strides_of_dimensions_of_one_do_not_matter(dev):
    """One token, one head or one column: its stride is never used, whatever it is."""
    s = Setup(dev, [40], [1], 4, 1, 64, 16, torch.bfloat16)
    want, pos, spec = s.attend(), i32([39], dev), rotary.RotarySpec(64)
    turned = rotary.apply_rotary(s.q, pos, spec)
    flat = torch.zeros(4 * 64 + 8, device=dev, dtype=torch.bfloat16)
    flat[:256] = s.q.flatten()
    q = flat.as_strided((1, 4, 64), (4 * 64 + 3, 64, 1))
    assert torch.equal(s.attend(q), want)
    into = torch.zeros_like(flat)
    rotary.apply_rotary(q, pos, spec, out=into.as_strided((1, 4, 64), (259, 64, 1)))
    assert torch.equal(into[:256], turned.flatten()) and not into[256:].any()
    k = s.k[:1].as_strided((1, 1, 64), (67, 65, 1))
    a, b = (kv4.KV4Cache(layers=1, kv_heads=1, head_dim=64, pages=1, page_size=16, device=dev) for _ in range(2))
    slot = torch.tensor([3], device=dev)
    out = kv4.append(a, 0, k, k, slot, q=q, positions=pos, rotary=spec)
    assert torch.equal(out, turned)
    kv4.append(b, 0, s.k[:1], s.k[:1], slot, positions=pos, rotary=spec)
    assert torch.equal(a.storage, b.storage)

    s = Setup(dev, [9, 5], [1, 1], 4, 1, 64, 16, torch.bfloat16)
    narrow(s, 1)
    want = s.attend()
    s.tables = torch.stack([s.tables[:, 0], s.tables[:, 0]], 1).contiguous().as_strided((2, 1), (2, 7))
    assert torch.equal(s.attend(), want)
    ring, state = paging.free_pages(4, dev)
    new = i32([1, 1], dev)
    plans = [paging.plan_step(ring, state, t, i32([0, 0], dev), new, page_size=16, tokens=2)
             for t in (torch.full((2, 1), -1, dtype=torch.int32, device=dev),
                       torch.full((2, 2), -1, dtype=torch.int32, device=dev).as_strided((2, 1), (2, 5)))]
    assert all(torch.equal(x, y) for x, y in zip(*plans))
    done = torch.ones(2, dtype=torch.bool, device=dev)
    held = torch.zeros(2, 2, dtype=torch.int32, device=dev).as_strided((2, 1), (2, 5))
    assert paging.release_pages(ring, plans[0].free_state, held, new, done, page_size=16).tolist() == [2, 6, 0]


def test_more_tokens_than_one_grid_has_blocks(dev):
    """A grid has fewer than 2^32 threads: 2^24 blocks of 256, of a token each, are more than one launch."""
    t, spec = (1 << 24) + 5, rotary.RotarySpec(2)
    some = torch.tensor([0, 1, 77, t // 2, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, t - 2, t - 1], device=dev)
    x = torch.empty(t, 1, 130, device=dev, dtype=torch.bfloat16).normal_()
    pos = torch.arange(t, device=dev, dtype=torch.int32) % 1000
    y = rotary.apply_rotary(x, pos, spec)
    assert torch.equal(y[some], rotary.apply_rotary(x[some], pos[some], spec))
    del y
    k = x.view(-1)[: t * 64].view(t, 1, 64)
    cache, few = (kv4.KV4Cache(layers=1, kv_heads=1, head_dim=64, pages=n, page_size=256, device=dev) for n in ((t + 255) // 256, 1))
    spec = rotary.RotarySpec(64)
    kv4.append(cache, 0, k, k, torch.arange(t, device=dev), positions=pos, rotary=spec)
    at = torch.arange(len(some), device=dev)
    kv4.append(few, 0, k[some], k[some], at, positions=pos[some], rotary=spec)
    for got, want in zip(kv4.read(cache, 0, some), kv4.read(few, 0, at)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,size,scale", [(torch.bfloat16, 1e-30, 1e-30), (torch.bfloat16, 2.0**-133, 1e-45),
                                              (torch.float16, 2.0**-24, 1e-45), (torch.float32, 1e-45, 1e-45),
                                              (torch.bfloat16, 0.0, 3e38), (torch.float16, 0.0, 3e38), (torch.float32, 0.0, 3e38)])
@pytest.mark.parametrize("new", [1, 40])
def test_scores_of_zero_weigh_all_tokens_alike(dev, new, dtype, size, scale):
    """Scores that are zero or far below a weight's step, from tiny queries and scales or from zeros at
    the largest scale: every visible token has the same weight, and hidden ones none."""
    s = Setup(dev, [77], [new], 8, 2, 64, 16, dtype, seed=new)
    s.q = torch.full_like(s.q, size)
    out = s.attend(scale=scale)
    s.q.zero_()
    s.check(out)


@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd_takes_the_inverse_turn_as_the_gradient(dev, layout, dtype):
    spec = rotary.RotarySpec(32, layout=layout, scaling={"type": "yarn", "factor": 4.0, "original": 64})
    x, g = (torch.randn(5, 3, 48, device=dev).to(dtype) for _ in range(2))
    pos = paging.plan_step(*paging.free_pages(4, dev), torch.zeros(1, 4, dtype=torch.int32, device=dev), i32([7], dev), i32([5], dev),
                           page_size=16, tokens=5).positions  # an inference tensor
    back = rotary.apply_rotary(g, pos, spec, inverse=True)
    for inverse, want in ((False, back), (True, rotary.apply_rotary(g, pos, spec))):
        leaf = x.clone().requires_grad_()
        y = rotary.apply_rotary(leaf * 2, pos, spec, inverse=inverse)
        assert torch.equal(y.detach(), rotary.apply_rotary(x * 2, pos, spec, inverse=inverse))
        y.backward(g)
        assert torch.equal(leaf.grad, want * 2)
    leaf = x.clone().requires_grad_()
    (wide,) = torch.autograd.grad(rotary.apply_rotary(leaf, pos, spec).sum(), leaf)  # a broadcast gradient
    assert torch.equal(wide, rotary.apply_rotary(torch.ones_like(x), pos, spec, inverse=True))
    with torch.no_grad():
        assert not rotary.apply_rotary(leaf, pos, spec).requires_grad
    with pytest.raises(ValueError, match="gradient"):
        rotary.apply_rotary(leaf, pos, spec, out=torch.empty_like(x))


def sizes(x):
    """Of cached values [n, h, d]: the largest code * s and |lo| that their groups' sums can hold, a value each."""
    g = x.reshape(*x.shape[:-1], -1, 64)
    top = (g.max(-1) - g.min(-1)) * 1.01 + abs(g).max(-1)  # codes 0 and 15 are not always there
    return np.repeat(top, 64, -1)


@pytest.mark.parametrize("hq,hkv,d,ctx,new", [(8, 2, 128, 3, 3), (4, 1, 64, 12, 1), (8, 2, 128, 20, 20), (4, 4, 64, 40, 40), (4, 1, 256, 9, 5),
                                              (4, 1, 256, 33, 12)])
def test_fp16_attention_multiplies_exact_codes(dev, hq, hkv, d, ctx, new):
    """Queries of zero give the mean of the values: weights of 1, scales of 11 bits in two bf16 parts and
    codes are exact, so fp16 results are off by their own rounding and by fp32 sums.  Values rounded to
    fp16, or weights to one bf16 part, would be off by more."""
    s = Setup(dev, [ctx], [new], hq, hkv, d, 16, torch.float16, seed=ctx + d)
    out, v = f64(s.attend(torch.zeros_like(s.q))), s.values[0]
    _, sc, lo = oa.kv4_quantize(v.astype(np.float32))
    one = torch.tensor(sc.astype(np.float32)).bfloat16().double().numpy()  # a scale's first part
    sc, lo, one = (np.repeat(x.astype(np.float64), 64, -1) for x in (sc, lo, one))
    zero = np.zeros(s.q.shape)

    def mean(x):
        return oa.attend(zero, s.keys, [x], s.starts, s.ctx, 1.0)[0]

    want, half = mean(v), HALF[torch.float16]
    bound = half * abs(want) + (ctx + 8) * 2.0**-24 * mean(15 * sc + abs(lo)) + TINY[torch.float16]
    assert (abs(out - want) <= bound).all()
    for other in (v.astype(np.float16).astype(np.float64), (v - lo) * one / sc + lo):  # the bound tells these apart
        assert (abs(mean(other) - want) > bound).any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctx,new", [(8, 1), (8, 8), (40, 5), (40, 40), (300, 1), (300, 90)])
def test_fp16_scores_use_exact_keys(dev, d, ctx, new):
    """At a scale of 1 scores are large, and their errors show: in fp32 sums of terms of some 700 they are
    about 2^-15, which beside the result's own rounding (0.29 of 2^-10 in the 2-norm) adds a hundredth
    to it.  Keys rounded to fp16 would add more than half."""
    s = Setup(dev, [ctx], [new], 8, 2, d, 16, torch.float16, seed=ctx + d)
    out, q = f64(s.attend(scale=1.0)), f64(s.q)
    want, _, _ = oa.attend(q, s.keys, s.values, s.starts, s.ctx, 1.0)
    own = np.linalg.norm(want.astype(np.float16) - want)
    assert np.linalg.norm(out - want) <= 1.1 * own
    if new > 1:  # one token's rows are too few for the norms to tell
        other, _, _ = oa.attend(q, [s.keys[0].astype(np.float16).astype(np.float64)], s.values, s.starts, s.ctx, 1.0)
        assert np.linalg.norm(other.astype(np.float16) - want) > 1.5 * own


@pytest.mark.parametrize("hq", [2, 80])
def test_fp16_rows_that_see_one_token(dev, hq):
    """They give its value rounded to fp16 once: a weight of 1 times a scale of 11 bits is exact in two parts."""
    s = Setup(dev, [1, 300], [1, 300], hq, 2, 128, 16, torch.float16, seed=11)
    out = f64(s.attend(window=1))
    for b in range(2):
        v = s.values[b][s.ctx[b] - s.new[b]:]
        want, size = (np.repeat(x, hq // 2, 1) for x in (v, sizes(v)))
        got = out[s.starts[b]: s.starts[b + 1]]
        assert (abs(got - want) <= HALF[torch.float16] * abs(want) + 2.0**-23 * size + TINY[torch.float16]).all()


@pytest.mark.parametrize("groups", [((4, 1280, 5300), (6, 1280, 1280)), ((40, 128, 5300), (60, 128, 1280)), ((3, 1000, 9000), (1, 3000, 3000))])
def test_more_parts_than_places(dev, groups):
    """Prompts of unequal contexts whose tiles alone are more than the blocks that run at once: cut tiles
    have a place for each part or are cut less.  Results as without parts, each off by the roundings of
    sums over its tokens."""
    new, ctx = (sum(([g[i]] * g[0] for g in groups), []) for i in (1, 2))
    d, P = 64, 64
    count = [-(-c // P) for c in ctx]
    cache = kv4.KV4Cache(layers=1, kv_heads=8, head_dim=d, pages=sum(count), page_size=P, device=dev)
    tables = torch.full((len(ctx), max(count)), -1, dtype=torch.int32, device=dev)
    order, at = torch.randperm(sum(count), device=dev).int(), 0
    for b, n in enumerate(count):
        tables[b, :n] = order[at: at + n]
        at += n
    k, v = (torch.randn(cache.pages * P, 8, d, device=dev) for _ in range(2))
    kv4.append(cache, 0, k, v, torch.arange(cache.pages * P, device=dev))
    q = torch.randn(sum(new), 8, d, device=dev)
    args = (q, cache, 0, tables, i32(np.cumsum([0] + new), dev), i32(ctx, dev))
    want = kv4.attend(*args, max_query=max(new), max_context=1).double()  # no parts
    for _ in range(2):
        got = kv4.attend(*args, max_query=max(new), max_context=max(ctx))
        assert float((got - want).norm() / want.norm()) <= 2 * (max(ctx) / 16) ** 0.5 * 2.0**-24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_contexts_of_few_tokens_beside_prompts(dev, dtype, d):
    """Contexts past 8192: requests of few rows are cut into parts in a launch of their own, whose blocks
    their number bounds; rows of padding after them are either kernel's."""
    s = Setup(dev, [300, 9001, 70, 12000], [150, 1, 70, 8], 4, 1, d, 64, dtype, seed=d)
    s.check(s.attend())
    s.check(s.attend(window=8500), window=8500)
    for pad in (3, 200):
        out = s.attend(torch.cat([s.q, torch.full((pad, 4, d), float("nan"), device=dev, dtype=dtype)]))
        assert not out[len(s.q):].any()
        s.check(out[: len(s.q)])


@pytest.mark.parametrize("B,new,ctx", [(6, 1, 5000), (6, 60, 5000), (70, 1, 3000), (70, 40, 3000)])
def test_starts_that_decrease_leave_later_calls_alone(dev, B, new, ctx):
    """Such starts are a caller's mistake that only the GPU sees.  Nothing is read or written out of
    place for them, and what calls share, the counters of finished parts, is as it was."""
    s = Setup(dev, [ctx] + [200] * (B - 1), [new] * B, 4, 1, 64, 16, torch.bfloat16, seed=B)
    want = s.attend()
    starts = s.starts.copy()
    starts[1:-1:2] = starts[-1]  # every other request has all rows, the next ones none
    out = torch.zeros_like(s.q)
    kv4.attend(s.q, s.cache, 0, s.tables, i32(starts, dev), i32(s.ctx, dev), max_query=new, max_context=ctx, out=out)
    assert torch.equal(s.attend(), want)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device_than_the_current_one(dev):
    """Calls run on their tensors' device, on its current stream, whatever the current device is; a tile
    of 68 KB of LDS (fp32 prompts, heads of 128) is allowed on each."""
    outs = []
    for at in (torch.device("cuda:0"), torch.device("cuda:1")):
        with torch.cuda.device(0):
            s = Setup(dev, [300, 40], [200, 1], 4, 2, 128, 16, torch.float32, seed=1)
            cache = kv4.KV4Cache(layers=1, kv_heads=2, head_dim=128, pages=s.cache.pages, page_size=16, device=at)
            k, v, slots = s.k.to(at), s.v.to(at), torch.tensor(np.concatenate(s.slots), device=at)
            spec, pos = rotary.RotarySpec(128), torch.arange(340, device=at)
            kv4.append(cache, 0, rotary.apply_rotary(k, pos, spec), v, slots)
            out = kv4.attend(s.q.to(at), cache, 0, s.tables.to(at), i32(s.starts, at), i32(s.ctx, at), max_query=200)
            ring, state = paging.free_pages(8, at)
            p = paging.plan_step(ring, state, torch.full((1, 4), -1, dtype=torch.int32, device=at), i32([0], at), i32([9], at),
                                 page_size=16, tokens=9)
            freed = paging.release_pages(ring, p.free_state, torch.zeros(1, 4, dtype=torch.int32, device=at), i32([9], at),
                                         torch.ones(1, dtype=torch.bool, device=at), page_size=16)
            outs.append([x.cpu() for x in (out, *kv4.read(cache, 0, slots), *p, freed)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
