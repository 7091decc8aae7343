"""Rotary positions, paging plans, the 4-bit KV cache and attention over it, on the GPU, against the
plain forms in 64 bits (``oracle.attention``)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from mrun_pub_amd import kv4, paging, rotary
from oracle import attention as oa

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a step, relative
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0**-25}  # half fp16's subnormal step
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def f64(t):
    return t.detach().double().cpu().numpy()


def i32(v, dev):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)


# ---- rotary ----------------------------------------------------------------------------------


def check_rotary(y, x, pos, spec, inverse=False):
    freq, mag = oa.rotary_frequencies(spec.dim, spec.base, spec.scaling)
    want, size = oa.rotary(f64(x), f64(pos), freq, mag, spec.layout, inverse)
    # cos and sin, the products and the sum are each off by half a step of fp32; the result by one of its type
    bound = HALF[x.dtype] * abs(want) + (3 + 1e-2) * 2.0**-24 * size * (1 + 2 * HALF[x.dtype]) + TINY[x.dtype]
    assert (abs(f64(y) - want) <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("t,h,d,rot", [(1, 1, 64, 64), (1, 12, 128, 128), (17, 5, 128, 64), (33, 3, 96, 48), (5, 7, 80, 20),
                                       (3, 2, 66, 2), (300, 40, 128, 128), (2, 3, 256, 256), (7, 1, 130, 130)])
def test_rotary(dev, dtype, layout, t, h, d, rot):
    g = torch.Generator(device=dev).manual_seed(t * d + rot)
    x = torch.randn(t, h, d, device=dev, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (t,), device=dev, generator=g)
    spec = rotary.RotarySpec(rot, layout=layout)
    y = rotary.apply_rotary(x, pos, spec)
    check_rotary(y, x, pos, spec)
    back = rotary.apply_rotary(x, pos, spec, inverse=True)
    check_rotary(back, x, pos, spec, inverse=True)
    assert torch.equal(y[..., rot:], x[..., rot:])
    z = x.clone()
    assert torch.equal(rotary.apply_rotary(z, pos, spec, out=z), y) and torch.equal(z, y)


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 4.0},
                                     {"type": "yarn", "factor": 8.0, "original": 4096}])
def test_rotary_far_positions_and_scalings(dev, scaling):
    x = torch.randn(6, 2, 128, device=dev)
    pos = i32([0, 1, 131071, 10**6 + 1, 2**30 + 7, 2**31 - 1], dev)
    for layout in rotary.LAYOUTS:
        spec = rotary.RotarySpec(128, base=1e6, layout=layout, scaling=scaling)
        check_rotary(rotary.apply_rotary(x, pos, spec), x, pos, spec)


def test_rotary_strides_and_empty(dev):
    spec = rotary.RotarySpec(64)
    qkv = torch.randn(9, 7, 64, device=dev).to(torch.bfloat16)
    pos = torch.arange(9, device=dev)
    part = qkv[:, 2:5]
    assert torch.equal(rotary.apply_rotary(part, pos, spec), rotary.apply_rotary(part.contiguous(), pos, spec))
    odd = torch.randn(9, 3, 67, device=dev).to(torch.bfloat16)[..., 1:65]  # no alignment
    assert torch.equal(rotary.apply_rotary(odd, pos, spec), rotary.apply_rotary(odd.contiguous(), pos, spec))
    turned = torch.randn(3, 64, 9, device=dev).to(torch.bfloat16).permute(2, 0, 1)
    assert torch.equal(rotary.apply_rotary(turned, pos, spec), rotary.apply_rotary(turned.contiguous(), pos, spec))
    into = torch.zeros(9, 5, 64, device=dev, dtype=torch.bfloat16)
    rotary.apply_rotary(part, pos, spec, out=into[:, 1:4])
    assert torch.equal(into[:, 1:4], rotary.apply_rotary(part, pos, spec))
    assert (into[:, 0] == 0).all() and (into[:, 4] == 0).all()
    assert rotary.apply_rotary(part[:0], pos[:0], spec).shape == (0, 3, 64)


def test_rotary_gradient_against_differences(dev):
    """Central differences of sum(g * rotary(x)) in fp32: the map is linear, so the difference is exact
    but for rounding: half a step of x + e, of the result, and of the sum over the head."""
    spec = rotary.RotarySpec(32, layout="interleaved")
    x, g = (torch.randn(2, 1, 32, device=dev) for _ in range(2))
    pos = i32([3, 900], dev)
    grad = rotary.apply_rotary(g, pos, spec, inverse=True)
    for d in (0, 1, 30, 31):
        for t in (0, 1):
            up, down = x.clone(), x.clone()
            up[t, 0, d] += 1.0
            down[t, 0, d] -= 1.0
            diff = ((rotary.apply_rotary(up, pos, spec).double() - rotary.apply_rotary(down, pos, spec).double()) * g.double()).sum() / 2
            size = float((abs(x) + 1).max() * abs(g).sum())
            assert abs(float(diff) - float(grad[t, 0, d])) <= 8 * 2.0**-24 * size


# ---- paging ----------------------------------------------------------------------------------


def run_plan(dev, past, new, P, width, tokens, avail, ring_size, head=0, seed=0):
    rng = np.random.default_rng(seed)
    B = len(past)
    order = rng.permutation(ring_size).astype(np.int32)
    tables = rng.integers(0, ring_size, (B, width)).astype(np.int32)  # unused columns hold anything
    state = np.array([head, head + avail, 5], np.int64)
    want = oa.plan_step(order, state, tables, past, new, P, tokens)
    t = torch.tensor(tables, device=dev)
    ring, st = torch.tensor(order, device=dev), torch.tensor(state, device=dev)
    for _ in range(2):  # the same step again gives the same
        p = paging.plan_step(ring, st, t, i32(past, dev), torch.tensor(new, device=dev), page_size=P, tokens=tokens)
        got = [t, p.slots, p.positions, p.requests, p.query_starts, p.context_lens, p.free_state]
        for a, b in zip(got, want):
            assert np.array_equal(a.cpu().numpy(), b)
    assert np.array_equal(ring.cpu().numpy(), order) and np.array_equal(st.cpu().numpy(), state)


@pytest.mark.parametrize("P", [1, 16, 64])
@pytest.mark.parametrize("B,most_past,most_new", [(1, 0, 1), (7, 100, 1), (64, 300, 9), (257, 90, 3), (700, 50, 0), (5, 10, 3000)])
def test_plan(dev, P, B, most_past, most_new):
    rng = np.random.default_rng(B + P)
    past, new = rng.integers(0, most_past + 1, B), rng.integers(0, most_new + 1, B)
    need = int(sum(-(-(p + n) // P) - -(-p // P) for p, n in zip(past, new)))
    width = int(max(-(-(p + n) // P) for p, n in zip(past, new))) + 1
    total = int(new.sum())
    size = need + 9
    run_plan(dev, past, new, P, width, total, need + 3, size)  # enough pages
    run_plan(dev, past, new, P, width, total + 5, need + 9, size, head=10**12 + size - 2, seed=1)  # padding, a wrapped ring
    run_plan(dev, past, new, P, width, total, max(0, need - 2), size, seed=2)  # too few
    run_plan(dev, past, new, P, max(1, width - 2), total, need, size, seed=3)  # a narrow table
    run_plan(dev, past, new, P, width, max(0, total - 3), need, size, seed=4)  # fewer rows than tokens


def test_plan_edges(dev):
    run_plan(dev, [-3, 5], [2, -1], 16, 2, 2, 4, 8)  # negative lengths count as none
    run_plan(dev, [0, 0], [0, 0], 16, 2, 0, 4, 8)
    run_plan(dev, [3], [1], 16, 1, 1, -4, 8)  # a tail before the head: no pages
    run_plan(dev, [15, 16, 17, 31, 32], [1, 1, 1, 1, 1], 16, 3, 5, 8, 8)
    ring, state = paging.free_pages(8, dev)
    empty = torch.zeros(0, dtype=torch.int32, device=dev)
    p = paging.plan_step(ring, state, torch.zeros(0, 4, dtype=torch.int32, device=dev), empty, empty, page_size=16, tokens=3)
    assert p.slots.tolist() == [-1] * 3 and p.query_starts.tolist() == [0] and p.free_state.tolist() == [0, 8, 0]


@pytest.mark.parametrize("B,P,most", [(1, 16, 40), (9, 16, 600), (300, 32, 100), (2, 16, 9000)])
def test_release(dev, B, P, most):
    rng = np.random.default_rng(B)
    lens = rng.integers(0, most + 1, B)
    width = int(max(-(-lens // P)))
    width = max(1, width - 1) if B == 9 else width + 1
    tables = rng.integers(-1, 5000, (B, width)).astype(np.int32)
    done = rng.random(B) < 0.6
    size = int(B * width + 3)
    order, state = np.full(size, -7, np.int32), np.array([5, size - 2, 1], np.int64)
    ring_w, state_w = oa.release_pages(order, state, tables, lens, done, P)
    ring = torch.tensor(order, device=dev)
    got = paging.release_pages(ring, torch.tensor(state, device=dev), torch.tensor(tables, device=dev), i32(lens, dev),
                               torch.tensor(done, device=dev), page_size=P)
    assert np.array_equal(ring.cpu().numpy(), ring_w) and np.array_equal(got.cpu().numpy(), state_w)


# ---- the cache ---------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,h,d,P", [(1, 1, 64, 16), (5, 2, 128, 16), (37, 3, 256, 32), (70, 8, 128, 64), (3, 1, 128, 256)])
def test_append_and_read(dev, dtype, t, h, d, P):
    g = torch.Generator(device=dev).manual_seed(t + d)
    k, v = ((torch.randn(t, h, d, device=dev, generator=g) * 10.0 ** torch.empty(t, 1, 1, device=dev).uniform_(-4, 3, generator=g)).to(dtype)
            for _ in range(2))
    pages = -(-t // P) + 1
    cache = kv4.KV4Cache(layers=2, kv_heads=h, head_dim=d, pages=pages, page_size=P, device=dev)
    slots = torch.randperm(pages * P, device=dev, generator=g)[:t]
    assert kv4.append(cache, 1, k, v, slots) is None
    kr, vr = kv4.read(cache, 1, slots)
    for x, r in ((k, kr), (v, vr)):
        want = oa.kv4_values(*oa.kv4_quantize(x.float().cpu().numpy()))
        assert np.array_equal(r.cpu().numpy(), want)
    assert not cache.storage[0].any()
    left = torch.ones(pages * P, dtype=torch.bool, device=dev)
    left[slots] = False
    other = left.nonzero().flatten()
    for x in kv4.read(cache, 1, other):
        assert not x.any()  # no other slot was written
    k16, v16 = kv4.read(cache, 1, slots.to(torch.int32), dtype=torch.float16)
    assert torch.equal(k16, kr.half()) and torch.equal(v16, vr.half())
    # again, over what is there: only the new values are left
    kv4.append(cache, 1, v, k, slots)
    k2, v2 = kv4.read(cache, 1, slots)
    assert torch.equal(k2, vr) and torch.equal(v2, kr)


def test_append_special_values_and_padding(dev):
    k = torch.zeros(6, 1, 64, device=dev)
    k[1] = 3.25
    k[2, 0, :3] = torch.tensor([float("nan"), float("inf"), -float("inf")], device=dev)
    k[3, 0, 7] = 1e38
    k[4] = torch.randn(64, device=dev) * 1e-7  # a scale below fp16's smallest
    cache = kv4.KV4Cache(layers=1, kv_heads=1, head_dim=64, pages=1, page_size=16, device=dev)
    slots = torch.tensor([0, 1, 2, 3, 4, -1], device=dev)
    kv4.append(cache, 0, k, -k, slots)
    kr, vr = kv4.read(cache, 0, torch.tensor([0, 1, 2, 3, 4, -1, 16, 5], device=dev))
    assert np.array_equal(kr[:5].cpu().numpy(), oa.kv4_values(*oa.kv4_quantize(k[:5].cpu().numpy())))
    assert np.array_equal(vr[:5].cpu().numpy(), oa.kv4_values(*oa.kv4_quantize(-k[:5].cpu().numpy())))
    assert torch.isfinite(kr).all() and not kr[5:].any() and not vr[5:].any()
    before = cache.storage.clone()
    kv4.append(cache, 0, k[:4], k[:4], torch.tensor([-1, 16, 1 << 40, -(1 << 40)], device=dev))
    kv4.append(cache, 0, k[:0], k[:0], slots[:0])
    assert torch.equal(before, cache.storage)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("hq,hkv,d,rot", [(4, 2, 128, 128), (3, 1, 64, 32), (16, 8, 64, 64), (6, 3, 256, 256), (5, 5, 128, 8)])
def test_append_turns_as_apply_rotary(dev, dtype, layout, hq, hkv, d, rot):
    t = 21
    spec = rotary.RotarySpec(rot, base=1e6, layout=layout, scaling={"type": "yarn", "factor": 4.0, "original": 2048})
    qkv = torch.randn(t, hq + 2 * hkv, d, device=dev).to(dtype)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    pos = torch.randint(0, 100000, (t,), device=dev)
    a, b = (kv4.KV4Cache(layers=1, kv_heads=hkv, head_dim=d, pages=2, page_size=32, device=dev) for _ in range(2))
    slots = torch.randperm(64, device=dev)[:t]
    slots[3] = -1
    out = kv4.append(a, 0, k, v, slots, q=q, positions=pos, rotary=spec)
    assert torch.equal(out, rotary.apply_rotary(q, pos, spec))  # the padding row's queries too
    kv4.append(b, 0, rotary.apply_rotary(k, pos, spec), v.contiguous(), slots)
    assert torch.equal(a.storage, b.storage)
    kv4.append(b, 0, k.contiguous(), v, slots, positions=pos, rotary=spec)
    assert torch.equal(a.storage, b.storage)


def test_append_unaligned_views(dev):
    x = torch.randn(9, 2, 66, device=dev).half()[..., 1:65]
    flat = torch.randn(9 * 2 * 64 + 1, device=dev).half()[1:].view(9, 2, 64)
    a, b = (kv4.KV4Cache(layers=1, kv_heads=2, head_dim=64, pages=1, page_size=16, device=dev) for _ in range(2))
    slots = torch.arange(9, device=dev)
    kv4.append(a, 0, x, flat, slots)
    kv4.append(b, 0, x.contiguous(), flat.clone(), slots)
    assert torch.equal(a.storage, b.storage)


# ---- attention ---------------------------------------------------------------------------------


class Setup:
    """A cache whose requests' pages are scattered; slots that no token owns hold bytes of 0xff."""

    def __init__(self, dev, ctx, new, hq, hkv, d, P, dtype, seed=0, spare=2, size=1.0, pages=None):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=dev).manual_seed(seed)
        count = [-(-c // P) for c in ctx]
        need = sum(count) + spare
        self.cache = kv4.KV4Cache(layers=1, kv_heads=hkv, head_dim=d, pages=pages or need, page_size=P, device=dev)
        order = rng.permutation(pages or need)[: sum(count)]
        width = max(max(count), 1) + 1
        tables = np.full((len(ctx), width), -1, np.int32)
        at, slots = 0, []
        for b, c in enumerate(count):
            tables[b, :c] = order[at: at + c]
            at += c
            t = np.arange(ctx[b])
            slots.append(tables[b, t // P].astype(np.int64) * P + t % P)
        self.slots = slots
        if pages is None:
            self.cache.storage.fill_(255)
        every = torch.tensor(np.concatenate(slots), device=dev)
        n = int(every.numel())
        shift = 0.3 * torch.randn(hkv, d, device=dev, generator=g)
        self.k, self.v = ((torch.randn(n, hkv, d, device=dev, generator=g) * size + shift).to(dtype) for _ in range(2))
        kv4.append(self.cache, 0, self.k, self.v, every)
        kr, vr = kv4.read(self.cache, 0, every)
        split = np.cumsum([0] + list(ctx))
        self.keys = [kr[a:b].double().cpu().numpy() for a, b in zip(split[:-1], split[1:])]
        self.values = [vr[a:b].double().cpu().numpy() for a, b in zip(split[:-1], split[1:])]
        self.ctx, self.new = list(ctx), list(new)
        self.starts = np.cumsum([0] + list(new))
        self.tables = torch.tensor(tables, device=dev)
        self.q = (1.5 * torch.randn(int(self.starts[-1]), hq, d, device=dev, generator=g)).to(dtype)
        self.dev, self.d = dev, d

    def attend(self, q=None, **kw):
        kw.setdefault("max_query", max(self.new, default=0))
        kw.setdefault("max_context", max(self.ctx, default=0))
        return kv4.attend(self.q if q is None else q, self.cache, 0, self.tables, i32(self.starts, self.dev), i32(self.ctx, self.dev), **kw)

    def check(self, out, window=None, scale=None):
        q = f64(self.q)
        s = scale or self.d**-0.5
        want, weight, reach = oa.attend(q, self.keys, self.values, self.starts, self.ctx, s, window)
        n = max(self.ctx + [1])
        dt = self.q.dtype
        if dt == torch.float32:
            op, p = 2.0**-24, 2.0**-24  # a cache value's sum, a weight
        else:
            op, p = 2.0**-11, 2.0**-11  # a cache value and a weight in fp16; queries are exact to 2^-18 of their row's largest
        # a score: its keys' rounding, the queries', the sum over d in fp32, the scale's and maximum's
        score = reach * (op + 2.0**-18 * (dt == torch.bfloat16) * math.sqrt(self.d) + (self.d + 6) * 2.0**-24) + 2.0**-20
        # weights: 2^x of the score (its own step, 2^-22), rounded; values; sums over the tokens in fp32;
        # weights below fp16's normal range, each off by 2^-25 of the largest
        rel = 2 * score + p + op + 2.0**-21 + (n + 64) * 2.0**-24
        top = np.concatenate([abs(v).max((0, 2), initial=0.0)[None] for v in self.values] or [np.zeros((1, 1))]).max()
        tiny = n * 2.0**-25 * top * (dt != torch.float32)
        bound = rel * weight * 1.02 + tiny + HALF[dt] * (abs(want) + rel * weight) + TINY[dt]
        got = f64(out)
        assert np.isfinite(got).all()
        worst = (abs(got - want) - bound).max(initial=-1.0)
        assert worst <= 0, f"over the bound by {worst}"


SHAPES = [(1, 1, 64, 16), (12, 2, 128, 16), (16, 4, 128, 32), (16, 8, 64, 64), (34, 2, 64, 16), (3, 3, 128, 128), (8, 1, 256, 16),
          (40, 2, 256, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,P", SHAPES)
def test_attend_decode(dev, dtype, hq, hkv, d, P):
    ctx = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 513, 1000]
    s = Setup(dev, ctx, [1] * len(ctx), hq, hkv, d, P, dtype)
    s.check(s.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,P", SHAPES)
@pytest.mark.parametrize("window", [None, 1, 7, 40])
def test_attend_ragged(dev, dtype, hq, hkv, d, P, window):
    """Prompts, chunks, drafts, single tokens, requests without tokens, in one call."""
    ctx, new = [1, 40, 5, 0, 150, 33, 200, 64], [1, 40, 0, 0, 70, 3, 1, 17]
    s = Setup(dev, ctx, new, hq, hkv, d, P, dtype, seed=hq)
    s.check(s.attend(window=window), window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_prompts(dev, dtype, d):
    s = Setup(dev, [129, 301], [129, 257], 8, 2, d, 32, dtype, seed=d)
    s.check(s.attend())
    s.check(s.attend(window=100), window=100)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_split_contexts(dev, dtype):
    """Few rows over long contexts: split between blocks, some of which have nothing to do."""
    s = Setup(dev, [20011, 77, 4097], [2, 1, 5], 6, 2, 128, 64, dtype, seed=3)
    s.check(s.attend())
    s.check(s.attend(window=9000), window=9000)
    s.check(s.attend(scale=0.02), scale=0.02)


def test_attend_long_context(dev):
    s = Setup(dev, [131072], [1], 4, 1, 128, 128, torch.float16, seed=4)
    s.check(s.attend())


def test_attend_bounds_only_choose_the_split(dev):
    """Bounds that are too small, too large or absent: other splits, the same results."""
    s = Setup(dev, [700, 40, 90], [50, 1, 33], 12, 2, 128, 16, torch.bfloat16, seed=5)
    for kw in ({"max_query": 1, "max_context": 1}, {"max_query": None, "max_context": None}, {"max_query": 0, "max_context": 0},
               {"max_query": 10**6, "max_context": 10**6}, {"max_query": 1, "max_context": 10**5}):
        s.check(s.attend(**kw))


def test_attend_rows_of_padding_and_empty_calls(dev):
    s = Setup(dev, [20, 9], [3, 1], 4, 2, 64, 16, torch.bfloat16)
    q = torch.cat([s.q, torch.full((21, 4, 64), float("nan"), device=dev, dtype=torch.bfloat16)])
    out = s.attend(q)
    assert torch.equal(out[:4], s.attend()) and not out[4:].any()
    none = i32([], dev)
    out = kv4.attend(q, s.cache, 0, s.tables[:0], i32([0], dev), none)
    assert not out.any()
    assert kv4.attend(q[:0], s.cache, 0, s.tables, i32([0, 0, 0], dev), i32([20, 9], dev)).shape == (0, 4, 64)
    out = kv4.attend(q[:4], s.cache, 0, s.tables, i32([0, 3, 4], dev), i32([0, -5], dev))  # nothing to see
    assert not out.any()
    out = kv4.attend(q[:4], s.cache, 0, s.tables[:, :0], i32([0, 3, 4], dev), i32([20, 9], dev))  # no pages
    assert not out.any()
    into = torch.full_like(s.q, 7)
    assert s.attend(out=into) is into and torch.equal(into, s.attend())


def test_attend_more_queries_than_context(dev):
    """Queries before the first token see nothing and give zeros; the others what their place sees."""
    s = Setup(dev, [5], [9], 4, 2, 64, 16, torch.float32)
    out = s.attend()
    assert not out[:4].any()
    s.check(out)


def test_attend_missing_pages(dev):
    """Table entries that are no page of the cache: their tokens are not seen."""
    ctx = [100, 64, 37]
    s = Setup(dev, ctx, [20, 1, 2], 4, 2, 128, 16, torch.bfloat16, seed=6)
    for b, col, value in ((0, 1, -1), (0, 6, 1 << 20), (1, 0, -7), (2, 2, s.cache.pages)):
        s.tables[b, col] = value
        for x in (s.keys, s.values):
            x[b][16 * col: 16 * col + 16] = np.nan
    out = s.attend()
    for x in s.values:
        x[np.isnan(x)] = 0
    s.check(out)


def test_attend_strided_queries_and_tables(dev):
    s = Setup(dev, [90, 33], [4, 1], 6, 2, 128, 16, torch.bfloat16, seed=7)
    want = s.attend()
    wide = torch.randn(5, 11, 128, device=dev).to(torch.bfloat16)
    wide[:, 3:9] = s.q
    assert torch.equal(s.attend(wide[:, 3:9]), want)
    odd = torch.zeros(5, 6, 131, device=dev, dtype=torch.bfloat16)
    odd[..., 1:129] = s.q
    assert torch.equal(s.attend(odd[..., 1:129]), want)
    big = torch.full((2, 40), -1, dtype=torch.int32, device=dev)
    w = s.tables.shape[1]
    big[:, 5:5 + w] = s.tables
    s.tables = big[:, 5:5 + w]
    assert torch.equal(s.attend(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_extreme_scores(dev, dtype):
    """One-hot weights: large queries; and queries of very unequal sizes, zeros among them."""
    s = Setup(dev, [200, 50], [3, 1], 4, 2, 64, 16, dtype, seed=8)
    s.q *= torch.tensor([30.0, 1e-3, 0.0, 1.0], device=dev).view(4, 1, 1).to(dtype)
    s.check(s.attend())


def test_attend_offsets_past_32_bits(dev):
    """A cache of over 4 GiB whose last pages are used."""
    d, P, hkv = 128, 256, 8
    block = 2 * P * 72 * hkv
    pages = (1 << 32) // block + 500
    s = Setup(dev, [600, 513], [2, 1], 16, hkv, d, P, torch.bfloat16, seed=9, pages=pages)
    assert s.cache.nbytes > 1 << 32
    last = torch.arange(pages - 6, pages, device=dev, dtype=torch.int32)
    tables = last.view(2, 3)
    for b in range(2):
        t = torch.arange(s.ctx[b], device=dev)
        lo = sum(s.ctx[:b])
        kv4.append(s.cache, 0, s.k[lo: lo + s.ctx[b]], s.v[lo: lo + s.ctx[b]], tables[b].long()[t // P] * P + t % P)
    want = s.attend()
    s.tables = tables
    assert torch.equal(s.attend(), want)
    s.check(want)


def test_attend_is_deterministic_and_runs_on_other_streams(dev):
    s = Setup(dev, [3000, 900], [3, 1], 12, 2, 128, 16, torch.bfloat16, seed=10)
    want = s.attend()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [s.attend() for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_a_step_in_a_graph(dev):
    """Plan, append and attend of a decode step, captured once and replayed as the lengths grow."""
    B, hq, hkv, d, P, pages = 3, 8, 2, 128, 16, 64
    spec = rotary.RotarySpec(d)
    spec.on(torch.device(dev))
    ring, state = paging.free_pages(pages, dev)

    def fresh():
        return dict(cache=kv4.KV4Cache(layers=1, kv_heads=hkv, head_dim=d, pages=pages, page_size=P, device=dev),
                    tables=torch.full((B, 8), -1, dtype=torch.int32, device=dev), state=state.clone(),
                    past=i32([0, 0, 0], dev), new=i32([1, 1, 1], dev),
                    qkv=torch.zeros(B, hq + 2 * hkv, d, device=dev, dtype=torch.bfloat16))

    def step(s):
        p = paging.plan_step(ring, s["state"], s["tables"], s["past"], s["new"], page_size=P, tokens=B)
        q, k, v = s["qkv"].split([hq, hkv, hkv], 1)
        q = kv4.append(s["cache"], 0, k, v, p.slots, q=q, positions=p.positions, rotary=spec)
        out = kv4.attend(q, s["cache"], 0, s["tables"], p.query_starts, p.context_lens, max_query=1, max_context=8 * P)
        s["state"].copy_(p.free_state)
        s["past"].copy_(p.context_lens)
        return out

    a, b = fresh(), fresh()
    step(fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(b)
    for i in range(40):
        x = torch.randn(B, hq + 2 * hkv, d, device=dev).to(torch.bfloat16)
        a["qkv"].copy_(x)
        b["qkv"].copy_(x)
        want = step(a)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)
        assert torch.equal(a["state"], b["state"]) and torch.equal(a["past"], b["past"])
    assert torch.equal(a["cache"].storage, b["cache"].storage) and a["past"].tolist() == [40] * 3
    done = torch.tensor([True, False, True], device=dev)
    after = paging.release_pages(ring, a["state"], a["tables"], a["past"], done, page_size=P)
    assert after.tolist() == [9, pages + 6, 0]
