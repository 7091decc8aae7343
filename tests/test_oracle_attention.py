"""CPU checks of the plain forms behind the 4-bit KV cache's operators, and of the host side."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from mrun_pub_amd import rotary
from oracle import attention as oa


def test_plan_hand_checked():
    tables = np.full((3, 3), -1, np.int32)
    tables[0, 0] = 7
    got = oa.plan_step(np.array([4, 5, 6]), [2, 5, 0], tables, [3, 0, 4], [2, 0, 1], 4, 4)
    assert got[0].tolist() == [[7, 6, -1], [-1, -1, -1], [-1, 4, -1]]
    assert got[1].tolist() == [31, 24, 16, -1]
    assert got[2].tolist() == [3, 4, 4, 0] and got[3].tolist() == [0, 0, 2, -1]
    assert got[4].tolist() == [0, 2, 2, 3] and got[5].tolist() == [5, 0, 5]
    assert got[6].tolist() == [4, 5, 0]


def test_quantized_values_stay_within_half_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((9, 2, 128)) * 10.0 ** rng.uniform(-3, 3, (9, 2, 1))).astype(np.float32)
    c, s, lo = oa.kv4_quantize(x)
    step, low = (np.repeat(a.astype(np.float64), 64, -1) for a in (s, lo))
    # half a step, the rounding of the lowest value, and of the step over 15 of them
    bound = step / 2 + abs(low) * 2.0**-11 + 15 * step * 2.0**-11 + 2.0**-23
    assert (abs(oa.kv4_values(c, s, lo) - x) <= bound * (1 + 1e-6)).all()
    assert c.min() == 0 and c.max() == 15


def test_quantize_edges():
    x = np.zeros((1, 5, 64), np.float32)
    x[0, 1] = 3.25
    x[0, 2, :2] = [np.nan, np.inf]
    x[0, 3, :2] = [-np.inf, 1e30]
    x[0, 4, 5] = 1e-12
    c, s, lo = oa.kv4_quantize(x)
    v = oa.kv4_values(c, s, lo)
    assert np.isfinite(v).all()
    assert (v[0, 0] == 0).all() and (v[0, 1] == 3.25).all() and (v[0, 4] == 0).all()
    assert v[0, 2, 0] == 0 and abs(v[0, 2, 1] - 60000) <= 60000 * 2.0**-11
    assert abs(v[0, 3, 0] + 60000) <= 60000 * 2.0**-11


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 4.0},
                                     {"type": "yarn", "factor": 8.0, "original": 4096},
                                     {"type": "yarn", "factor": 8.0, "original": 4096, "magnitude": 1.0, "beta_fast": 16.0}])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_rotary_frequencies(dim, scaling):
    spec = rotary.RotarySpec(dim, base=1e6, scaling=scaling)
    freq, mag = oa.rotary_frequencies(dim, 1e6, scaling)
    assert np.allclose(spec.frequencies.numpy(), freq, rtol=1e-14, atol=0) and math.isclose(spec.magnitude, mag)


def test_rotary_ntk_keeps_the_fastest_and_slows_the_slowest():
    plain, ntk = (rotary.RotarySpec(64, base=1e4, scaling=s).frequencies for s in (None, {"type": "ntk", "factor": 8.0}))
    assert ntk[0] == plain[0] == 1.0
    assert math.isclose(float(plain[-1] / ntk[-1]), 8.0, rel_tol=1e-12)


@pytest.mark.parametrize("make", [
    lambda: rotary.RotarySpec(0), lambda: rotary.RotarySpec(63), lambda: rotary.RotarySpec(64, layout="other"),
    lambda: rotary.RotarySpec(64, base=0.0), lambda: rotary.RotarySpec(64, scaling={"type": "other", "factor": 2.0}),
    lambda: rotary.RotarySpec(64, scaling={"type": "linear", "factor": 0.5}),
    lambda: rotary.RotarySpec(64, scaling={"type": "linear", "factor": 2.0, "extra": 1}),
    lambda: rotary.RotarySpec(64, scaling={"type": "yarn", "factor": 2.0}),
    lambda: rotary.RotarySpec(2, scaling={"type": "ntk", "factor": 2.0}),
])
def test_rotary_spec_refusals(make):
    with pytest.raises(ValueError):
        make()


def test_rotary_inverse_is_the_transpose():
    rng = np.random.default_rng(1)
    x, g = rng.standard_normal((2, 5, 3, 40))
    freq, mag = oa.rotary_frequencies(32, 1e4)
    pos = rng.integers(0, 1000, 5)
    for layout in rotary.LAYOUTS:
        y, _ = oa.rotary(x, pos, freq, mag, layout)
        back, _ = oa.rotary(g, pos, freq, mag, layout, inverse=True)
        assert math.isclose(float((y * g).sum()), float((x * back).sum()), rel_tol=1e-12)


def test_attention_weights_sum_to_one_and_window_one_is_the_own_value():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((4, 6, 64)), rng.standard_normal((9, 2, 64)), rng.standard_normal((9, 2, 64))
    out, weight, _ = oa.attend(q, [k], [np.ones_like(v)], [0, 4], [9], 0.125)
    assert np.allclose(out, 1.0) and np.allclose(weight, 1.0)
    out, _, _ = oa.attend(q, [k], [v], [0, 4], [9], 0.125, window=1)
    assert np.allclose(out, np.repeat(v[5:], 3, 1))
    out, _, _ = oa.attend(q, [k[:0]], [v[:0]], [0, 4], [0], 0.125)
    assert (out == 0).all()


# ---- the C entry points' refusals, which touch no device -------------------------------------


def _lib():
    import mrun_pub_amd._native as nat

    if not nat.LIB_PATH.exists():
        pytest.skip("library not built")
    return nat, nat.load()


FAKE = 1 << 20  # an aligned pointer that is never read: the checks come first


def _plan(**over):
    a = dict(ring=FAKE, ring_size=8, state=FAKE, state_out=FAKE + 64, tables=FAKE, ld=4, width=4, past=FAKE, fresh=FAKE,
             B=2, P=16, T=3, slots=FAKE, positions=FAKE, requests=FAKE, starts=FAKE, context=FAKE, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over", [
    {"ring": None}, {"state": None}, {"past": None}, {"slots": None}, {"tables": None}, {"ring_size": 0}, {"B": -1},
    {"T": -1}, {"P": 0}, {"P": 24}, {"ld": 3}, {"state_out": FAKE}, {"T": 1 << 31}, {"B": 1 << 21}, {"width": 1 << 31, "ld": 1 << 31},
])
def test_plan_refusals(over):
    nat, lib = _lib()
    assert lib.qs_plan_step(*_plan(**over)) in (nat.QS_ERR_INVALID, nat.QS_ERR_LIMIT)
    assert b"plan_step" in lib.qs_last_error()


@pytest.mark.parametrize("over", [{1: 0}, {0: None}, {7: None}, {8: None}, {10: 24}, {9: -1}, {3: FAKE}])
def test_release_refusals(over):
    nat, lib = _lib()
    a = [FAKE, 8, FAKE, FAKE + 64, FAKE, 4, 4, FAKE, FAKE, 2, 16, None]
    for i, v in over.items():
        a[i] = v
    assert lib.qs_release_pages(*a) == nat.QS_ERR_INVALID
    assert b"release_pages" in lib.qs_last_error()


@pytest.mark.parametrize("over", [{0: None}, {1: 3}, {4: None}, {5: None}, {6: 0}, {6: 7}, {6: 130}, {10: None}, {13: -1}, {14: 0},
                                  {15: 5000, 6: 64}])
def test_rotary_refusals(over):
    nat, lib = _lib()
    a = [FAKE, 1, 1536, 128, FAKE, FAKE, 128, 0, 0, 1.0, FAKE, 1536, 128, 4, 12, 128, None]
    for i, v in over.items():
        a[i] = v
    assert lib.qs_rotary(*a) in (nat.QS_ERR_INVALID, nat.QS_ERR_LIMIT)
    assert b"rotary" in lib.qs_last_error()


@pytest.mark.parametrize("over,status", [
    ({0: None}, -1), ({3: None}, -1), ({7: None}, -1), ({8: None}, -1), ({6: 3}, -1), ({1: 258}, -1), ({0: FAKE + 2}, -1),
    ({9: 0}, -1), ({9: 1 << 31}, -4), ({10: 24}, -2), ({12: 96}, -2), ({11: 0}, -1), ({21: 132, 19: FAKE}, -1), ({21: 12}, -1), ({19: None}, -1),
    ({14: None}, -1), ({13: 1 << 31}, -4),
])
def test_append_refusals(over, status):
    nat, lib = _lib()
    a = [FAKE, 256, 128, FAKE, 256, 128, 1, FAKE, FAKE, 4, 16, 2, 128, 5, FAKE, 1536, 128, 12, FAKE, FAKE, FAKE, 128, 0,
         1.0, None]
    for i, v in over.items():
        a[i] = v
    assert lib.qs_kv4_append(*a) == status
    assert b"kv4_append" in lib.qs_last_error()


@pytest.mark.parametrize("over,status", [({0: None}, -1), ({2: 48}, -2), ({4: 80}, -2), ({5: None}, -1), ({6: -1}, -1),
                                         ({7: None, 8: None}, -1), ({7: FAKE + 2}, -1), ({9: 3}, -1), ({3: 0}, -1)])
def test_read_refusals(over, status):
    nat, lib = _lib()
    a = [FAKE, 4, 16, 2, 128, FAKE, 3, FAKE, FAKE, 1, None]
    for i, v in over.items():
        a[i] = v
    assert lib.qs_kv4_read(*a) == status
    assert b"kv4_read" in lib.qs_last_error()


@pytest.mark.parametrize("over,status", [
    ({0: None}, -1), ({1: 3}, -1), ({2: 1540}, -1), ({0: FAKE + 2}, -1), ({4: None}, -1), ({5: 0}, -1), ({6: 8}, -2), ({9: 112}, -2),
    ({8: 13}, -1), ({7: 0}, -1), ({10: None}, -1), ({11: 3}, -1), ({13: None}, -1), ({14: None}, -1), ({19: 0.0}, -1),
    ({19: -1.0}, -1), ({19: float("nan")}, -1), ({19: float("inf")}, -1), ({20: -1}, -1), ({21: None}, -1), ({16: 1 << 30}, -4),
    ({18: 1 << 20}, -1),  # a split needs a workspace
])
def test_attend_refusals(over, status):
    nat, lib = _lib()
    a = [FAKE, 1, 1536, 128, FAKE, 9, 16, 2, 12, 128, FAKE, 4, 4, FAKE, FAKE, 2, 2, 1, 60, 0.1, 0, FAKE, None, 0, None]
    for i, v in over.items():
        a[i] = v
    assert lib.qs_kv4_attend(*a) == status
    assert b"kv4_attend" in lib.qs_last_error()


def test_block_bytes():
    _nat, lib = _lib()
    assert lib.qs_kv4_block_bytes(128, 16) == 2 * 16 * 72
    assert lib.qs_kv4_block_bytes(64, 256) == 2 * 256 * 36
    assert lib.qs_kv4_block_bytes(96, 16) == 0 and lib.qs_kv4_block_bytes(128, 24) == 0


def test_host_tensors_are_refused():
    _lib()
    from mrun_pub_amd import kv4, paging

    spec = rotary.RotarySpec(64)
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="HIP"):
        rotary.apply_rotary(x, torch.zeros(3, dtype=torch.int32), spec)
    with pytest.raises(ValueError):
        rotary.apply_rotary(x, torch.zeros(2, dtype=torch.int32), spec)
    with pytest.raises(ValueError):
        rotary.apply_rotary(x, torch.zeros(3), spec)
    with pytest.raises(ValueError):
        rotary.apply_rotary(x[..., :32], torch.zeros(3, dtype=torch.int32), spec)
    with pytest.raises(ValueError):
        rotary.apply_rotary(x[0], torch.zeros(3, dtype=torch.int32), spec)
    ring, state = paging.free_pages(8, "cpu", first=1)
    assert ring.tolist() == [1, 2, 3, 4, 5, 6, 7] and state.tolist() == [0, 7, 0]
    lens = torch.zeros(2, dtype=torch.int32)
    tables = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP"):
        paging.plan_step(ring, state, tables, lens, lens, page_size=16, tokens=2)
    for bad in (dict(tables=tables[:1]), dict(tables=tables.long()), dict(ring=ring.long()), dict(state=state[:2]),
                dict(lens=lens.float()), dict(tokens=-1)):
        a = dict(ring=ring, state=state, tables=tables, lens=lens, tokens=2) | bad
        with pytest.raises(ValueError):
            paging.plan_step(a["ring"], a["state"], a["tables"], a["lens"], lens, page_size=16, tokens=a["tokens"])
    with pytest.raises(ValueError):
        paging.free_pages(4, "cpu", first=4)
    for bad in (dict(head_dim=96), dict(page_size=24), dict(pages=0), dict(layers=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            kv4.KV4Cache(**(dict(layers=1, kv_heads=2, head_dim=64, pages=2, page_size=16, device="cpu") | bad))
    cache = kv4.KV4Cache(layers=1, kv_heads=2, head_dim=64, pages=2, page_size=16, device="cpu")
    assert cache.nbytes == 2 * 2 * 2 * 16 * 36
    slots = torch.zeros(3, dtype=torch.int64)
    pos = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP"):
        kv4.append(cache, 0, x, x, slots)
    for kw in (dict(layer=1), dict(v=x.half()), dict(k=x.double(), v=x.double()), dict(slots=slots[:2]), dict(slots=pos.float()),
               dict(k=x[:, :1]), dict(v=x[..., :32]), dict(positions=pos), dict(rotary=spec), dict(q=x),
               dict(positions=pos, rotary=rotary.RotarySpec(12)), dict(positions=pos, rotary=rotary.RotarySpec(128))):
        a = dict(layer=0, k=x, v=x, slots=slots) | kw
        with pytest.raises(ValueError):
            kv4.append(cache, a.pop("layer"), a.pop("k"), a.pop("v"), a.pop("slots"), **a)
    with pytest.raises(ValueError):
        kv4.read(cache, 0, slots, dtype=torch.int32)
    ctx, starts = torch.ones(2, dtype=torch.int32), torch.tensor([0, 1, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP"):
        kv4.attend(x, cache, 0, tables, starts, ctx)
    for kw in (dict(q=x[0]), dict(q=x.double()), dict(q=torch.zeros(3, 3, 64)), dict(q=torch.zeros(3, 2, 128)), dict(tables=tables[:1]),
               dict(tables=tables.long()), dict(starts=starts[:2]), dict(starts=starts.long()), dict(ctx=ctx.long()),
               dict(window=0), dict(max_query=-1)):
        a = dict(q=x, layer=0, tables=tables, starts=starts, ctx=ctx) | kw
        with pytest.raises(ValueError):
            kv4.attend(a.pop("q"), cache, a.pop("layer"), a.pop("tables"), a.pop("starts"), a.pop("ctx"), **a)
