"""The operators between a decoder layer's q/k/v and its output projection, as cases that can be
timed and checked: paging metadata, rotary positions, the 4-bit KV cache and attention over it.

Kinds:

* ``plan``   -- one scheduler step's block tables, slot map and positions from request lengths;
* ``rotary`` -- rotary positions of one activation;
* ``append`` -- new keys and values, rotated, into the 4-bit cache (the queries rotated with them),
  and the values that the cache then holds for those tokens;
* ``attend`` -- attention of new tokens over the cache: single tokens, drafted ones, prompts.

With ``own`` false every operator is computed in elementary torch operations, in 32 bits (the
angles in 64), rounded once at the end; with ``own`` true by this package's entry points.

The cache's format: a token's key (or value) of one head in groups of 64 values, each with
``lo = fp16(min)``, ``s = fp16((max - min) / 15)`` and codes ``clamp(rint((x - lo) / s), 0, 15)``
(0 where s is 0); a code stands for ``code * s + lo``.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
GROUP = 64
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# (query heads, KV heads, head size): the layers whose linears this package's cases multiply
HEADS = [(12, 2, 128), (32, 8, 128), (16, 4, 128), (16, 8, 64)]

# the most that a drawn case does, as the largest listed ones
MAX_ROTARY_VALUES = 8191 * 40 * 128
MAX_APPEND_TOKENS = 4099
MAX_ATTEND_PAIRS = 32 * (4095 * 4096 // 2)
MAX_ATTEND_CACHE = 2 * 131072 * 8


def listed() -> list[dict]:
    return [
        # A decode step of a few requests: the smallest plan, all latency.
        {"name": "plan_b7", "kind": "plan", "b": 7, "past": 900, "new": 1, "page": 16, "mix": 1, "short": False},
        # A step that takes in many prompts and runs out of pages on the way.
        {"name": "plan_b511", "kind": "plan", "b": 511, "past": 2000, "new": 190, "page": 16, "mix": 2, "short": True},
        # One token's queries, plain rotary positions in bf16.
        {"name": "rotary_t1", "kind": "rotary", "t": 1, "heads": 12, "d": 128, "rot": 128, "layout": "half",
         "scaling": "none", "dtype": "bf16", "far": 4000, "strided": False},
        # A long prompt's fused q/k rows, interleaved pairs, half of each head, scaled for a long context.
        {"name": "rotary_t8191", "kind": "rotary", "t": 8191, "heads": 40, "d": 128, "rot": 64,
         "layout": "interleaved", "scaling": "yarn", "dtype": "bf16", "far": 1000000, "strided": True},
        # Decode of a batch: a token each into the cache.
        {"name": "append_t13", "kind": "append", "t": 13, "hq": 12, "hkv": 2, "d": 128, "rot": 128, "layout": "half",
         "scaling": "none", "dtype": "bf16", "far": 30000, "page": 16, "pad": 2},
        # A prompt into the cache.
        {"name": "append_t4099", "kind": "append", "t": 4099, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "layout": "half", "scaling": "linear", "dtype": "bf16", "far": 100000, "page": 64, "pad": 0},
        # One sequence, one token, a short context: all latency.
        {"name": "attend_b1", "kind": "attend", "b": 1, "hq": 12, "hkv": 2, "d": 128, "ctx": 513, "new": 1, "mix": 3,
         "page": 16, "window": 0, "dtype": "bf16", "even": True},
        # Decode of a ragged batch.
        {"name": "attend_b29", "kind": "attend", "b": 29, "hq": 32, "hkv": 8, "d": 128, "ctx": 8100, "new": 1, "mix": 4,
         "page": 64, "window": 0, "dtype": "bf16", "even": False},
        # Two sequences with long contexts, a token each.
        {"name": "attend_long", "kind": "attend", "b": 2, "hq": 32, "hkv": 8, "d": 128, "ctx": 131000, "new": 1,
         "mix": 5, "page": 128, "window": 0, "dtype": "f16", "even": True},
        # Drafted tokens of several requests, to be verified.
        {"name": "attend_draft", "kind": "attend", "b": 11, "hq": 16, "hkv": 4, "d": 128, "ctx": 6001, "new": 5,
         "mix": 6, "page": 32, "window": 0, "dtype": "bf16", "even": False},
        # A whole prompt.
        {"name": "attend_prompt", "kind": "attend", "b": 1, "hq": 32, "hkv": 8, "d": 128, "ctx": 4095, "new": 4095,
         "mix": 7, "page": 64, "window": 0, "dtype": "bf16", "even": True},
        # Chunks of prompts over a sliding window, small heads, in the fp32 stores' type.
        {"name": "attend_window", "kind": "attend", "b": 3, "hq": 16, "hkv": 8, "d": 64, "ctx": 5000, "new": 701,
         "mix": 8, "page": 16, "window": 1024, "dtype": "f32", "even": False},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], even over its logarithm, odd as often as even."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng) -> dict:
    kind = rng.choice(["plan", "rotary", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        b = _log_int(rng, 1, 511)
        return {"kind": kind, "b": b, "past": _log_int(rng, 1, 4000), "new": _log_int(rng, 1, min(4000, 80000 // b)),
                "page": page, "mix": rng.randrange(1 << 20), "short": rng.random() < 0.3}
    layout, scaling = rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "ntk", "yarn"])
    if kind == "rotary":
        heads, d = rng.randrange(1, 41), rng.choice([64, 96, 128, 128, 256])
        return {"kind": kind, "t": _log_int(rng, 1, min(8191, MAX_ROTARY_VALUES // (heads * d))), "heads": heads, "d": d,
                "rot": rng.choice([d, d // 2, d // 4]), "layout": layout, "scaling": scaling,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "far": _log_int(rng, 10, 1000000),
                "strided": rng.random() < 0.5}
    hq, hkv, d = rng.choice(HEADS)
    if kind == "append":
        t = _log_int(rng, 1, MAX_APPEND_TOKENS)
        return {"kind": kind, "t": t, "hq": hq, "hkv": hkv, "d": d, "rot": rng.choice([d, d, d // 2]), "layout": layout,
                "scaling": scaling, "dtype": rng.choice(["bf16", "bf16", "f16"]), "far": _log_int(rng, 10, 1000000),
                "page": page, "pad": rng.choice([0, 0, min(t - 1, 3)])}
    how = rng.choice(["decode", "decode", "draft", "prompt", "chunk"])
    if how in ("decode", "draft"):
        b = _log_int(rng, 1, 64)
        new = 1 if how == "decode" else rng.randrange(2, 9)
        ctx = max(new, _log_int(rng, 1, min(131000, MAX_ATTEND_CACHE // (b * hkv))))
    else:
        b = rng.randrange(1, 4)
        new = _log_int(rng, 17, 2000)
        new = max(1, min(new, MAX_ATTEND_PAIRS // (hq * b * 400)))
        ctx = new if how == "prompt" else min(20000, new + _log_int(rng, 1, max(1, MAX_ATTEND_PAIRS // (hq * b * new))))
    return {"kind": kind, "b": b, "hq": hq, "hkv": hkv, "d": d, "ctx": ctx, "new": new, "mix": rng.randrange(1 << 20),
            "page": page, "window": rng.choice([0, 0, 0, rng.randrange(1, 5000)]),
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "even": rng.random() < 0.4}


# ---- lengths, by the case alone ----------------------------------------------------------


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Each request's (tokens cached before the step, tokens of the step)."""
    r = random.Random(case["mix"])
    if case["kind"] == "plan":
        past = [r.randrange(0, case["past"] + 1) for _ in range(case["b"])]
        new = [1 if case["new"] == 1 else r.randrange(0, case["new"] + 1) for _ in range(case["b"])]
        return past, new
    if case["even"]:
        return [case["ctx"] - case["new"]] * case["b"], [case["new"]] * case["b"]
    new = [case["new"]] + [1 if case["new"] == 1 else r.randrange(1, case["new"] + 1) for _ in range(case["b"] - 1)]
    ctx = [case["ctx"]] + [r.randrange(n, case["ctx"] + 1) for n in new[1:]]
    return [c - n for c, n in zip(ctx, new)], new


def _cdiv(a, b):
    return (a + b - 1) // b


# ---- rotary frequencies ------------------------------------------------------------------

BASE = 1000000.0
FACTOR = 8.0
ORIGINAL = 32768


def _scaling(name: str):
    """The scaling as this package's entry points take it."""
    if name == "none":
        return None
    return {"type": name, "factor": FACTOR, **({"original": ORIGINAL} if name == "yarn" else {})}


def _frequencies(rot: int, scaling: str) -> tuple[np.ndarray, float]:
    """fp64 angle per position of each pair, and the factor on cos and sin."""
    i = np.arange(rot // 2, dtype=np.float64)
    base = BASE * FACTOR ** (rot / (rot - 2)) if scaling == "ntk" else BASE
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / FACTOR, 1.0
    if scaling == "yarn":
        def where(turns):
            return rot * math.log(ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(BASE))

        low, high = max(0, math.floor(where(32.0))), min(rot - 1, math.ceil(where(1.0)))
        ramp = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
        return f / FACTOR * ramp + f * (1.0 - ramp), 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


# ---- inputs ------------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(*shape, device=DEV, generator=g)


def _i32(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _keys(g, t, h, d, dtype):
    """Keys (or values) of t tokens: normal, with channels of unequal size and offset."""
    size, shift = 0.6 + 0.8 * torch.rand(h, d, device=DEV, generator=g), 0.3 * _randn(g, h, d)
    return (_randn(g, t, h, d) * size + shift).to(dtype)


def _spec(s: dict, case: dict) -> None:
    f, s["mag"] = _frequencies(case["rot"], case["scaling"])
    s["freq"] = torch.from_numpy(f).to(DEV)
    if own:
        from mrun_pub_amd import rotary

        s["spec"] = rotary.RotarySpec(case["rot"], base=BASE, layout=case["layout"], scaling=_scaling(case["scaling"]))


def _package() -> None:
    import __graft_entry__

    __graft_entry__.load_package()


def prepare(case: dict, seed: int) -> dict:
    if own:
        _package()
    g = _gen(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "plan":
        past, new = _lengths(case)
        P, b = case["page"], case["b"]
        owned = [_cdiv(p, P) for p in past]
        need = [_cdiv(p + n, P) - o for p, n, o in zip(past, new, owned)]
        width = max(o + n for o, n in zip(owned, need)) + 1
        pages = sum(owned) + sum(need) + 5
        order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
        at = torch.arange(width, device=DEV)
        first = torch.tensor(np.cumsum([0] + owned[:-1]), device=DEV)
        held = torch.tensor(owned, device=DEV)
        index = (first[:, None] + at[None, :]).clamp_(max=pages - 1)
        s["tables"] = torch.where(at[None, :] < held[:, None], order[index], -1)
        ring = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
        avail = pages - sum(owned) - (5 + sum(need) // 4 if case["short"] else 0)
        head = pages - 3  # the ring's free part wraps
        where = (head + torch.arange(avail, device=DEV)) % pages
        ring[where] = order[sum(owned): sum(owned) + avail]
        s |= {"ring": ring, "free": torch.tensor([head, head + avail, 0], dtype=torch.int64, device=DEV),
              "past": _i32(past), "new": _i32(new), "tokens": sum(new) + 3}  # three rows of padding
    elif kind == "rotary":
        dtype, (t, h, d) = _DT[case["dtype"]], (case["t"], case["heads"], case["d"])
        if case["strided"]:  # the middle of a fused projection's rows
            s["x"] = _randn(g, t, h + 3, d).to(dtype)[:, 1:h + 1]
        else:
            s["x"] = _randn(g, t, h, d).to(dtype)
        s["pos"] = torch.randint(0, case["far"], (t,), device=DEV, generator=g, dtype=torch.int32)
        _spec(s, case)
    elif kind == "append":
        dtype, t, d = _DT[case["dtype"]], case["t"], case["d"]
        qkv = torch.cat([_randn(g, t, case["hq"], d).to(dtype), _keys(g, t, case["hkv"], d, dtype),
                         _keys(g, t, case["hkv"], d, dtype)], 1)  # the rows of one fused projection
        s["q"], s["k"], s["v"] = qkv.split([case["hq"], case["hkv"], case["hkv"]], 1)
        s["pos"] = torch.randint(0, case["far"], (t,), device=DEV, generator=g, dtype=torch.int32)
        pages = _cdiv(t, case["page"]) + 2
        slots = torch.randperm(pages * case["page"], device=DEV, generator=g)[:t]
        if case["pad"]:
            slots[t - case["pad"]:] = -1  # rows of padding, which no page takes
        s["slots"] = slots
        _spec(s, case)
        if own:
            from mrun_pub_amd import kv4

            s["cache"] = kv4.KV4Cache(layers=1, kv_heads=case["hkv"], head_dim=d, pages=pages,
                                      page_size=case["page"], device=DEV)
    else:
        dtype, d, hkv, P = _DT[case["dtype"]], case["d"], case["hkv"], case["page"]
        past, new = _lengths(case)
        ctx = [p + n for p, n in zip(past, new)]
        count = [_cdiv(c, P) for c in ctx]
        pages = sum(count) + 2
        order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
        width = max(count)
        first = torch.tensor(np.cumsum([0] + count[:-1]), device=DEV)
        held = torch.tensor(count, device=DEV)
        at = torch.arange(width, device=DEV)
        index = (first[:, None] + at[None, :]).clamp_(max=pages - 1)
        s["tables"] = torch.where(at[None, :] < held[:, None], order[index], -1).to(torch.int32)
        s["ctx"], s["starts"] = _i32(ctx), _i32([0] + np.cumsum(new).tolist())
        s["max_new"], s["max_ctx"] = max(new), max(ctx)
        # queries near keys that they look for: some weights are large, as in earnest
        s["q"] = (1.3 * _randn(g, sum(new), case["hq"], d)).to(dtype)
        k, v = (_keys(g, pages * P, hkv, d, dtype) for _ in range(2))
        if own:
            from mrun_pub_amd import kv4

            s["cache"] = kv4.KV4Cache(layers=1, kv_heads=hkv, head_dim=d, pages=pages, page_size=P, device=DEV)
            # what the plain codes stand for is coded as these codes again: both sides attend over one cache,
            # whatever the rounding of the scales
            k, v = (_values(*_quantize(x)) for x in (k, v))
            kv4.append(s["cache"], 0, k, v, torch.arange(pages * P, device=DEV))
        else:
            s["kc"], s["ks"], s["kl"] = _quantize(k)
            s["vc"], s["vs"], s["vl"] = _quantize(v)
    return s


# ---- the plain forms ---------------------------------------------------------------------


def _quantize(x):
    """Codes (two a byte), scales and lowest values of [t, h, d] in groups of 64."""
    t, h, d = x.shape
    g = x.float().view(t, h, d // GROUP, GROUP)
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    lo, sc = low.half(), ((high - low) / 15.0).half()
    q = torch.where(sc > 0, torch.round((g - lo.float()) / sc.float()).clamp_(0, 15), 0.0).to(torch.uint8).view(t, h, d)
    return q[..., 0::2] | (q[..., 1::2] << 4), sc.squeeze(-1), lo.squeeze(-1)


def _values(codes, sc, lo):
    """What [..., d/2] codes stand for, in fp32."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return (q.unflatten(-1, (-1, GROUP)) * sc.float().unsqueeze(-1) + lo.float().unsqueeze(-1)).flatten(-2)


def _rotate(x, s):
    """Rotary positions of [t, h, d] in fp32, angles in fp64, in x's type."""
    case = s["case"]
    rot = case["rot"]
    angle = s["pos"].double()[:, None] * s["freq"][None, :]
    c, n = ((f(angle) * s["mag"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    y = x.float()
    if case["layout"] == "half":
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        r = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        r = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([r, y[..., rot:]], -1).to(x.dtype)


def _plan(s):
    P, T = s["case"]["page"], s["tokens"]
    past, new, tables, ring = s["past"].long(), s["new"].long(), s["tables"], s["ring"]
    head, avail = s["free"][0], s["free"][1] - s["free"][0]
    owned, total = (past + P - 1) // P, (past + new + P - 1) // P
    need = total - owned
    base = need.cumsum(0) - need
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    at = torch.arange(tables.shape[1], device=DEV)
    rank = base[:, None] + at[None, :] - owned[:, None]
    page = torch.where(rank < avail, ring[(head + rank) % ring.numel()], -1)
    tables = torch.where((at >= owned[:, None]) & (at < total[:, None]), page, tables)
    tok = torch.arange(T, device=DEV)
    valid = tok < starts[-1]
    req = torch.searchsorted(starts[1:], tok, right=True).clamp_(max=past.numel() - 1)
    pos = past[req] + tok - starts[req]
    page = tables[req, (pos // P).clamp(max=tables.shape[1] - 1)].long()
    slots = torch.where(valid & (page >= 0), page * P + pos % P, -1)
    taken = torch.minimum(need.sum(), avail)
    free = torch.stack([head + taken, s["free"][1], need.sum() - taken])
    return {"tables": tables, "slots": slots, "positions": torch.where(valid, pos, 0).int(),
            "requests": torch.where(valid, req, -1).int(), "starts": starts.int(), "context": (past + new).int(),
            "free": free}


def _attend(s):
    case = s["case"]
    hkv, d, P = case["hkv"], case["d"], case["page"]
    grp = case["hq"] // hkv
    q, starts, ctx = s["q"], s["starts"].long(), s["ctx"].long()
    n, m = s["max_new"], s["max_ctx"]
    at = torch.arange(m, device=DEV)
    slot = s["tables"].long()[:, at // P].clamp_(min=0) * P + at % P  # [b, m]
    k, v = (_values(s[a + "c"][slot], s[a + "s"][slot], s[a + "l"][slot]).permute(0, 2, 1, 3) for a in "kv")
    new = starts[1:] - starts[:-1]
    row = torch.arange(n, device=DEV)
    src = (starts[:-1, None] + row).clamp_(max=q.shape[0] - 1)  # [b, n]
    rows = q[src].float().view(-1, n, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(-1, hkv, grp * n, d)
    pos = (ctx - new)[:, None] + row  # [b, n]
    see = (at <= pos[..., None]) & (at < ctx[:, None, None])
    if case["window"]:
        see &= at > pos[..., None] - case["window"]
    w = torch.matmul(rows, k.transpose(2, 3).contiguous()).view(-1, hkv, grp, n, m) * (1.0 / math.sqrt(d))
    w = w.masked_fill_(~see[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(-1, hkv, grp * n, m), v.contiguous()).view(-1, hkv, grp, n, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, n, hkv * grp, d)  # [b, n, hq, d]
    tok = torch.arange(q.shape[0], device=DEV)
    req = torch.searchsorted(starts[1:], tok, right=True)
    return o[req, tok - starts[req]].to(q.dtype)


def run(s: dict):
    case = s["case"]
    kind = case["kind"]
    if own:
        from mrun_pub_amd import kv4, paging, rotary

        if kind == "plan":
            p = paging.plan_step(s["ring"], s["free"], s["tables"], s["past"], s["new"], page_size=case["page"],
                                 tokens=s["tokens"])
            return {"tables": s["tables"], "slots": p.slots, "positions": p.positions, "requests": p.requests,
                    "starts": p.query_starts, "context": p.context_lens, "free": p.free_state}
        if kind == "rotary":
            return rotary.apply_rotary(s["x"], s["pos"], s["spec"])
        if kind == "append":
            q = kv4.append(s["cache"], 0, s["k"], s["v"], s["slots"], q=s["q"], positions=s["pos"], rotary=s["spec"])
            k, v = kv4.read(s["cache"], 0, s["slots"], dtype=s["k"].dtype)
            return {"q": q, "k": k, "v": v}
        return kv4.attend(s["q"], s["cache"], 0, s["tables"], s["starts"], s["ctx"], max_query=s["max_new"],
                          max_context=s["max_ctx"], window=case["window"] or None)
    if kind == "plan":
        return _plan(s)
    if kind == "rotary":
        return _rotate(s["x"], s)
    if kind == "append":
        put = (s["slots"] >= 0)[:, None, None]
        k, v = (torch.where(put, _values(*_quantize(x)), 0.0).to(x.dtype) for x in (_rotate(s["k"], s), s["v"]))
        return {"q": _rotate(s["q"], s), "k": k, "v": v}
    return _attend(s)


# ---- what a pass cannot do without -------------------------------------------------------


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "plan":
        past, new = _lengths(case)
        need = sum(_cdiv(p + n, case["page"]) - _cdiv(p, case["page"]) for p, n in zip(past, new))
        # lengths in; starts, context and three words a request and token out; a table entry in or out a page
        return {"bytes": 16 * case["b"] + 16 * (sum(new) + 3) + 8 * need + 4 * case["b"], "flops": 10 * sum(new)}
    if kind == "rotary":
        values = case["t"] * case["heads"] * case["d"]
        return {"bytes": 2 * values * _BYTES[case["dtype"]] + 4 * case["t"],
                "flops": 3 * case["t"] * case["heads"] * case["rot"]}
    cell = case["d"] // 2 + 4 * (case["d"] // GROUP)  # a token's key of one head in the cache
    if kind == "append":
        t, size = case["t"], _BYTES[case["dtype"]]
        q, kv = t * case["hq"] * case["d"], 2 * t * case["hkv"] * case["d"]
        # q in and out, k and v in, into the cache, out of it and out
        return {"bytes": 2 * q * size + 2 * kv * size + 2 * 2 * t * case["hkv"] * cell + 12 * t,
                "flops": 3 * q + 10 * kv}
    past, new = _lengths(case)
    win = case["window"] or 1 << 40
    pairs = seen = 0
    for p, n in zip(past, new):
        lo = max(0, p + 1 - win)
        seen += p + n - lo
        full = max(0, min(n, p + n - win))  # queries that see a whole window
        part = n - full
        pairs += full * win + part * (p + 1) + part * (part - 1) // 2
    q = sum(new) * case["hq"] * case["d"] * _BYTES[case["dtype"]]
    return {"bytes": 2 * q + 2 * seen * case["hkv"] * cell, "flops": 4 * pairs * case["hq"] * case["d"]}


# ---- the definitions in 64 bits ----------------------------------------------------------


def _exact_rotate(x, pos, case):
    f, mag = _frequencies(case["rot"], case["scaling"])
    y, half = x.double().clone(), case["rot"] // 2
    turn = torch.polar(torch.full((x.shape[0], 1, half), mag, dtype=torch.float64, device=DEV),
                       (pos.double()[:, None] * torch.from_numpy(f).to(DEV)[None, :])[:, None, :])
    one, two = ((slice(0, half), slice(half, 2 * half)) if case["layout"] == "half"
                else (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    z = torch.complex(y[..., one], y[..., two]) * turn
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_cached(x):
    """What the cache holds for the values x (of their own type), in fp64."""
    out = x.double()
    for j in range(0, x.shape[-1], GROUP):
        part = out[..., j:j + GROUP]
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        lo, step = low.half().double(), ((high - low) / 15).half().double()
        code = ((part - lo) / step.clamp(min=1e-30)).round().clamp(0, 15) * (step > 0)
        out[..., j:j + GROUP] = code * step + lo
    return out


def exact(case: dict, seed: int):
    global own
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers: the plain form has to be met exactly
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if kind == "rotary":
        return _exact_rotate(s["x"], s["pos"], case)
    if kind == "append":
        kept = (s["slots"] >= 0).double()[:, None, None]
        k = _exact_rotate(s["k"], s["pos"], case).to(s["k"].dtype)
        return {"q": _exact_rotate(s["q"], s["pos"], case), "k": _exact_cached(k) * kept,
                "v": _exact_cached(s["v"]) * kept}
    past, new = _lengths(case)
    hkv, d, P = case["hkv"], case["d"], case["page"]
    grp = case["hq"] // hkv
    k, v = (((torch.stack([s[a + "c"] & 15, s[a + "c"] >> 4], -1).view(-1, hkv, d // GROUP, GROUP).double())
             * s[a + "s"].double()[..., None] + s[a + "l"].double()[..., None]).view(-1, hkv, d) for a in "kv")
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for b in range(case["b"]):
        n = past[b] + new[b]
        t = torch.arange(n, device=DEV)
        at = s["tables"][b].long()[t // P] * P + t % P
        for h in range(case["hq"]):
            kh, vh = k[at, h // grp], v[at, h // grp]
            for i in range(0, new[b], 1024):
                j = min(new[b], i + 1024)
                pos = torch.arange(past[b] + i, past[b] + j, device=DEV)[:, None]
                sc = s["q"][row + i:row + j, h].double() @ kh.t() / math.sqrt(d)
                hide = (t[None, :] > pos) | (t[None, :] <= pos - (case["window"] or 1 << 40))
                out[row + i:row + j, h] = torch.softmax(sc.masked_fill(hide, -math.inf), -1) @ vh
        row += new[b]
    return out
