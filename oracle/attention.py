"""Plain numpy forms of the operators around the paged 4-bit KV cache, in 64 bits where they compute.

* ``plan_step`` / ``release_pages``: request by request, page by page.
* ``rotary``: the turned pairs in fp64.
* ``kv4_quantize`` / ``kv4_values``: codes, scales and lowest values of groups of 64; fp32 IEEE
  operations, which are the format's definition.
* ``attend``: softmax over each query's visible tokens in fp64, with the sums that an error bound needs.
"""

from __future__ import annotations

import math

import numpy as np

GROUP = 64
MAX = np.float32(60000.0)


def plan_step(ring, state, tables, past, new, page_size, tokens):
    """``(tables, slots, positions, requests, starts, context, state)`` of one step."""
    tables = np.array(tables)
    head, tail = int(state[0]), int(state[1])
    avail = min(max(0, tail - head), len(ring))
    taken = missing = 0
    slots, positions, requests, starts, context = [], [], [], [], []
    row = 0
    for b, (p, n) in enumerate(zip(past, new)):
        p, n = max(0, int(p)), max(0, int(n))
        starts.append(min(row, tokens))
        asked = n
        n = max(0, min(n, tokens - row))
        context.append(p + n)
        owned, last = -(-p // page_size), min(-(-(p + n) // page_size), tables.shape[1])
        for c in range(owned, last):
            if taken < avail:
                tables[b, c] = ring[(head + taken) % len(ring)]
                taken += 1
            else:
                tables[b, c] = -1
                missing += 1
        for pos in range(p, p + n):
            c = pos // page_size
            page = int(tables[b, c]) if c < tables.shape[1] else -1
            slots.append(page * page_size + pos % page_size if page >= 0 else -1)
            positions.append(pos)
            requests.append(b)
        row += asked
    starts.append(min(row, tokens))
    pad = tokens - len(slots)
    return (tables, np.array(slots + [-1] * pad, np.int64), np.array(positions + [0] * pad, np.int32),
            np.array(requests + [-1] * pad, np.int32), np.array(starts, np.int32), np.array(context, np.int32),
            np.array([head + taken, tail, missing], np.int64))


def release_pages(ring, state, tables, lens, done, page_size):
    ring, tail = np.array(ring), int(state[1])
    for b, gone in enumerate(done):
        if not gone:
            continue
        for c in range(min(-(-max(0, int(lens[b])) // page_size), tables.shape[1])):
            if tables[b, c] >= 0:
                ring[tail % len(ring)] = tables[b, c]
                tail += 1
    return ring, np.array([int(state[0]), tail, 0], np.int64)


def rotary_frequencies(dim, base, scaling=None):
    """Angles per position of each pair in fp64, and the factor on cos and sin."""
    out, mag = [], 1.0
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        if scaling is not None and scaling["type"] == "linear":
            f /= scaling["factor"]
        elif scaling is not None and scaling["type"] == "ntk":
            f = (base * scaling["factor"] ** (dim / (dim - 2))) ** (-2.0 * i / dim)
        elif scaling is not None:
            s, n = scaling["factor"], scaling["original"]
            edge = [dim * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))
                    for turns in (scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0))]
            low, high = max(0, math.floor(edge[0])), min(dim - 1, math.ceil(edge[1]))
            ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            f = f / s * ramp + f * (1 - ramp)
            mag = scaling.get("magnitude", 0.1 * math.log(s) + 1)
        out.append(f)
    return np.array(out), mag


def rotary(x, positions, freq, mag, layout, inverse=False):
    """``x [t, h, d]`` turned, in fp64, and for each value the sum of sizes that its error scales with."""
    x = np.asarray(x, np.float64)
    half = len(freq)
    angle = np.asarray(positions, np.float64)[:, None, None] * freq
    c, s = np.cos(angle) * mag, np.sin(angle) * mag * (-1 if inverse else 1)
    one = slice(0, half) if layout == "half" else slice(0, 2 * half, 2)
    two = slice(half, 2 * half) if layout == "half" else slice(1, 2 * half, 2)
    y, size = x.copy(), np.zeros_like(x)
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    size[..., one] = size[..., two] = (abs(x[..., one]) + abs(x[..., two])) * mag
    return y, size


def kv4_quantize(x):
    """Codes uint8 ``[t, h, d]``, scales and lowest values fp16 ``[t, h, d/64]`` of fp32 values."""
    x = np.asarray(x, np.float32)
    t, h, d = x.shape
    g = np.where(np.isnan(x), np.float32(0), np.clip(x, -MAX, MAX)).reshape(t, h, d // GROUP, GROUP)
    low, high = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    lo, s = low.astype(np.float16), ((high - low) / np.float32(15)).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.clip(np.rint((g - lo.astype(np.float32)) / s.astype(np.float32)), 0, 15)
    q = np.where(s > 0, q, 0).astype(np.uint8)
    return q.reshape(t, h, d), s[..., 0], lo[..., 0]


def kv4_values(codes, s, lo):
    """What codes stand for, in fp32."""
    g = codes.reshape(*codes.shape[:-1], -1, GROUP).astype(np.float32)
    return (g * s.astype(np.float32)[..., None] + lo.astype(np.float32)[..., None]).reshape(codes.shape)


def attend(q, keys, values, starts, context, scale, window=None):
    """``keys[b]``, ``values[b]``: ``[context, hkv, d]`` of request b, NaN rows for tokens that are not
    seen.  Returns the output ``[t, hq, d]`` in fp64 and, of the same shape, ``sum w |v|`` and the
    largest ``scale * sum |q| |k|`` of a query's visible tokens."""
    t, hq, d = q.shape
    q = np.asarray(q, np.float64)
    out, weight, reach = np.zeros((t, hq, d)), np.zeros((t, hq, d)), np.zeros((t, hq, 1))
    for b in range(len(context)):
        k, v = np.asarray(keys[b], np.float64), np.asarray(values[b], np.float64)
        n = int(starts[b + 1]) - int(starts[b])
        hkv = k.shape[1]
        for i in range(n):
            pos = int(context[b]) - n + i
            first = max(0, pos - window + 1) if window else 0
            at = np.arange(first, min(pos + 1, k.shape[0]))
            at = at[~np.isnan(k[at, 0, 0])] if len(at) else at
            if not len(at):
                continue
            for h in range(hq):
                kh, vh = k[at, h // (hq // hkv)], v[at, h // (hq // hkv)]
                row = q[starts[b] + i, h]
                x = kh @ row * scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[starts[b] + i, h] = w @ vh
                weight[starts[b] + i, h] = w @ abs(vh)
                reach[starts[b] + i, h] = (abs(kh) @ abs(row)).max() * scale
    return out, weight, reach
