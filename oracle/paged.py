"""Rotary positions and attention over a paged cache in 64 bits, from their definitions, with the bounds
that a kernel's roundings leave. Test infrastructure."""
from __future__ import annotations

import math

import numpy as np

HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def rotate(x, positions, frequencies, magnitude=1.0, layout="half", inverse=False):
    """x [rows, heads, hd] with its first 2 * len(frequencies) elements turned."""
    x = np.asarray(x, np.float64)
    d = 2 * len(frequencies)
    t = np.asarray(positions, np.float64)[:, None, None] * np.asarray(frequencies, np.float64)
    c, s = magnitude * np.cos(t), magnitude * np.sin(t) * (-1 if inverse else 1)
    a, b = (x[..., :d // 2], x[..., d // 2:d]) if layout == "half" else (x[..., :d:2], x[..., 1:d:2])
    y = x.copy()
    if layout == "half":
        y[..., :d // 2], y[..., d // 2:d] = a * c - b * s, a * s + b * c
    else:
        y[..., :d:2], y[..., 1:d:2] = a * c - b * s, a * s + b * c
    return y


def rotate_bound(x, y, frequencies, magnitude, layout, out, angle=2.0**-22, positions=None):
    """How far a kernel's result may be from y: its rounding to `out`; and of each element of a pair,
    by the size of the pair, cosine and sine (2^-22: their series, evaluated in fp32, to 2^-23, the
    angle, cut to 2^-32 of a turn and rounded as fp32, to 2^-23) and the sum in fp32 (2^-23). Positions
    at which the 64-bit product p f is itself off by more than that are the caller's to add."""
    x = np.abs(np.asarray(x, np.float64))
    d = 2 * len(frequencies)
    pair = np.zeros_like(x)
    a, b = (x[..., :d // 2], x[..., d // 2:d]) if layout == "half" else (x[..., :d:2], x[..., 1:d:2])
    both = (a + b) * abs(magnitude) * (angle + 2.0**-23)
    if layout == "half":
        pair[..., :d // 2] = pair[..., d // 2:d] = both
    else:
        pair[..., :d:2] = pair[..., 1:d:2] = both
    tiny = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-134}[out]  # half a subnormal's step
    turned = np.zeros_like(x)
    turned[..., :d] = HALF_STEP[out] * np.abs(y[..., :d]) + tiny
    return turned + pair * (1 + HALF_STEP[out])


def key_ends(kind, pos0, rows, keys, prompt_len=0, block=1):
    """How many of the sequence's keys each row sees, always the first ones."""
    out = []
    for p in range(pos0, pos0 + rows):
        if kind == "full":
            out.append(keys)
        elif kind == "causal":
            out.append(min(keys, p + 1))
        elif p < prompt_len:
            out.append(min(keys, prompt_len))
        else:
            out.append(min(keys, prompt_len + ((p - prompt_len) // block + 1) * block))
    return out


def attention(q, k, v, ends, kind="f16", out="f32"):
    """(o, bound) [rows, heads, 128] of q [rows, heads, 128] over k, v [keys, kv_heads, 128] (what the
    cache holds), row r over its first ends[r] keys; no key: zeros.

    The bound counts what changes a weight alike above and below the fraction, so that it moves the
    result by w |v - o| times as much: the weight's rounding to the cache's type `kind`, its score's fp32
    sum (130 roundings of its products' magnitudes), the exponent's argument and the power (2^-18: the
    argument is rounded to 2^-24 of up to 2^5 once the base is off). Then the sums in fp32 (2^-18: single
    roundings in chains of a few dozen). Weights of fp16 below its smallest normal one are off by 2^-25
    each of at least one whole weight in the sum. Then the result's rounding to `out`."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rows, hq, hd = q.shape
    g = hq // k.shape[1]
    o, bound = np.zeros((rows, hq, hd)), np.zeros((rows, hq, hd))
    for r in range(rows):
        n = ends[r]
        if n == 0:
            continue
        for h in range(hq):
            kk, vv = k[:n, h // g], v[:n, h // g]
            s = kk @ q[r, h] / math.sqrt(hd)
            size = np.abs(kk) @ np.abs(q[r, h]) / math.sqrt(hd)
            w = np.exp(s - s.max())
            total = w.sum()
            w /= total
            o[r, h] = w @ vv
            per = HALF_STEP[kind] + 130 * 2.0**-24 * size + 2.0**-18
            apart = np.abs(vv - o[r, h])
            bound[r, h] = (w * per) @ apart + 2.0**-18 * (w @ np.abs(vv) + np.abs(o[r, h]))
            if kind == "f16":
                bound[r, h] += 2.0**-25 * apart.sum(0) / total
            bound[r, h] += HALF_STEP[out] * (np.abs(o[r, h]) + bound[r, h])
    return o, bound
