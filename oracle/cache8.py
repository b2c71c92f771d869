"""The 8-bit K/V cache and the block-sparse attention in float64 (oracle; test-only).

The reference has neither (its K/V stays in the compute dtype,
``backends/mlx_ops.py:347-443``): these are the definitions of
``diffusorrt_amd.kernels.PrefixKVCache``'s, parity unpinned.
"""
from __future__ import annotations

import numpy as np

TILE = 32
MIN_EXP, MAX_EXP = -40, 40


def exponent(most: float):
    """The least e >= -40 with most <= 127 * 2^e; None where the tile is NaN."""
    if not np.isfinite(most) or most > 127 * 2.0 ** MAX_EXP:
        return None
    e = MIN_EXP
    while 127 * 2.0 ** e < most:
        e += 1
    return e


def quantize_tile(x):
    """One head's 32 keys ``[32, 128]`` -> (whole numbers or None, exponent or None)."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        e = exponent(np.abs(x).max())
    return (None, None) if e is None else (np.rint(x * 2.0 ** -e), e)  # rint: ties to even


class Cache8:
    """Values an 8-bit cache reads as, ``[tiles * 32, hkv, 128]``, with its tile exponents."""

    def __init__(self, hkv: int, capacity: int):
        tiles = -(-capacity // TILE)
        self.hkv = hkv
        self.values = np.zeros((2, tiles * TILE, hkv, 128))
        self.scales = np.ones((hkv, tiles, 2))

    def store(self, k, v, pos0: int) -> None:
        n = len(k)
        for w, x in enumerate((k, v)):
            self.values[w, pos0:pos0 + n] = np.asarray(x, np.float64)
        for t in range(pos0 // TILE, (pos0 + n - 1) // TILE + 1):
            for h in range(self.hkv):
                for w in range(2):
                    tile = self.values[w, t * TILE:(t + 1) * TILE, h]
                    q, e = quantize_tile(tile)
                    tile[:] = np.nan if e is None else q * 2.0 ** e
                    self.scales[h, t, w] = np.nan if e is None else 2.0 ** e

    def sums(self):
        """``[hkv, tiles, 128]``: each tile's keys added up."""
        return tile_sums(self.values[0])


def tile_sums(k):
    return np.asarray(k, np.float64).reshape(-1, TILE, *k.shape[1:]).sum(1).transpose(1, 0, 2)


def key_ends(rows: int, n_keys: int, row_pos0: int, mask=None):
    """Keys that each row sees, always the first ones; mask: None or (prompt_len, block)."""
    p = row_pos0 + np.arange(rows)
    if mask is None:
        return np.full(rows, n_keys)
    prompt, block = mask
    return np.minimum(n_keys, np.where(p < prompt, prompt,
                                       prompt + ((p - prompt) // block + 1) * block))


def select_blocks(q, sums, ends, *, block: int, count: int, sinks: int = 0, local: int = 1):
    """int32 ``[rows, hkv, count]``: forced blocks and the best scores, ascending, -1 behind."""
    q = np.asarray(q, np.float64)
    rows, hq, _ = q.shape
    hkv, tiles, _ = sums.shape
    m = block // TILE
    out = np.full((rows, hkv, count), -1, np.int32)
    for r in range(rows):
        n = -(-int(ends[r]) // block)
        for h in range(hkv):
            if n <= count:
                out[r, h, :n] = np.arange(n)
                continue
            mid = np.arange(sinks, n - local)
            whole = sums[h, :(n - 1) * m].reshape(n - 1, m, 128).sum(1)
            g = hq // hkv
            score = whole[mid] @ q[r, h * g:(h + 1) * g].sum(0)
            score = np.where(np.isnan(score), np.inf, score)
            best = mid[np.lexsort((mid, -score))][:count - sinks - local]
            out[r, h] = np.sort(np.concatenate([np.arange(sinks), best,
                                                np.arange(n - local, n)]))
    return out


def attention(q, k, v, ends, blocks=None, block: int = 0):
    """(out, weight) ``[rows, hq, 128]``: softmax(q k^T / sqrt(128)) v over each row's first
    ``ends`` keys (those of its listed blocks), and the same sum of |v|. No key: zeros."""
    q = np.asarray(q, np.float64)
    rows, hq, _ = q.shape
    hkv = k.shape[1]
    out, weight = np.zeros((2, rows, hq, 128))
    for r in range(rows):
        for h in range(hq):
            kv = h // (hq // hkv)
            keys = np.arange(ends[r])
            if blocks is not None:
                keys = keys[np.isin(keys // block, blocks[r, kv])]  # (a list is a set)
            if not len(keys):
                continue
            s = k[keys, kv] @ q[r, h] * 128 ** -0.5
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h] = p @ v[keys, kv]
            weight[r, h] = p @ np.abs(v[keys, kv])
    return out, weight


def attention_bound(q, k, v, ends, weight, p_half: float, n_keys: int, *, q_bf16_scaled=False,
                    scales8=(0.0, 0.0)):
    """How far a kernel's fp32 result may be from :func:`attention`'s, from its roundings.

    - a weighted value p is rounded once to the product's type: ``p_half`` of it (2^-11 for
      fp16, 2^-8 for bf16), or below fp16's normal numbers 2^-25 absolute against a largest of
      at least 1, times a code of at most 127 where the tile's largest is over 63: 2^-24 of the
      largest |v| per key;
    - a score is a sum of 128 exact products in fp32, and two more roundings: 130 * 2^-24 of
      the sum of their magnitudes, in the exponent, so that times p; once in p, once in the
      normaliser; exp2 and the sums over keys in fp32 add (n_keys / 32 + 64) * 2^-24;
    - over 8 bits (scales8: the largest scales of a tile's K and V) both go into the products as
      bytes code + 128 <= 255, and 128 times the sum of the query, or of the weights, is taken off:
      |k| is up to 128 scales larger, and O an fp32 sum of up to 255 scales instead of |v|,
      which a product rounds at most once a key and a fold once more (a tile's sum of weights: 32
      times), 2 n_keys times in all;
    - bf16 queries that are scaled to fp16 lose at most 2^-25 of the vector's largest each.

    From a few thousand keys on this is wider than a tile's part of the result (8224 keys: 0.020,
    results 0.018): it holds, but tells little there. :func:`attention_limit` does.
    """
    q = np.abs(np.asarray(q, np.float64))
    k, v = np.abs(np.nan_to_num(k)), np.abs(np.nan_to_num(v))
    kmax = k.max(0) + 128 * scales8[0]                                   # [hkv, 128]
    g = q.shape[1] // k.shape[1]
    s = (q * kmax.repeat(g, 0)[None]).sum(-1) * 128 ** -0.5              # [rows, hq]
    e = 130 * 2.0 ** -24 * s
    if q_bf16_scaled:
        e = e + 128 ** -0.5 * 2.0 ** -25 * q.max(-1) * kmax.sum(-1).repeat(g)[None]
    rel = p_half + 2 * e + (n_keys / 32 + 64) * 2.0 ** -24
    floor = n_keys * 2.0 ** -24 * v.max() + (2 * n_keys + 4) * 2.0 ** -24 * 255 * scales8[1]
    return rel[..., None] * weight + floor


def attention_terms(q, k, v, ends, scales=None, blocks=None, block: int = 0):
    """:func:`attention` with what :func:`attention_limit` is made of, for each (row, head):

    - out, weight ``[rows, hq, 128]`` as :func:`attention`;
    - keys: how many it attends to; score: the largest sum of |q| (|k| + 128 K scales) / sqrt(128)
      of one; kside: the largest sum of |k| + 128 K scales;
    - most: the largest p |code| scale (8 bits) or p |v|, at its largest |code| or |v|;
    - span: the sum of p 255 V scales (8 bits), 0 otherwise;
    - tiles ``[rows, hq, tiles]``: what each tile of keys has of the weights' sum (1).

    scales: ``[hkv, tiles, 2]`` of an 8-bit cache."""
    q = np.asarray(q, np.float64)
    rows, hq, _ = q.shape
    n, hkv, _ = k.shape
    g, pad = hq // hkv, -n % TILE
    t = {"out": np.zeros((rows, hq, 128)), "weight": np.zeros((rows, hq, 128)),
         "tiles": np.zeros((rows, hq, (n + pad) // TILE))}
    t |= {name: np.zeros((rows, hq)) for name in ("keys", "score", "kside", "most", "span")}
    key = np.arange(n)
    for h in range(hkv):
        seen = key[None] < np.asarray(ends)[:, None]
        if blocks is not None:
            hit = np.zeros((rows, -(-n // block)), bool)
            r, at = np.nonzero((blocks[:, h] >= 0) & (blocks[:, h] < hit.shape[1]))
            hit[r, blocks[r, h, at]] = True
            seen = seen & hit[:, key // block]
        sk, sv = np.zeros((2, n)) if scales is None else \
            np.repeat(scales[h], TILE, 0)[:n].T
        kk, vv = k[:, h], v[:, h]
        kabs = np.abs(kk) + 128 * sk[:, None]
        for j in range(g):
            i = h * g + j
            s = np.where(seen, q[:, i] @ kk.T * 128 ** -0.5, -np.inf)
            top = s.max(1)
            p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)[:, None]), 0.0)
            p /= np.maximum(p.sum(1), 1e-300)[:, None]
            t["out"][:, i], t["weight"][:, i] = p @ vv, p @ np.abs(vv)
            t["keys"][:, i] = seen.sum(1)
            t["score"][:, i] = np.where(seen, np.abs(q[:, i]) @ kabs.T * 128 ** -0.5, 0).max(1)
            t["kside"][:, i] = np.where(seen, kabs.sum(1), 0).max(1)
            t["most"][:, i] = (p * (127 * sv)).max(1) if scales is not None else \
                p.max(1) * np.abs(vv).max()
            t["span"][:, i] = 255 * (p @ sv)
            t["tiles"][:, i] = np.pad(p, ((0, 0), (0, pad))).reshape(rows, -1, TILE).sum(2)
    return t


def attention_limit(q, t, p_half: float, n_keys: int, ranges: int, *, q_bf16_scaled=False):
    """:func:`attention_bound` by what each (row, head) attends to: no more than the roundings can
    add up to there, so that a tile or a block left out passes it. ranges: the call's key ranges.

    - A wave has every fourth tile at most of a range, and no keys but the row's own weigh more than
      zero: ``keys`` of a wave below. What it sums is rounded once a key, the weights' sum of 8
      bits as often, both once more a tile (a fold, or a change of base), and joined with the other
      waves' and ranges' (64 roundings and 64 more at most). As every rounding is at most
      half a step of a partial sum of magnitudes, and the waves' sums of magnitudes add up to the
      row's, that is so many times 2^-24 of ``weight`` or, over 8 bits, of ``span``.
    - A weight is rounded to the product's type: ``p_half`` of it, or 2^-25 of a unit that is no
      more than the largest of its wave: ``most`` for each key.
    - Scores as in attention_bound, with the sums of one key's magnitudes for those of the
      largest of every head dim."""
    q = np.abs(np.asarray(q, np.float64))
    e = 130 * 2.0 ** -24 * t["score"]
    if q_bf16_scaled:
        e = e + 128 ** -0.5 * 2.0 ** -25 * q.max(-1) * t["kside"]
    wave = np.minimum(t["keys"], TILE * ((-(-n_keys // TILE)) // (4 * ranges) + 2))
    steps = (2 * wave + 2 * (wave / TILE + 1) + 128) * 2.0 ** -24
    rel = p_half + 2 * e + steps
    floor = t["keys"] * 2.0 ** -25 * t["most"] + steps * t["span"]
    return rel[..., None] * t["weight"] + floor[..., None]
