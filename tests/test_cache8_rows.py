"""Attention over an 8-bit cache and over listed blocks at the sizes of prompts, long prefixes and
key ranges, within a limit that a tile of keys left out passes. The tests without a GPU take each
tile out of the reference and look whether the limit would tell; those on the GPU hold the kernels
to it. Every tile's V is large in one head dim (``_inputs``), so that each has its say."""
from __future__ import annotations

import functools

import numpy as np
import pytest

from diffusorrt_amd import _lib
from oracle import cache8 as X

torch = pytest.importorskip("torch")

TDT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"i8": 2.0 ** -11, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of the product's type

# rows, hq, hkv, keys, first row's position, mask, queries, out
DENSE = [
    (1, 28, 4, 1337, 1336, None, "bf16", "f32"),
    (1, 28, 4, 8192, 8191, None, "f16", "bf16"),         # one token, key ranges
    (9, 28, 4, 1337, 1328, None, "f16", "f32"),
    (32, 16, 8, 8224, 8192, (0, 32), "bf16", "f32"),     # a block, key ranges
    (64, 4, 2, 5000, 4936, (0, 32), "f16", "f32"),
    (97, 4, 4, 1280, 1183, (10, 32), "bf16", "f32"),     # blocks off the tile grid
    # many rows: work-groups of two query tiles (384 and more of them: 416, 400, 388, 400)
    (400, 64, 32, 431, 31, (5, 24), "bf16", "f32"),      # 25 query tiles a head, the last alone
    (1600, 16, 8, 1633, 33, (40, 32), "f16", "bf16"),
    (880, 28, 4, 900, 20, (0, 1), "bf16", "bf16"),       # causal, seven heads a group
    (1540, 16, 16, 700, 0, None, "f16", "f32"),          # rows behind the keys, one head a group
]

# cache, rows, hq, hkv, keys, first row's position, mask, queries over 8 bits, out, block, count
LISTED = [
    (9, 28, 4, 20000, 19991, None, "f16", "f32", 64, 16),        # key ranges
    (32, 16, 8, 9000, 8968, (0, 32), "bf16", "f32", 64, 32),
    (5, 4, 1, 70000, 69995, None, "f16", "f32", 32, 40),         # two windows of blocks
    (3, 40, 1, 400, 397, None, "bf16", "f32", 32, 6),            # 40 heads a group: two tiles
    (9, 66, 2, 3000, 2991, None, "f16", "bf16", 96, 20),         # 33: one alone, key ranges
    # more than 256 work-groups: four waves each (608, 520, 300, 400)
    (600, 32, 16, 700, 100, (7, 40), "bf16", "f32", 32, 5),
    (1030, 16, 8, 1100, 70, (0, 32), "f16", "bf16", 64, 6),
    (300, 28, 4, 2000, 1700, (3, 7), "f16", "f32", 96, 4),
    (200, 33, 1, 900, 700, None, "bf16", "f32", 32, 12),
]
TYPES = ["i8", "f16", "bf16"]


def _inputs(case, dtype, rows, hq, hkv, n, qdt):
    """(q, k, v) as float32 arrays of the types the call takes; tile t's V larger by 8 in one
    head dim, another one for each 128 tiles in a row."""
    rng = np.random.default_rng(case)
    q = rng.standard_normal((rows, hq, 128), np.float32)
    k, v = rng.standard_normal((2, n, hkv, 128), np.float32)
    t = np.arange(n) // X.TILE
    v[np.arange(n), :, t * 37 % 128] += 8.0
    q = torch.from_numpy(q).to(TDT[qdt])
    return q, torch.from_numpy(k), torch.from_numpy(v)


def _held(k, v, dtype):
    """The rows as a cache of the type reads them, and its scales."""
    if dtype != "i8":
        return (*(x.to(TDT[dtype]).double().numpy() for x in (k, v)), None)
    ref = X.Cache8(k.shape[1], len(k))
    ref.store(k.numpy(), v.numpy(), 0)
    return ref.values[0][:len(k)], ref.values[1][:len(k)], ref.scales


def _lists(case, rows, hkv, ends, block, count):
    """Each row's last block and others it sees, half of them its neighbours' too, -1 behind."""
    rng = np.random.default_rng(1000 + case)
    out = np.full((rows, hkv, count), -1, np.int32)
    for r in range(rows):
        n = -(-int(ends[r]) // block)
        if r % 8 == 0:
            common = rng.random((hkv, -(-int(ends.max()) // block)))
        for h in range(hkv):
            score = common[h, :n] + (rng.random(n) < 4 / n)
            score[n - 1] = 3.0
            best = np.argsort(-score)[:count]
            out[r, h, :len(best)] = np.sort(best)
    return out


@functools.lru_cache(maxsize=1)
def _dense(i):
    rows, hq, hkv, n, pos0, mask, qdt, _ = DENSE[i]
    q, k, v = _inputs(i, "i8", rows, hq, hkv, n, qdt)
    return q, k, v, X.key_ends(rows, n, pos0, mask), None


@functools.lru_cache(maxsize=1)
def _listed(i, dtype):
    rows, hq, hkv, n, pos0, mask, qdt, _, block, count = LISTED[i]
    q, k, v = _inputs(100 + i, dtype, rows, hq, hkv, n, qdt if dtype == "i8" else dtype)
    ends = X.key_ends(rows, n, pos0, mask)
    return q, k, v, ends, _lists(i, rows, hkv, ends, block, count)


def _ranges(name, rows, hq, *rest):
    """Key ranges of a call, from the workspace it asks for (130 fp32 a range, row and head)."""
    if not _lib.LIB_PATH.exists():
        from diffusorrt_amd import build
        build.build()
    return max(1, getattr(_lib.load(), name)(rows, hq, *rest) // (rows * hq * 130 * 4))


def _dense_ranges(i):
    rows, hq, hkv, n = DENSE[i][:4]
    return _ranges("drt_op_attention_kv8_workspace_bytes", rows, hq, hkv, n)


def _listed_ranges(i):
    rows, hq, hkv, block, count = *LISTED[i][:3], *LISTED[i][8:]
    return _ranges("drt_op_sparse_attention_workspace_bytes", rows, hq, hkv, block, count)


def _limit(q, t, dtype, n, ranges, out_dtype):
    qd = q.double().numpy()
    limit = X.attention_limit(qd, t, HALF[dtype], n, ranges,
                              q_bf16_scaled=dtype == "i8" and q.dtype == torch.bfloat16)
    last = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24
    return limit + last * (np.abs(t["out"]) + limit)


# ---------------------------------------------------------------- the limits, without a GPU

def _each_tile_has_its_say(q, k, v, ends, lists, block, dtype, ranges, out_dtype):
    """A few rows' results without any one tile of keys, and, for lists, any one listed block:
    further from the whole one than the limit in at least one row that sees it."""
    rows, hq, n = q.shape[0], q.shape[1], len(k)
    some = np.unique(np.linspace(0, rows - 1, 12).astype(int))
    k, v, scales = _held(k, v, dtype)
    mine = None if lists is None else lists[some]
    t = X.attention_terms(q[some].double().numpy(), k, v, ends[some], scales, mine, block)
    tol = _limit(q[some], t, dtype, n, ranges, out_dtype)
    worst = np.full(t["tiles"].shape[2], np.inf)
    for h in range(hq):
        kv = h // (hq // k.shape[1])
        for tile in range(len(worst)):
            share = t["tiles"][:, h, tile]
            if not share.any():
                continue
            lo, hi = tile * X.TILE, min(n, tile * X.TILE + X.TILE)
            s = q[some, h].double().numpy() @ k[lo:hi, kv].T * 128 ** -0.5
            p = np.exp(s - s.max(1)[:, None])
            p[np.arange(lo, hi)[None] >= ends[some][:, None]] = 0
            p *= (share / np.maximum(p.sum(1), 1e-300))[:, None]
            whole = np.maximum(1 - share, 1e-300)[:, None]
            off = (t["out"][:, h] - p @ v[lo:hi, kv]) / whole - t["out"][:, h]
            ratio = (np.abs(off) / tol[:, h]).max()
            worst[tile] = ratio if worst[tile] == np.inf else max(worst[tile], ratio)
    assert worst.min() > 2, worst.min()


@pytest.mark.parametrize("i", range(len(DENSE)))
def test_the_limit_tells_a_tile_left_out(i):
    q, k, v, ends, _ = _dense(i)
    _each_tile_has_its_say(q, k, v, ends, None, 0, "i8", _dense_ranges(i), TDT[DENSE[i][7]])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(LISTED)))
def test_the_limit_tells_a_tile_of_a_list_left_out(i, dtype):
    q, k, v, ends, lists = _listed(i, dtype)
    _each_tile_has_its_say(q, k, v, ends, lists, LISTED[i][8], dtype, _listed_ranges(i),
                           TDT[LISTED[i][7]])


def test_terms_are_those_of_attention():
    rng = np.random.default_rng(7)
    q, (k, v) = rng.standard_normal((5, 6, 128)), rng.standard_normal((2, 100, 2, 128))
    ends = np.array([1, 40, 100, 99, 64])
    lists = rng.integers(-2, 5, (5, 2, 3))
    lists[4] = -1
    for args in ((), (lists, 32)):
        t = X.attention_terms(q, k, v, ends, None, *args)
        out, weight = X.attention(q, k, v, ends, *args)
        np.testing.assert_allclose(t["out"], out, rtol=1e-12, atol=1e-13)
        np.testing.assert_allclose(t["weight"], weight, rtol=1e-12, atol=1e-13)
        sums = t["tiles"].sum(2)
        assert np.all((np.abs(sums - 1) < 1e-12) | ((sums == 0) & (t["keys"] == 0)))


# ---------------------------------------------------------------- the kernels

def _say(*a):
    print("[case]", *a, flush=True)


def _cache(k, v, dtype):
    from diffusorrt_amd.kernels import PrefixKVCache

    cache = PrefixKVCache(1, k.shape[1], len(k), dtype=dtype)
    cache.store(0, k.cuda(), v.cuda(), 0)
    return cache


def _call(cache, q, n, pos0, mask, out_dtype, lists=None, block=0):
    kw = dict(n_keys=n, row_pos0=pos0, kind="full" if mask is None else "d2f_hybrid",
              mask_geometry=mask, out_dtype=out_dtype)
    if lists is None:
        y = cache.attention(0, q.cuda(), **kw)
    else:
        y = cache.sparse_attention(0, q.cuda(), torch.from_numpy(lists).cuda(), block_size=block,
                                   **kw)
    return y.double().cpu().numpy().reshape(q.shape)


def _within(got, t, tol, rows=slice(None)):
    ratio = np.abs(got - t["out"])[rows] / np.maximum(tol[rows], 1e-300)
    _say(f"  largest error / limit = {ratio.max():.3f}")
    assert np.isfinite(got[rows]).all() and ratio.max() <= 1, ratio.max()


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(DENSE)))
def test_attention_of_rows(i):
    rows, hq, hkv, n, pos0, mask, qdt, odt = DENSE[i]
    _say("attention i8", *DENSE[i], "ranges", _dense_ranges(i))
    q, k, v, ends, _ = _dense(i)
    got = _call(_cache(k, v, "i8"), q, n, pos0, mask, TDT[odt])
    t = X.attention_terms(q.double().numpy(), *_held(k, v, "i8")[:2], ends, _held(k, v, "i8")[2])
    _within(got, t, _limit(q, t, "i8", n, _dense_ranges(i), TDT[odt]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(LISTED)))
def test_listed_blocks_of_rows(i, dtype):
    rows, hq, hkv, n, pos0, mask, _, odt, block, count = LISTED[i]
    _say("listed", dtype, *LISTED[i], "ranges", _listed_ranges(i))
    q, k, v, ends, lists = _listed(i, dtype)
    got = _call(_cache(k, v, dtype), q, n, pos0, mask, TDT[odt], lists, block)
    kh, vh, scales = _held(k, v, dtype)
    t = X.attention_terms(q.double().numpy(), kh, vh, ends, scales, lists, block)
    _within(got, t, _limit(q, t, dtype, n, _listed_ranges(i), TDT[odt]))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["dense", "i8", "f16", "bf16"])
def test_many_rows_over_tiles_of_very_different_scales(form):
    """V tiles from 1e-9 to 1e9 and zero, K tiles zero and large, over the many-row kernels (416
    work-groups of two query tiles; 800 of a list's)."""
    rows, hq, hkv, n = 400, 64, 32, 32 * 12
    _say("scale spread", form)
    dtype = "i8" if form == "dense" else form
    rng = np.random.default_rng(5)
    q = torch.from_numpy(rng.standard_normal((rows, hq, 128), np.float32)).to(
        TDT[dtype] if dtype != "i8" else torch.float16) * 3
    k, v = (torch.from_numpy(rng.standard_normal((n, hkv, 128), np.float32)) for _ in range(2))
    sizes = [0.0, 1e-9, 1.0, 1e9, 0.0, 1e-6, 1e3, 0.0, 1e-9, 1e-3, 1e-7, 0.0]
    for at, s in enumerate(sizes):
        v[32 * at:32 * at + 32] *= s if dtype != "f16" else min(s, 1e3)
    k[64:128] = 0.0
    k[320:] *= 30.0
    cache = _cache(k, v, dtype)
    kh, vh, scales = _held(k, v, dtype)
    for n_keys in (32, 64, 96, 352, n):
        ends = X.key_ends(rows, n_keys, 0)
        lists = None if form == "dense" else \
            np.tile(np.arange(n_keys // 32, dtype=np.int32), (rows, hkv, 1))
        got = _call(cache, q, n_keys, 0, None, torch.float32, lists, 32)
        t = X.attention_terms(q.double().numpy(), kh[:n_keys], vh[:n_keys], ends,
                              None if scales is None else scales[:, :n_keys // 32], lists, 32)
        _within(got, t, _limit(q, t, dtype, n_keys, 1, torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("form", ["dense", "i8", "f16", "bf16"])
def test_nan_among_many_rows_reaches_those_that_see_it(form, where):
    """Blocks of 32 rows under the mask: a NaN key or value in block 2 reaches rows 64 and on, a NaN
    query its own head; what is not finite behind n_keys reaches none. The other rows keep their
    results."""
    rows, hq, hkv, n = 416, 64, 32, 448
    n_keys = 416
    _say("nan", form, where)
    dtype = "i8" if form == "dense" else form
    rng = np.random.default_rng(13)
    q = torch.from_numpy(rng.standard_normal((rows, hq, 128), np.float32)).to(
        TDT[dtype] if dtype != "i8" else torch.bfloat16)
    k, v = (torch.from_numpy(rng.standard_normal((n, hkv, 128), np.float32)) for _ in range(2))
    held = _held(k, v, dtype)
    (k if where == "k" else v)[70, :, 5] = float("nan")
    k[n_keys:], v[n_keys:] = float("nan"), float("inf")
    q_nan = q.clone()
    q_nan[3, 1, 0] = float("nan")
    lists = None if form == "dense" else \
        np.tile(np.arange(n_keys // 32, dtype=np.int32), (rows, hkv, 1))
    got = _call(_cache(k, v, dtype), q_nan, n_keys, 0, (0, 32), torch.float32, lists, 32)
    want = np.zeros((rows, hq), bool)
    want[64:] = True
    want[3, 1] = True
    np.testing.assert_array_equal(np.isnan(got).any(2), want)
    if dtype == "i8" or where == "k":  # (a NaN of V in 16 bits is one head dim's)
        np.testing.assert_array_equal(np.isnan(got).all(2), want)
    else:
        assert np.isfinite(got[64:, :, :5]).all() and np.isfinite(got[64:, :, 6:]).all()
    ends = X.key_ends(rows, n_keys, 0, (0, 32))
    some = np.r_[0:3, 4:64]
    t = X.attention_terms(q.double().numpy()[some], held[0][:n_keys], held[1][:n_keys], ends[some],
                          None if held[2] is None else held[2][:, :n_keys // 32],
                          None if lists is None else lists[some], 32)
    _within(got[some], t, _limit(q[some], t, dtype, n_keys, 1, torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,hq,hkv,blocks", [
    (600, 32, 16, 20),    # four waves a work-group
    (40, 8, 4, 20),       # eight, key ranges
    (6, 8, 4, 2200),      # two windows of blocks, key ranges
    (520, 16, 1, 2200),   # two windows, four waves
])
def test_values_that_are_not_finite_among_lists(dtype, rows, hq, hkv, blocks):
    """Neighbouring rows, every third of which lists two blocks (of each window, if there are two)
    with infinities and a NaN in V and every fifth one with a NaN in K; the others keep theirs."""
    _say("not finite", dtype, rows, hq, hkv, blocks)
    n, count = 32 * blocks, 12
    rng = np.random.default_rng(blocks + rows)
    q = torch.from_numpy(rng.standard_normal((rows, hq, 128), np.float32)).to(TDT[dtype])
    k, v = (torch.from_numpy(rng.standard_normal((n, hkv, 128), np.float32)) for _ in range(2))
    kh, vh, _ = _held(k, v, dtype)
    odd, nan = (1, blocks - 2), blocks - 4
    for b in odd:
        v[32 * b + 9, :, 3], v[32 * b + 30, :, 4] = float("inf"), -float("inf")
        v[32 * b + 17, :, 5] = float("nan")
    k[32 * nan + 11, :, 7] = float("nan")
    free = np.setdiff1d(np.arange(blocks), (*odd, nan))
    lists = np.full((rows, hkv, count), -1, np.int32)
    for r in range(rows):
        for h in range(hkv):
            lists[r, h, :9] = rng.choice(free, 9, replace=False)
            if r % 3 == 0:
                lists[r, h, 9:11] = odd
            if r % 5 == 0:
                lists[r, h, 11] = nan
    got = _call(_cache(k, v, dtype), q, n, 0, None, torch.float32, lists, 32)
    ends = X.key_ends(rows, n, 0)
    r = np.arange(rows)
    assert np.isnan(got[r % 5 == 0]).all()
    mine = got[(r % 3 == 0) & (r % 5 != 0)]
    assert (mine[..., 3] == np.inf).all() and (mine[..., 4] == -np.inf).all()
    assert np.isnan(mine[..., 5]).all()
    some = np.unique(np.linspace(0, rows - 1, 64).astype(int))
    t = X.attention_terms(q[some].double().numpy(), kh, vh, ends[some], None, lists[some], 32)
    tol = _limit(q[some], t, dtype, n, _ranges("drt_op_sparse_attention_workspace_bytes", rows, hq,
                                               hkv, 32, count), torch.float32)
    off = ~(np.abs(got[some] - t["out"]) <= tol)
    off[some % 5 == 0] = False
    off[some % 3 == 0, :, 3:6] = False
    assert not off.any(), np.argwhere(off)[:5]
