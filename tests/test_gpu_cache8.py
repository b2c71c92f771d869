"""The 8-bit cache and the block-sparse attention on the GPU, against the float64 oracle
(oracle/cache8.py). Whole numbers and stored values are compared exactly; attention within the
bound that its roundings give (``attention_bound``). Each test prints its case first."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import cache8 as X

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"i8": 2.0 ** -11, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of the product's type


def _say(*a):
    print("[case]", *a, flush=True)


def _np(t):
    return t.detach().double().cpu().numpy()


def _kv(gen, n, hkv, scale=1.0):
    return (torch.randn((n, hkv, 128), generator=gen) * scale for _ in range(2))


def _filled(gen, n, hkv, dtype, capacity=None, block_sums=True):
    """(cache with n rows of layer 1, its k and v in float64, the cache's shape of tiles)."""
    from diffusorrt_amd.kernels import PrefixKVCache

    cache = PrefixKVCache(2, hkv, capacity or n, dtype=dtype, block_sums=block_sums)
    k, v = _kv(gen, n, hkv)
    cache.store(1, k.cuda(), v.cuda(), 0)
    if dtype == "i8":
        ref = X.Cache8(hkv, cache.capacity)
        ref.store(k.numpy(), v.numpy(), 0)
        return cache, ref.values[0], ref.values[1]
    pad = torch.zeros((cache.capacity - n, hkv, 128))
    return (cache, *(_np(torch.cat([x, pad]).to(TDT[dtype])) for x in (k, v)))


def _scales(cache, layer):
    """The largest scales of a tile's K and V of an 8-bit cache, for attention_bound."""
    if cache.scales is None:
        return (0.0, 0.0)
    x = torch.nan_to_num(cache.scales[layer]).amax((0, 1))
    return float(x[0]), float(x[1])


def _check(got, out, bound, out_dtype):
    g = _np(got).reshape(out.shape)
    last = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24
    tol = bound + last * (np.abs(out) + bound)
    bad = np.abs(g - out) > tol
    worst = float((np.abs(g - out) / np.maximum(tol, 1e-300)).max())
    _say(f"  largest error / bound = {worst:.3f}")
    assert np.isfinite(g).all() and not bad.any(), worst


# ---------------------------------------------------------------- store, load, sums

def _same_as(cache, layer, ref):
    k, v = cache.load(layer, 0, cache.capacity)
    for got, want in ((k, ref.values[0]), (v, ref.values[1])):
        np.testing.assert_array_equal(_np(got), want)
    written = cache.sums is not None
    np.testing.assert_array_equal(_np(cache.scales[layer]), ref.scales)
    if written:
        np.testing.assert_array_equal(_np(cache.sums[layer]), ref.sums())


@pytest.mark.parametrize("stores", [[(0, 1)], [(0, 32)], [(5, 3)], [(31, 2)], [(0, 128)],
                                    [(17, 70)], [(0, 40), (40, 1), (41, 55)],
                                    [(0, 128), (64, 32)], [(0, 100), (30, 5), (90, 38)]])
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_store_quantizes_tiles_as_a_whole(stores, src):
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("store", stores, src)
    gen = torch.Generator().manual_seed(len(stores) * 7 + stores[0][1])
    cache, ref = PrefixKVCache(2, 3, 128, dtype="i8", block_sums=True), X.Cache8(3, 128)
    for i, (pos0, n) in enumerate(stores):
        k, v = (x.to(TDT[src]) for x in _kv(gen, n, 3, 4.0 ** i))
        cache.store(1, k.cuda(), v.cuda(), pos0)
        ref.store(_np(k), _np(v), pos0)
    assert bool((cache.data[0] == 128).all())  # the other layer
    _same_as(cache, 1, ref)
    assert cache.length == max(p + n for p, n in stores)


def test_store_of_single_rows_of_growing_size():
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("store rows one by one")
    rng = np.random.default_rng(9)
    cache, ref = PrefixKVCache(1, 2, 64, dtype="i8", block_sums=True), X.Cache8(2, 64)
    for r in list(range(40)) + [3, 35, 3]:
        k, v = (rng.standard_normal((1, 2, 128)).astype(np.float32) * np.float32(1.3) ** r
                for _ in range(2))
        cache.store(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), r)
        ref.store(k, v, r)
    _same_as(cache, 0, ref)


def test_store_at_the_ends_of_the_scales_and_beyond():
    """Zeros, denormal and tiny values, exactly 127 * 2^e, the largest that fits; NaN and
    infinity and one step beyond the largest make their tile, and no other, NaN."""
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("store extremes")
    most = [0.0, 1e-42, 1e-30, 127 * 2.0 ** -40, 127 * 2.0 ** -39, 127.0, 127.00001, 63.5, 254.0,
            127 * 2.0 ** 40, 127.1 * 2.0 ** 40, 3e38, np.inf, -np.inf, np.nan, 1.0]
    x = np.random.default_rng(2).uniform(-1, 1, (32 * len(most), 1, 128)).astype(np.float32)
    for t, m in enumerate(most):
        tile = x[32 * t:32 * t + 32]
        with np.errstate(all="ignore"):
            tile *= np.float32(m if np.isfinite(m) else 1.0)
        tile[7, 0, 9] = m
    y = np.ones_like(x)
    cache, ref = PrefixKVCache(1, 1, len(x), dtype="i8", block_sums=True), X.Cache8(1, len(x))
    cache.store(0, torch.from_numpy(x).cuda(), torch.from_numpy(y).cuda(), 0)
    ref.store(x, y, 0)
    _same_as(cache, 0, ref)
    assert int(torch.isnan(cache.scales[0, 0, :, 0]).sum()) == 5
    # a NaN tile stays NaN until every row of it is new
    t = most.index(3e38)
    cache.store(0, torch.ones((31, 1, 128)).cuda(), torch.ones((31, 1, 128)).cuda(), 32 * t)
    assert bool(torch.isnan(cache.load(0, 32 * t, 32)[0]).all())
    cache.store(0, torch.ones((32, 1, 128)).cuda(), torch.ones((32, 1, 128)).cuda(), 32 * t)
    assert bool((cache.load(0, 32 * t, 32)[0] == 1).all())


def test_a_cleared_cache_serves_another_sequence():
    """Large and NaN rows of the sequence before have no part in the next one's scales."""
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("clear")
    gen = torch.Generator().manual_seed(31)
    cache, ref = PrefixKVCache(2, 2, 96, dtype="i8", block_sums=True), X.Cache8(2, 96)
    k, v = _kv(gen, 96, 2, 1000.0)
    k[70] = float("nan")
    cache.store(1, k.cuda(), v.cuda(), 0)
    assert bool(torch.isnan(cache.scales).any())
    cache.clear()
    k, v = _kv(gen, 70, 2, 1.0)
    for at, n in ((0, 40), (40, 1), (41, 29)):
        cache.store(1, k[at:at + n].cuda(), v[at:at + n].cuda(), at)
        ref.store(_np(k[at:at + n]), _np(v[at:at + n]), at)
    _same_as(cache, 1, ref)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_load_and_sums_of_a_16_bit_cache(dtype):
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("load", dtype)
    gen = torch.Generator().manual_seed(5)
    cache = PrefixKVCache(2, 3, 160, dtype=dtype, block_sums=True)
    plain = PrefixKVCache(2, 3, 160, dtype=dtype)
    want = torch.zeros((2, 160, 3, 128))
    for pos0, n in ((0, 70), (70, 1), (71, 60), (40, 5)):
        k, v = _kv(gen, n, 3)
        for c in (cache, plain):
            c.store(1, k.cuda(), v.cuda(), pos0)
        for w, x in enumerate((k, v)):
            want[w, pos0:pos0 + n] = x.to(TDT[dtype]).float()
    assert torch.equal(cache.data, plain.data) and plain.sums is None
    for odt in (torch.float32, torch.bfloat16):
        k, v = cache.load(1, 33, 100, out_dtype=odt)
        assert torch.equal(k.cpu(), want[0, 33:133].to(odt))
        assert torch.equal(v.cpu(), want[1, 33:133].to(odt))
    sums = X.tile_sums(want[0].double().numpy()).astype(np.float32)
    np.testing.assert_array_equal(cache.sums[1].cpu().numpy(), sums)


# ---------------------------------------------------------------- attention over 8 bits

@pytest.mark.parametrize("rows,hq,hkv,n_keys,pos0,mask,qdt,odt", [
    (1, 2, 1, 1, 0, None, "f16", "f32"),            # one key
    (1, 28, 4, 33, 32, None, "bf16", "bf16"),       # one token, one key of a second tile
    (1, 7, 1, 1000, 999, None, "f16", "f32"),       # one token over key ways and ranges
    (9, 28, 4, 1337, 1328, None, "bf16", "bf16"),   # two query tiles, the second nearly full
    (32, 16, 8, 2080, 2048, (0, 32), "f16", "f32"),
    (32, 8, 4, 8224, 8192, (0, 32), "bf16", "f32"),
    (5, 40, 2, 300, 295, (0, 1), "f16", "f32"),     # causal; 20 heads a group
    (64, 4, 2, 700, 636, (0, 32), "f16", "bf16"),   # four query tiles
    (70, 4, 2, 70, 0, (0, 32), "f16", "f32"),       # five: ragged in rows and keys
    (97, 4, 4, 128, 31, (10, 32), "bf16", "f32"),   # blocks off the tile grid
    (300, 4, 1, 300, 0, (100, 8), "f16", "f32"),    # a prompt, then blocks inside tiles
    (257, 2, 2, 513, 256, None, "f16", "f32"),
    (40, 2, 1, 64, 0, (64, 32), "f16", "f32"),      # every row sees the prompt only
    (3, 2, 1, 40, 100, (0, 32), "f16", "f32"),      # rows behind the keys
])
def test_attention_over_8_bits(rows, hq, hkv, n_keys, pos0, mask, qdt, odt):
    _say("attention i8", rows, hq, hkv, n_keys, pos0, mask, qdt, odt)
    gen = torch.Generator().manual_seed(rows + n_keys)
    cache, k, v = _filled(gen, n_keys, hkv, "i8")
    q = torch.randn((rows, hq, 128), generator=gen).to(TDT[qdt])
    got = cache.attention(1, q.cuda(), n_keys=n_keys, row_pos0=pos0,
                          kind="full" if mask is None else "d2f_hybrid", mask_geometry=mask,
                          out_dtype=TDT[odt])
    ends = X.key_ends(rows, n_keys, pos0, mask)
    out, weight = X.attention(_np(q), k, v, ends)
    bound = X.attention_bound(_np(q), k, v, ends, weight, HALF["i8"], n_keys,
                              q_bf16_scaled=qdt == "bf16", scales8=_scales(cache, 1))
    _check(got, out, bound, TDT[odt])


def test_attention_of_the_kernel_table_over_8_bits():
    from diffusorrt_amd.kernels import KernelTable

    _say("attention(kv_dtype=i8)")
    gen = torch.Generator().manual_seed(6)
    k, v = _kv(gen, 96, 2)
    q = torch.randn((32, 4, 128), generator=gen).half()
    got = KernelTable().attention(q.cuda(), k.cuda(), v.cuda(), head_dim=128, kind="full",
                                  kv_dtype="i8")
    ref = X.Cache8(2, 96)
    ref.store(k.numpy(), v.numpy(), 0)
    ends = X.key_ends(32, 96, 64)
    out, weight = X.attention(_np(q), *ref.values, ends)
    bound = X.attention_bound(_np(q), *ref.values, ends, weight, HALF["i8"], 96,
                              scales8=ref.scales.max((0, 1)))
    assert got.dtype == torch.float16 and got.shape == (32, 512)
    assert (np.abs(_np(got).reshape(out.shape) - out)
            <= bound + 2.0 ** -11 * (np.abs(out) + bound)).all()


@pytest.mark.parametrize("rows,sparse", [(2, False), (200, False), (2, True)])
def test_tiles_of_very_different_scales(rows, sparse):
    """V tiles from 1e-11 to 1e9 and zero, K tiles zero and large: a row's weights lie on tiles of
    any size, and small results beside large ones keep their own precision only as far as the
    large ones' weight lets them."""
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("scale spread", rows, sparse)
    gen = torch.Generator().manual_seed(8)
    n = 32 * 12
    k, v = _kv(gen, n, 1)
    sizes = [0.0, 1e-11, 1.0, 1e9, 0.0, 1e-6, 1e3, 0.0, 1e-11, 1e-3, 1e-9, 0.0]
    for t, s in enumerate(sizes):
        v[32 * t:32 * t + 32] *= s
    k[64:128] = 0.0
    k[320:] *= 30.0
    cache, ref = PrefixKVCache(1, 1, n, dtype="i8"), X.Cache8(1, n)
    cache.store(0, k.cuda(), v.cuda(), 0)
    ref.store(k.numpy(), v.numpy(), 0)
    q = torch.randn((rows, 2, 128), generator=gen).half() * 3
    for n_keys in (32, 64, 96, 352, n):
        ends = X.key_ends(rows, n_keys, 0)
        blocks = np.arange(n_keys // 32, dtype=np.int32)[None, None].repeat(rows, 0)
        if sparse:
            got = cache.sparse_attention(0, q.cuda(), torch.from_numpy(blocks).cuda(),
                                         block_size=32, n_keys=n_keys, row_pos0=0, kind="full")
        else:
            got = cache.attention(0, q.cuda(), n_keys=n_keys, row_pos0=0, kind="full")
        k8, v8 = ref.values[0][:n_keys], ref.values[1][:n_keys]
        out, weight = X.attention(_np(q), k8, v8, ends)
        _check(got, out, X.attention_bound(_np(q), k8, v8, ends, weight, HALF["i8"], n_keys,
                                            scales8=ref.scales[:, :n_keys // 32].max((0, 1))),
               torch.float32)


@pytest.mark.parametrize("qsize", [1e-38, 1e-20, 1e20, 5e37])
def test_bf16_queries_of_any_size(qsize):
    _say("bf16 q *", qsize)
    gen = torch.Generator().manual_seed(12)
    cache, k, v = _filled(gen, 96, 1, "i8")
    q = (torch.randn((3, 2, 128), generator=gen) * qsize).bfloat16()
    q[1, 0] = 0
    blocks = torch.arange(3, dtype=torch.int32).expand(3, 1, 3).contiguous()
    for got in (cache.attention(1, q.cuda(), n_keys=90, row_pos0=0, kind="full"),
                cache.sparse_attention(1, q.cuda(), blocks.cuda(), block_size=32, n_keys=90,
                                       row_pos0=0, kind="full")):
        ends = X.key_ends(3, 90, 0)
        out, weight = X.attention(_np(q), k, v, ends)
        if qsize > 1:  # one key takes all: its row of V, unless two scores are within a few units
            assert np.isfinite(_np(got)).all()
            s = np.einsum("rhd,kd->rhk", _np(q), k[:90, 0]) * 128 ** -0.5
            order = np.sort(s, -1)
            sure = order[..., -1] - order[..., -2] > 1e-3 * np.abs(s).max(-1)
            assert sure.sum() >= 3
            off = np.abs(_np(got).reshape(out.shape) - out).max(-1)
            assert (off[sure] <= 2.0 ** -20 * np.abs(out).max()).all()
        else:
            _check(got, out, X.attention_bound(_np(q), k, v, ends, weight, HALF["i8"], 90,
                                               q_bf16_scaled=True, scales8=_scales(cache, 1)),
                   torch.float32)


@pytest.mark.parametrize("dtype", ["i8", "f16", "bf16"])
def test_nan_reaches_the_rows_that_see_it_only(dtype):
    """Rows of blocks of 32: a NaN key or value in block 2 reaches rows of blocks 2 and later;
    rows behind n_keys hold NaN and infinity and reach none; a NaN query its own heads."""
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("nan", dtype)
    gen = torch.Generator().manual_seed(13)
    for where in ("k", "v"):
        cache = PrefixKVCache(1, 1, 160, dtype=dtype)
        k, v = _kv(gen, 160, 1)
        (k if where == "k" else v)[70, 0, 5] = float("nan")
        if dtype != "i8":  # (an 8-bit tile is NaN as a whole: these lie in one of their own)
            k[120:] = float("nan")
            v[120:] = float("inf")
        else:
            k[128:] = float("nan")
            v[128:] = float("inf")
        cache.store(0, k.cuda(), v.cuda(), 0)
        n_keys = 120
        q = torch.randn((120, 2, 128), generator=gen).to(TDT.get(dtype, torch.float16))
        q[3, 1, 0] = float("nan")
        blocks = torch.arange(4, dtype=torch.int32).expand(120, 1, 4).contiguous().cuda()
        kw = dict(n_keys=n_keys, row_pos0=0, kind="d2f_hybrid", mask_geometry=(0, 32))
        outs = [cache.sparse_attention(0, q.cuda(), blocks, block_size=32, **kw)]
        if dtype == "i8":  # (many rows and few)
            outs += [cache.attention(0, q.cuda(), **kw),
                     torch.cat([cache.attention(0, q[r:r + 8].contiguous().cuda(),
                                                **(kw | {"row_pos0": r}))
                                for r in range(0, 120, 8)])]
        for got in outs:
            nan = torch.isnan(got.view(120, 2, 128)).any(-1).cpu()
            whole = torch.isnan(got.view(120, 2, 128)).all(-1).cpu()
            want = torch.zeros((120, 2), dtype=torch.bool)
            want[64:] = True
            want[3, 1] = True
            assert torch.equal(nan, want)
            if dtype == "i8" or where == "k":  # (a NaN of V in 16 bits is one head dim's)
                assert torch.equal(whole, want)


@pytest.mark.parametrize("dtype", ["i8", "f16", "bf16"])
def test_values_that_are_not_finite_stay_with_the_rows_that_list_them(dtype):
    """16 neighbouring rows, which the kernel takes together, list the 16 subsets of four blocks. V
    of block 1 has infinities and a NaN, K of block 3 a NaN; row 16 on lists them all."""
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("not finite", dtype)
    gen = torch.Generator().manual_seed(17)
    cache = PrefixKVCache(1, 1, 128, dtype=dtype)
    k, v = _kv(gen, 128, 1)
    clean = v.clone(), k.clone()
    v[40, 0, 3], v[41, 0, 4], v[63, 0, 5] = float("inf"), -float("inf"), float("nan")
    k[100, 0, 7] = float("nan")
    cache.store(0, k.cuda(), v.cuda(), 0)
    blocks = np.full((32, 1, 4), -1, np.int32)
    for r in range(32):
        mine = [b for b in range(4) if r >= 16 or r >> b & 1]
        blocks[r, 0, :len(mine)] = mine
    q = torch.randn((32, 2, 128), generator=gen).to(TDT.get(dtype, torch.float16))
    q[0, 1, 0] = float("nan")  # (row 0 lists nothing: zeros)
    got = cache.sparse_attention(0, q.cuda(), torch.from_numpy(blocks).cuda(), block_size=32,
                                 n_keys=128, row_pos0=0, kind="full")
    got = _np(got).reshape(32, 2, 128)
    if dtype == "i8":
        ref = X.Cache8(1, 128)
        ref.store(clean[1].numpy(), clean[0].numpy(), 0)
        k8, v8 = ref.values
    else:
        k8, v8 = (_np(x.to(TDT[dtype])) for x in (clean[1], clean[0]))
    ends = X.key_ends(32, 128, 0)
    qn = np.nan_to_num(_np(q))
    out, weight = X.attention(qn, k8, v8, ends, blocks, 32)
    bound = X.attention_bound(qn, k8, v8, ends, weight, HALF[dtype], 128,
                              scales8=_scales(cache, 0))
    for r in range(32):
        lists = set(blocks[r, 0].tolist())
        if 3 in lists or (dtype == "i8" and 1 in lists):
            assert np.isnan(got[r]).all(), r
            continue
        ok = np.ones(128, bool)
        if 1 in lists:
            assert (got[r, :, 3] == np.inf).all() and (got[r, :, 4] == -np.inf).all()
            assert np.isnan(got[r, :, 5]).all()
            ok[3:6] = False
        assert (np.abs(got[r] - out[r]) <= bound[r] * 1.001)[:, ok].all(), r
    assert not got[0].any()


def test_attention_over_more_8_bit_keys_than_4_gib_hold():
    from diffusorrt_amd.kernels import PrefixKVCache

    keys, rows = (1 << 24) + 4096, 40  # 256 bytes a key: one head passes 4 GiB
    _say("attention i8 over", keys, "keys")
    cache = PrefixKVCache(1, 1, keys, dtype="i8", block_sums=True)
    # K is zero, so every key weighs the same; V differs from zero in the last 4096 keys only
    v = torch.randn((4096, 1, 128), generator=torch.Generator().manual_seed(38)).cuda() * 1000
    cache.store(0, torch.zeros_like(v), v, keys - 4096)
    held = cache.load(0, keys - 4096, 4096)[1][:, 0].double()
    for rows in (2, 300):
        q = torch.randn((rows, 1, 128), device="cuda").half()
        y = cache.attention(0, q, n_keys=keys, row_pos0=keys - rows, kind="full").double()
        want = held.sum(0) / keys
        # weights of one over 2^24 keys; sums in fp32 over tiles, ranges and their joining
        assert ((y - want).norm(dim=1) <= 1e-4 * want.norm()).all()
    q = torch.randn((2, 1, 128), device="cuda").half()
    last = keys // 4096 - 1
    blocks = torch.tensor([[[last]], [[0]]], dtype=torch.int32, device="cuda")
    y = cache.sparse_attention(0, q, blocks, block_size=4096, n_keys=keys, row_pos0=0,
                               kind="full").double()
    assert ((y[0] - held.mean(0)).norm() <= 1e-3 * held.mean(0).norm()) and not y[1].any()
    cache.sums[0, 0, -128:, 3] = torch.arange(128, device="cuda")
    q.zero_()
    q[:, 0, 3] = 1
    got = cache.select_blocks(0, q, block_size=32, count=3, n_keys=keys, row_pos0=0, kind="full")
    n = keys // 32
    assert got[0, 0].tolist() == [n - 3, n - 2, n - 1]


# ---------------------------------------------------------------- selection

@pytest.mark.parametrize("rows,hq,hkv,n_keys,pos0,mask,qdt,dtype,block,count,sinks,local", [
    (1, 4, 2, 32, 0, None, "f16", "i8", 32, 1, 0, 1),          # one block
    (3, 4, 2, 70, 0, None, "f16", "i8", 32, 5, 1, 1),          # fewer than listed
    (33, 8, 4, 1000, 967, (0, 32), "bf16", "i8", 32, 7, 0, 1),
    (20, 28, 4, 2000, 100, (0, 8), "f16", "f16", 64, 9, 2, 3),
    (17, 4, 1, 3000, 2983, None, "bf16", "bf16", 96, 10, 0, 1),
    (40, 4, 2, 9000, 4500, (33, 50), "f16", "i8", 32, 16, 1, 2),  # 282 blocks
    (5, 2, 2, 40000, 39990, None, "f16", "i8", 32, 100, 0, 1),    # 1250
    (3, 2, 1, 70000, 69990, None, "f16", "f16", 32, 60, 0, 1),    # 2188
    (5, 2, 1, 640, 0, None, "f16", "i8", 32, 4, 2, 2),            # nothing left to score
    # enough rows and heads for one launch: 47, 375 and 938 blocks, and none to score
    (260, 8, 8, 3000, 2740, (0, 32), "bf16", "bf16", 64, 12, 1, 2),
    (257, 16, 8, 12000, 5000, (2, 40), "f16", "i8", 32, 20, 0, 1),
    (250, 8, 8, 30000, 29750, None, "f16", "i8", 32, 33, 3, 1),
    (700, 4, 4, 700, 0, (0, 1), "f16", "i8", 32, 5, 0, 1),
    (256, 8, 8, 100, 0, None, "f16", "i8", 32, 4, 0, 1),
    # as many blocks as one launch takes for few rows, and one more
    (3, 7, 1, 4096, 4090, None, "f16", "f16", 32, 9, 1, 2),
    (19, 4, 2, 4097, 4000, (5, 9), "bf16", "i8", 32, 9, 1, 2),
    (2, 4, 2, 12288, 12000, None, "f16", "i8", 96, 40, 0, 3),
])
def test_select_blocks(rows, hq, hkv, n_keys, pos0, mask, qdt, dtype, block, count, sinks, local):
    _say("select", rows, hq, hkv, n_keys, pos0, mask, qdt, dtype, block, count, sinks, local)
    gen = torch.Generator().manual_seed(rows + n_keys)
    cache, k, _ = _filled(gen, n_keys, hkv, dtype, capacity=n_keys + 40)
    q = torch.randn((rows, hq, 128), generator=gen).to(TDT[qdt])
    got = cache.select_blocks(1, q.cuda(), block_size=block, count=count, n_keys=n_keys,
                              row_pos0=pos0, kind="full" if mask is None else "d2f_hybrid",
                              mask_geometry=mask, sinks=sinks, local=local)
    sums = X.tile_sums(k).astype(np.float32).astype(np.float64)
    want = X.select_blocks(_np(q), sums, X.key_ends(rows, n_keys, pos0, mask), block=block,
                           count=count, sinks=sinks, local=local)
    assert got.dtype == torch.int32
    np.testing.assert_array_equal(got.cpu().numpy(), want)


# (blocks and rows: each of the kernels' forms)
@pytest.mark.parametrize("n,rows", [(100, 4), (400, 4), (700, 4), (1500, 4), (2500, 4), (100, 2048),
                                    (400, 2048), (700, 2048)])
def test_select_blocks_with_equal_and_nan_scores(n, rows):
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("select ties", n, rows)
    cache = PrefixKVCache(1, 1, 32 * n, dtype="f16", block_sums=True)
    rng = np.random.default_rng(n)
    sums = np.zeros((1, n, 128))
    sums[0, :, 0] = rng.integers(-2, 3, n)
    sums[0, :, 1] = -0.0
    q = torch.zeros((4, 1, 128), dtype=torch.float16)
    q[0, 0, 0], q[1, 0, 0], q[2, 0, 1] = 1.0, -0.5, 1.0  # (row 2: zeros of both signs)
    q[3, 0, 2] = 1.0
    sums[0, rng.integers(0, n - 1, 5), 2] = np.nan
    sums[0, rng.integers(0, n - 1, 5), 3] = -np.inf
    ends = X.key_ends(4, 32 * n, 0)
    cache.sums[0] = torch.from_numpy(sums).float().cuda()
    got = cache.select_blocks(0, q.repeat(rows // 4, 1, 1).cuda(), block_size=32, count=20,
                              n_keys=32 * n, row_pos0=0, kind="full")
    with np.errstate(invalid="ignore"):
        want = X.select_blocks(_np(q), sums, ends, block=32, count=20)
    np.testing.assert_array_equal(got.cpu().numpy(), np.tile(want, (rows // 4, 1, 1)))


def test_select_never_hears_of_hidden_keys():
    """A row's blocks stay the same whatever lies behind the keys it sees."""
    _say("select hidden")
    gen = torch.Generator().manual_seed(3)
    cache, _, _ = _filled(gen, 1024, 2, "i8")
    q = torch.randn((32, 4, 128), generator=gen).half().cuda()
    kw = dict(block_size=64, count=4, row_pos0=512, kind="d2f_hybrid", mask_geometry=(0, 32))
    a = cache.select_blocks(1, q, n_keys=1024, **kw)
    k, v = _kv(gen, 480, 2, 50.0)
    cache.store(1, k.cuda(), v.cuda(), 544)
    assert torch.equal(a, cache.select_blocks(1, q, n_keys=1024, **kw))
    assert torch.equal(a, cache.select_blocks(1, q, n_keys=544, **kw))


# ---------------------------------------------------------------- attention over blocks

@pytest.mark.parametrize("dtype", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("rows,hq,hkv,n_keys,pos0,mask,qdt,odt,block,count", [
    (1, 2, 1, 1, 0, None, "f16", "f32", 32, 1),
    (1, 28, 4, 1337, 1336, None, "bf16", "bf16", 64, 8),      # key ranges
    (9, 28, 4, 1000, 991, None, "f16", "f32", 32, 5),         # odd tiles: pairs across blocks
    (33, 16, 8, 1100, 1067, (0, 32), "bf16", "f32", 96, 4),
    (70, 4, 2, 70, 0, (0, 32), "f16", "f32", 64, 3),
    (45, 40, 2, 300, 255, (7, 5), "f16", "f32", 32, 6),       # 20 heads a group
    (600, 8, 4, 600, 0, (0, 1), "f16", "bf16", 32, 4),        # one range, causal
    (5, 4, 1, 70000, 69995, None, "f16", "f32", 32, 40),      # more blocks than a bitmap holds
    (1100, 2, 1, 1100, 0, None, "bf16", "bf16", 32, 3),       # 16 rows a tile, four ways
    (40, 1, 1, 900, 860, (3, 7), "f16", "f32", 64, 5),        # one head a group: 32 rows a tile
])
def test_sparse_attention(dtype, rows, hq, hkv, n_keys, pos0, mask, qdt, odt, block, count):
    if dtype != "i8":
        qdt = dtype
    _say("sparse", dtype, rows, hq, hkv, n_keys, pos0, mask, qdt, odt, block, count)
    gen = torch.Generator().manual_seed(rows + n_keys)
    cache, k, v = _filled(gen, n_keys, hkv, dtype)
    q = torch.randn((rows, hq, 128), generator=gen).to(TDT[qdt])
    kw = dict(block_size=block, n_keys=n_keys, row_pos0=pos0,
              kind="full" if mask is None else "d2f_hybrid", mask_geometry=mask)
    blocks = cache.select_blocks(1, q.cuda(), count=count, **kw)
    got = cache.sparse_attention(1, q.cuda(), blocks, out_dtype=TDT[odt], **kw)
    ends = X.key_ends(rows, n_keys, pos0, mask)
    out, weight = X.attention(_np(q), k, v, ends, blocks.cpu().numpy(), block)
    bound = X.attention_bound(_np(q), k, v, ends, weight, HALF[dtype], n_keys,
                              q_bf16_scaled=dtype == "i8" and qdt == "bf16",
                              scales8=_scales(cache, 1))
    _check(got, out, bound, TDT[odt])


@pytest.mark.parametrize("dtype", ["i8", "f16"])
@pytest.mark.parametrize("rows", [6, 3000])  # with key ranges and without
def test_sparse_attention_of_lists_of_any_origin(dtype, rows):
    """Unsorted, repeated, negative and far entries, an empty list, a list longer than a wave's
    64 lanes, a block behind the row's keys and one the row's end cuts."""
    _say("sparse lists", dtype, rows)
    gen = torch.Generator().manual_seed(21)
    n_keys, count = 3000, 130
    cache, k, v = _filled(gen, n_keys, 1, dtype, capacity=3008)
    q = torch.randn((rows, 2, 128), generator=gen).half()
    rng = np.random.default_rng(5)
    blocks = rng.integers(-3, 110, (rows, 1, count)).astype(np.int32)
    blocks[0] = -1
    blocks[1, 0] = [2**31 - 1, -2**31] + [0] * (count - 2)
    blocks[2, 0] = np.arange(count)[::-1]
    blocks[3, 0] = np.arange(count)
    blocks[4, 0, :5], blocks[4, 0, 5:] = [93, 93, 94, 93, 200], -1
    blocks[5, 0, :70], blocks[5, 0, 70:] = 1, np.arange(60) * 2
    pos0 = 2900
    kw = dict(block_size=32, n_keys=n_keys, row_pos0=pos0, kind="d2f_hybrid",
              mask_geometry=(2950, 24))
    got = cache.sparse_attention(1, q.cuda(), torch.from_numpy(blocks).cuda(), **kw)
    some = slice(0, 6)
    ends = X.key_ends(rows, n_keys, pos0, (2950, 24))
    out, weight = X.attention(_np(q[some]), k, v, ends[some], blocks[some], 32)
    _check(got[some], out, X.attention_bound(_np(q[some]), k, v, ends[some], weight, HALF[dtype],
                                             n_keys, scales8=_scales(cache, 1)), torch.float32)
    assert not got[0].any() and got[1].any()


def test_all_blocks_are_dense_attention():
    _say("sparse = dense")
    gen = torch.Generator().manual_seed(31)
    cache, _, _ = _filled(gen, 2048, 2, "i8")
    q = torch.randn((40, 4, 128), generator=gen).half().cuda()
    kw = dict(n_keys=2048, row_pos0=2000, kind="d2f_hybrid", mask_geometry=(0, 32))
    blocks = cache.select_blocks(1, q, block_size=128, count=16, **kw)
    a = cache.sparse_attention(1, q, blocks, block_size=128, **kw)
    b = cache.attention(1, q, **kw)
    assert ((a - b).abs() <= 2 * 2.0 ** -10 * b.abs().max()).all()  # (both within 2^-11 of the values' weight)


# ---------------------------------------------------------------- as a program uses them

def _step(cache, k, v, q, w, pos0, n_keys):
    """One layer's attention of a block: its rows stored, their blocks chosen, attention over
    them and over all, the output projection of both."""
    from diffusorrt_amd.kernels import KernelTable

    rows = q.shape[0]
    kw = dict(n_keys=n_keys, row_pos0=pos0, kind="d2f_hybrid", mask_geometry=(0, 32))
    cache.store(0, k, v, pos0)
    blocks = cache.select_blocks(0, q, block_size=64, count=5, sinks=1, **kw)
    a = cache.sparse_attention(0, q, blocks, block_size=64, out_dtype=torch.bfloat16, **kw)
    b = cache.attention(0, q, out_dtype=torch.bfloat16, **kw)
    assert a.shape[0] == rows
    return blocks, a, b, KernelTable().linear(a, w), KernelTable().linear(b, w)


@pytest.mark.parametrize("dtype", ["i8", "f16"])
def test_a_blocks_step_against_the_oracle(dtype):
    from diffusorrt_amd.kernels import DeviceBF16Weight, PrefixKVCache

    _say("step", dtype)
    gen = torch.Generator().manual_seed(41)
    prefix, rows = 1000, 24  # the block's rows begin inside a tile
    cache, ref = PrefixKVCache(1, 2, 1024, dtype=dtype, block_sums=True), X.Cache8(2, 1024)
    k, v = (x.bfloat16() for x in _kv(gen, 1024, 2))
    w = (torch.randn((256, 512), generator=gen) * 0.05).bfloat16()
    cache.store(0, k[:prefix].cuda().contiguous(), v[:prefix].cuda().contiguous(), 0)
    q = torch.randn((rows, 4, 128), generator=gen).half()
    blocks, a, b, ya, yb = _step(cache, k[prefix:].cuda(), v[prefix:].cuda(), q.cuda(),
                                 DeviceBF16Weight(w.cuda()), prefix, 1024)
    if dtype == "i8":
        ref.store(_np(k[:prefix]), _np(v[:prefix]), 0)
        ref.store(_np(k[prefix:]), _np(v[prefix:]), prefix)
        k8, v8 = ref.values
    else:
        k8, v8 = _np(k.half()), _np(v.half())
    ends = X.key_ends(rows, 1024, prefix, (0, 32))
    sums = X.tile_sums(k8).astype(np.float32).astype(np.float64)
    want = X.select_blocks(_np(q), sums, ends, block=64, count=5, sinks=1)
    np.testing.assert_array_equal(blocks.cpu().numpy(), want)
    for got, y, lists in ((a, ya, want), (b, yb, None)):
        out, weight = X.attention(_np(q), k8, v8, ends, lists, 64)
        bound = X.attention_bound(_np(q), k8, v8, ends, weight, HALF[dtype], 1024,
                                  scales8=_scales(cache, 0))
        if dtype == "i8" or lists is not None:
            _check(got, out, bound, torch.bfloat16)
        # the projection of what came out: half a bf16 step and the fp32 sums
        x = _np(got)
        exact, mag = x @ _np(w).T, np.abs(x) @ np.abs(_np(w)).T
        assert (np.abs(_np(y) - exact) <= np.abs(exact) * 2.0 ** -8 + mag * 512 * 2.0 ** -24).all()


def test_a_step_captured_and_replayed():
    """One graph of the whole step, replayed over new inputs with eager work between, bit for
    bit as the eager calls; two graphs in turn keep workspaces of their own."""
    from diffusorrt_amd.kernels import DeviceBF16Weight, PrefixKVCache

    _say("graph")
    gen = torch.Generator().manual_seed(51)
    caches = [PrefixKVCache(1, 2, 4096, dtype="i8", block_sums=True) for _ in range(3)]
    k0, v0 = (x.cuda() for x in _kv(gen, 4064, 2))
    for c in caches:
        c.store(0, k0, v0, 0)
    w = DeviceBF16Weight((torch.randn((256, 512), generator=gen) * 0.05).bfloat16().cuda())
    k, v = (x.cuda() for x in _kv(gen, 32, 2))
    q = torch.randn((32, 4, 128), generator=gen).half().cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in caches:
            _step(c, k, v, q, w, 4064, 4096)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in caches[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(c, k, v, q, w, 4064, 4096))
        graphs.append(g)
    for i in range(4):
        gen = torch.Generator().manual_seed(60 + i)
        k.copy_(torch.randn(k.shape, generator=gen) * (i + 1))
        v.copy_(torch.randn(v.shape, generator=gen))
        q.copy_(torch.randn(q.shape, generator=gen))
        for g in graphs if i % 2 else graphs[::-1]:
            g.replay()
        want = _step(caches[2], k, v, q, w, 4064, 4096)
        torch.cuda.synchronize()
        for got in outs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    _say("two streams")
    gen = torch.Generator().manual_seed(71)
    cache, _, _ = _filled(gen, 4096, 2, "i8")
    q = torch.randn((32, 4, 128), generator=gen).half().cuda()
    kw = dict(n_keys=4096, row_pos0=4064, kind="full")

    def work():
        b = cache.select_blocks(1, q, block_size=64, count=8, **kw)
        return b, cache.sparse_attention(1, q, b, block_size=64, **kw), cache.attention(1, q, **kw)

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_refusals():
    from diffusorrt_amd.kernels import PrefixKVCache

    _say("refusals")
    cache = PrefixKVCache(1, 2, 128, dtype="i8", block_sums=True)
    half = PrefixKVCache(1, 2, 128, dtype="f16")
    q = torch.zeros((4, 4, 128), dtype=torch.float16, device="cuda")
    x = torch.zeros((4, 2, 128), device="cuda")
    b = torch.zeros((4, 2, 3), dtype=torch.int32, device="cuda")
    at = dict(n_keys=64, row_pos0=0, kind="full")
    sel = dict(block_size=32, count=2) | at
    sp = dict(block_size=32) | at
    bad = [
        lambda: cache.store(1, x, x, 0), lambda: cache.store(0, x, x, 126),
        lambda: cache.store(0, x[:0], x[:0], 0), lambda: cache.store(0, x.half(), x.half(), 0),
        lambda: cache.store(0, x.cpu(), x.cpu(), 0), lambda: cache.store(0, x[:, :1], x[:, :1], 0),
        lambda: cache.store(0, x.transpose(0, 1), x.transpose(0, 1), 0),
        lambda: cache.load(0, 100, 29), lambda: cache.load(0, -1, 2), lambda: cache.load(0, 0, 0),
        lambda: cache.load(2, 0, 4), lambda: cache.load(0, 0, 4, out_dtype=torch.float16),
        lambda: cache.attention(0, q.float(), **at), lambda: cache.attention(0, q[:, :3], **at),
        lambda: cache.attention(0, q[:0], **at), lambda: cache.attention(1, q, **at),
        lambda: cache.attention(0, q, **(at | {"n_keys": 129})),
        lambda: cache.attention(0, q, **(at | {"n_keys": 0})),
        lambda: cache.attention(0, q, **(at | {"row_pos0": -1})),
        lambda: cache.attention(0, q, **(at | {"row_pos0": 2**31 - 2})),
        lambda: cache.attention(0, q, **(at | {"kind": "causal"})),
        lambda: cache.attention(0, q, **(at | {"kind": "d2f_hybrid"})),
        lambda: cache.attention(0, q, out_dtype=torch.float16, **at),
        lambda: cache.attention(0, q[..., :64].contiguous(), **at),
        lambda: half.select_blocks(0, q, **sel),
        lambda: cache.select_blocks(0, q, **(sel | {"block_size": 48})),
        lambda: cache.select_blocks(0, q, **(sel | {"count": 0})),
        lambda: cache.select_blocks(0, q, **(sel | {"count": 1025})),
        lambda: cache.select_blocks(0, q, sinks=2, **sel),
        lambda: cache.select_blocks(0, q, local=0, **sel),
        lambda: cache.select_blocks(0, q, **(sel | {"n_keys": 200})),
        lambda: cache.sparse_attention(0, q, b.long(), **sp),
        lambda: cache.sparse_attention(0, q, b[:3], **sp),
        lambda: cache.sparse_attention(0, q, b.cpu(), **sp),
        lambda: cache.sparse_attention(0, q, b[:, :, :0], **sp),
        lambda: cache.sparse_attention(0, q, b[:, :, :2], **sp),
        lambda: cache.sparse_attention(0, q, b, **(sp | {"block_size": 0})),
        lambda: half.sparse_attention(0, q.bfloat16(), b, **sp),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            _say("not refused:", i)
