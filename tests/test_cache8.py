"""The 8-bit cache and the block-sparse attention without a GPU: the oracle's definitions on
closed forms, and the entry points' refusals, which come before any device work (the
pointers here are never followed)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from diffusorrt_amd import _lib
from oracle import cache8 as X

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from diffusorrt_amd import build
        build.build()
    return _lib.load()


# ---------------------------------------------------------------- the definitions

@pytest.mark.parametrize("most,e", [(0.0, -40), (127.0, 0), (127.00001, 1), (63.5, -1), (254.0, 1),
                                    (1.0, -6), (127 * 2.0 ** 40, 40), (2.0 ** -60, -40)])
def test_exponent_is_the_least_that_holds(most, e):
    assert X.exponent(most) == e


@pytest.mark.parametrize("most", [np.inf, np.nan, 127.01 * 2.0 ** 40])
def test_tiles_beyond_the_range_are_nan(most):
    assert X.exponent(most) is None


def test_stores_of_a_tile_stay_within_one_step():
    """Rows written one by one, each larger than all before: every store requantizes."""
    rng = np.random.default_rng(3)
    cache, rows = X.Cache8(1, 32), []
    for r in range(32):
        x = rng.standard_normal((1, 1, 128)) * 1.5 ** r
        rows.append(x)
        cache.store(x, -x, r)
        for w, sign in ((0, 1), (1, -1)):
            off = np.abs(cache.values[w, :r + 1] - sign * np.concatenate(rows))
            assert off.max() < cache.scales[0, 0, w]
    # a tile stored whole forgets what was there
    x = rng.standard_normal((32, 1, 128))
    cache.store(x, x, 0)
    assert np.abs(cache.values[0] - x).max() <= cache.scales[0, 0, 0] / 2


def test_select_takes_forced_blocks_then_scores_then_lower_blocks():
    q = np.zeros((3, 2, 128))
    q[:, :, 0] = 0.5
    sums = np.zeros((1, 10, 128))
    sums[0, :, 0] = [5, 1, 7, 7, 1, 7, 0, 9, 9, 9]
    ends = X.key_ends(3, 320, 0, None)
    ends[1], ends[2] = 65, 8 * 32
    got = X.select_blocks(q, sums, ends, block=32, count=4, sinks=1, local=1)
    assert got[0, 0].tolist() == [0, 7, 8, 9]
    assert got[1, 0].tolist() == [0, 1, 2, -1]
    assert got[2, 0].tolist() == [0, 2, 3, 7]  # 7 ties 2, 3 and 5: the lower two


def test_a_list_is_a_set():
    rng = np.random.default_rng(4)
    q, k, v = rng.standard_normal((1, 1, 128)), *rng.standard_normal((2, 128, 1, 128))
    ends = np.array([100])
    a = X.attention(q, k, v, ends, np.array([[[3, 1, 1, -5, 3, 9]]]), 32)[0]
    b = X.attention(q, k, v, ends, np.array([[[1, 3]]]), 32)[0]
    assert np.array_equal(a, b)
    assert not X.attention(q, k, v, ends, np.array([[[-1, 4, 9]]]), 32)[0].any()


# ---------------------------------------------------------------- refusals at the C-ABI

P = 0x10000  # (an address; nothing reads it)


def _store(**kw):
    a = dict(k=P, v=P, src=_lib.F32, n=32, hkv=2, pos0=0, cache=P, stride=8192 * 4, scales=P,
             sums=None, stream=None) | kw
    return "drt_op_kv8_store", list(a.values())


def _store16(**kw):
    a = dict(k=P, v=P, src=_lib.F32, n=32, hkv=2, pos0=0, cache=P, stride=8192 * 4,
             dtype=_lib.F16, sums=P, stream=None) | kw
    return "drt_op_kv16_store", list(a.values())


def _load(**kw):
    a = dict(cache=P, stride=8192 * 4, dtype=_lib.I8, scales=P, n=32, hkv=2, pos0=0, k=P, v=P,
             out=_lib.F32, stream=None) | kw
    return "drt_op_kv_load", list(a.values())


def _attend(**kw):
    a = dict(q=P, qdt=_lib.F16, cache=P, stride=8192 * 128, scales=P, rows=8, hq=4, hkv=2,
             n_keys=4096, pos0=0, mask=_lib.MASK_D2F_HYBRID, prompt=0, block=32, out=P,
             odt=_lib.F32, ws=P, ws_bytes=1 << 40, stream=None) | kw
    return "drt_op_attention_kv8", list(a.values())


def _select(**kw):
    a = dict(q=P, qdt=_lib.F16, sums=P, tiles=4, rows=8, hq=4, hkv=2, n_keys=128, pos0=0,
             mask=_lib.MASK_D2F_HYBRID, prompt=0, block=32, size=32, count=4, sinks=0, local=1,
             blocks=P, ws=P, ws_bytes=1 << 40, stream=None) | kw
    return "drt_op_select_blocks", list(a.values())


def _sparse(**kw):
    a = dict(q=P, qdt=_lib.F16, cache=P, stride=8192 * 4, dtype=_lib.I8, scales=P, rows=8, hq=4,
             hkv=2, n_keys=128, pos0=0, mask=_lib.MASK_D2F_HYBRID, prompt=0, block=32, blocks=P,
             size=32, count=64, out=P, odt=_lib.F32, ws=P, ws_bytes=1 << 40, stream=None) | kw
    return "drt_op_sparse_attention", list(a.values())


REFUSED = (
    [_store(**kw) for kw in (
        {"k": None}, {"v": None}, {"cache": None}, {"scales": None}, {"src": _lib.F16}, {"n": 0},
        {"n": -1}, {"hkv": 0}, {"hkv": 70000}, {"pos0": -1}, {"pos0": 97}, {"n": 129},
        {"pos0": 2**31 - 1}, {"stride": 8192 * 4 + 1}, {"stride": 0}, {"cache": P + 8},
        {"scales": P + 4})]
    + [_store16(**kw) for kw in (
        {"k": None}, {"v": None}, {"cache": None}, {"sums": None}, {"dtype": _lib.I8}, {"n": 0},
        {"src": _lib.F16}, {"hkv": 0}, {"hkv": 70000}, {"pos0": 97}, {"pos0": -1},
        {"stride": 8192 * 4 - 8}, {"cache": P + 8})]
    + [_load(**kw) for kw in (
        {"cache": None}, {"k": None}, {"v": None}, {"scales": None}, {"dtype": _lib.F32},
        {"out": _lib.F16}, {"n": 0}, {"pos0": 97}, {"k": P + 4})]
    + [_attend(**kw) for kw in (
        {"q": None}, {"cache": None}, {"scales": None}, {"out": None}, {"ws": None},
        {"ws_bytes": 0}, {"qdt": _lib.F32}, {"odt": _lib.F16}, {"rows": 0}, {"hq": 5}, {"hkv": 0},
        {"n_keys": 0}, {"n_keys": 4097}, {"n_keys": 2**31 - 1}, {"pos0": -1}, {"pos0": 2**31 - 4},
        {"mask": 2}, {"block": 0}, {"prompt": -1}, {"q": P + 2}, {"out": P + 8}, {"ws": P + 8},
        {"rows": 2**30, "ws_bytes": 1 << 60})]
    + [_select(**kw) for kw in (
        {"q": None}, {"sums": None}, {"blocks": None},
        {"n_keys": 8192, "tiles": 256, "ws": None}, {"n_keys": 8192, "tiles": 256, "ws_bytes": 8},
        {"qdt": _lib.I8}, {"rows": 0}, {"hq": 3}, {"n_keys": 0}, {"n_keys": 129}, {"pos0": -1},
        {"size": 0}, {"size": 48}, {"size": -32}, {"count": 0}, {"count": 1025}, {"sinks": -1},
        {"local": 0}, {"sinks": 3, "local": 2}, {"sinks": 2**31 - 1, "local": 2**31 - 1},
        {"mask": 7}, {"block": 0}, {"ws": P + 4}, {"q": P + 8})]
    + [_sparse(**kw) for kw in (
        {"q": None}, {"cache": None}, {"scales": None}, {"blocks": None}, {"out": None},
        {"ws": None}, {"ws_bytes": 8}, {"dtype": _lib.F32}, {"dtype": _lib.BF16},
        {"qdt": _lib.F32}, {"rows": 0}, {"hq": 3}, {"n_keys": 0}, {"n_keys": 129}, {"pos0": -1},
        {"size": 16}, {"size": 0}, {"count": 0}, {"count": 1025}, {"mask": 7}, {"block": 0},
        {"odt": _lib.F16}, {"cache": P + 2})]
)


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refused_before_any_device_work(lib, i):
    name, args = REFUSED[i]
    assert getattr(lib, name)(*args) == _lib.INVALID_ARGUMENT, (name, args)
    assert _lib.last_error()


@pytest.mark.parametrize("name,args", [
    ("drt_op_attention_kv8_workspace_bytes", (0, 4, 2, 128)),
    ("drt_op_attention_kv8_workspace_bytes", (8, 5, 2, 128)),
    ("drt_op_select_blocks_workspace_bytes", (8, 2, 128, 33)),
    ("drt_op_sparse_attention_workspace_bytes", (8, 4, 2, 64, 0))])
def test_workspace_of_a_refused_shape_is_zero(lib, name, args):
    assert getattr(lib, name)(*args) == 0


def test_select_workspace_is_bounded(lib):
    assert 0 < lib.drt_op_select_blocks_workspace_bytes(1 << 20, 8, 1 << 20, 32) <= 1 << 28


def test_a_host_tensor_is_refused():
    from diffusorrt_amd.kernels import PrefixKVCache

    x = torch.zeros((4, 2, 128))
    for dtype in ("i8", "f16"):
        cache = PrefixKVCache(1, 2, 64, dtype=dtype, device="cpu", block_sums=True)
        with pytest.raises(ValueError):
            cache.store(0, x, x, 0)
        with pytest.raises(ValueError):
            cache.load(0, 0, 4)
        with pytest.raises(ValueError):
            cache.select_blocks(0, x.half(), block_size=32, count=1, n_keys=32, row_pos0=0,
                                kind="full")


@pytest.mark.parametrize("geometry", [(-1, 32), (0, 0), (2**31, 32), (0, 2**31), (2**32, 32),
                                      (0, 2**32 + 32)])
def test_mask_geometry_beyond_32_bits_is_refused(geometry):
    from diffusorrt_amd.kernels import _mask_args

    with pytest.raises(ValueError):
        _mask_args("d2f_hybrid", geometry)
    assert _mask_args("d2f_hybrid", (2**31 - 1, 2**31 - 1))[1:] == (2**31 - 1, 2**31 - 1)


@pytest.mark.parametrize("dtype", ["i8", "f16", "bf16"])
def test_clear_is_a_new_cache(dtype):
    from diffusorrt_amd.kernels import PrefixKVCache

    new, used = (PrefixKVCache(2, 3, 64, dtype=dtype, device="cpu", block_sums=True)
                 for _ in range(2))
    used.data.fill_(7)
    used.sums.fill_(float("nan"))
    if used.scales is not None:
        used.scales.fill_(float("nan"))
    used.length = 40
    used.clear()
    assert used.length == 0 and used.kv_dtype == new.kv_dtype
    for name in ("data", "scales", "sums"):
        a, b = getattr(new, name), getattr(used, name)
        assert (a is None) == (b is None)
        assert a is None or (a.dtype == b.dtype and torch.equal(a, b))


def test_an_8_bit_cache_is_half_the_bytes():
    from diffusorrt_amd.kernels import PrefixKVCache

    a, b = (PrefixKVCache(2, 4, 4096, dtype=d, device="cpu") for d in ("i8", "f16"))
    assert a.nbytes == b.nbytes // 2 + 2 * 4 * 128 * 8
    assert bool((a.data == 128).all()) and bool((a.scales == 1).all()) and a.sums is None
