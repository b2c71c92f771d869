"""What the paged cache's C entries refuse, on the CPU."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from diffusorrt_amd import _lib
from diffusorrt_amd.paged import PagedKVCache

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")


def test_no_event_is_refused():
    assert _lib.load().drt_event_wait(None) == _lib.INVALID_ARGUMENT


def _plan(page_size, pages, hq, hkv, keys=(1,), rows=(1,), table=None, width=1):
    n = len(keys)
    i32 = C.c_int32 * n
    table = (C.c_int32 * (n * width))() if table is None else table
    info = _lib.PagedBatch()
    status = _lib.load().drt_paged_plan(
        C.addressof(table) if isinstance(table, C.Array) else table.ctypes.data, width, n, i32(*rows),
        i32(*keys), i32(*[k - r for k, r in zip(keys, rows)]), None, page_size, pages, hq, hkv,
        _lib.MASK_BIDIRECTIONAL, 1, None, 0, info)
    return status, info


@pytest.mark.parametrize("page_size, pages, hkv", [
    (2**25, 2**30, 2**14),      # 2^20 * 2^30 * 2^14 tiles: 2^64
    (2**30, 2**30, 2**14),      # 2^69
    (2**30, 2**31 - 1, 2**13),  # a product whose 64 bits are negative
    (32, 2**31 - 1, 2), (2**30, 64, 1)])
def test_layers_of_more_tiles_than_31_bits_are_refused(page_size, pages, hkv):
    status, _ = _plan(page_size, pages, hkv, hkv)
    assert status == _lib.INVALID_ARGUMENT and "tiles" in _lib.last_error()


def test_the_largest_layer_is_taken():
    assert _plan(32, 2**31 - 1, 7, 1)[0] == _lib.OK
    assert _plan(2**30, 63, 1, 1)[0] == _lib.OK


def test_lists_of_more_pages_than_31_bits_are_refused():
    # 33 sequences of 2^26 - 2 pages each (one page again and again: zeros that no memory stands behind)
    width = 2**26 - 2
    table = np.zeros(33 * width, dtype=np.int32)
    status, _ = _plan(32, 1, 1, 1, keys=[width * 32 - 1] * 33, rows=[1] * 33, table=table, width=width)
    assert status == _lib.INVALID_ARGUMENT and "pages" in _lib.last_error()


def test_numpy_heads():
    cache = PagedKVCache(1, 2, 4, device="cpu")
    assert cache.batch([[1]], [3], [1], heads=np.int64(4)).heads == 4
    for bad in (np.float64(4), True, np.True_, "4", None):
        with pytest.raises(ValueError, match="whole number"):
            cache.batch([[1]], [3], [1], heads=bad)
