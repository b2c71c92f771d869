"""Which kernel a batch's attention goes to, and whether its keys are cut, on the CPU: one batch of each
kind, looked at by itself."""
from __future__ import annotations

import numpy as np
import pytest

from diffusorrt_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")


def _plan(sequences, hq, hkv, page_size=64):
    """(the batch, its list) of sequences (keys, rows), the rows their last, causal."""
    keys, rows = (np.array(x, dtype=np.int32) for x in zip(*sequences))
    need = -(-keys // page_size)
    table = np.zeros((len(keys), need.max()), dtype=np.int32)
    for s, n in enumerate(need):
        table[s, :n] = need[:s].sum() + np.arange(n)
    pos0, words, info = keys - rows, np.zeros(1 << 18, dtype=np.int32), _lib.PagedBatch()
    _lib.check(_lib.load().drt_paged_plan(
        table.ctypes.data, table.shape[1], len(keys), rows.ctypes.data, keys.ctypes.data,
        pos0.ctypes.data, None, page_size, int(need.sum()), hq, hkv, _lib.MASK_D2F_HYBRID, 1,
        words.ctypes.data, words.size, info))
    assert info.words <= words.size
    return info, words


@pytest.mark.parametrize("sequences, hq, hkv, small, large, cut", [
    ([(40, 40)], 16, 8, True, False, False),
    ([(1337, 1)], 16, 8, True, False, True),
    ([(131072, 1)], 16, 8, True, False, True),
    ([(60000, 32)], 28, 4, True, False, True),
    ([(10240, 2048)], 28, 4, False, True, False),
    ([(20000, 2000)], 32, 16, False, True, False),
    ([(70000, 2048)], 28, 4, False, True, True),
    ([(9000, 900)] * 5, 32, 16, False, True, True),
    ([(20000, 1400), (500, 1), (9000, 1)], 64, 32, True, True, True),
])
def test_kernels_and_cuts(sequences, hq, hkv, small, large, cut):
    info, _ = _plan(sequences, hq, hkv)
    assert (info.n_small > 0, info.n_large > 0, info.slots > 0) == (small, large, cut)
    assert (info.n_joins > 0) == cut


@pytest.mark.parametrize("sequences, hq, hkv, wide", [
    ([(1337, 1)], 16, 8, 0), ([(16384, 1), (3000, 1)], 28, 4, 0), ([(300 + 500 * i, 32) for i in range(16)], 16, 8, 1)])
def test_units_of_32_and_of_64_query_vectors(sequences, hq, hkv, wide):
    info, words = _plan(sequences, hq, hkv)
    pieces = words[info.small:info.small + 16 * info.n_small].reshape(-1, 16)
    assert (pieces[:, 11] == wide).all()
