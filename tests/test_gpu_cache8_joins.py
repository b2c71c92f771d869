"""Attention over listed blocks in several key ranges, whose parts a second launch joins: values
that are not finite come out as they do of one range. Each test prints its case first."""
from __future__ import annotations

import numpy as np
import pytest

from diffusorrt_amd import _lib
from oracle import cache8 as X

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of the product's type


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,count,at", [
    (9, 16, 15), (9, 16, 0), (9, 16, 7),  # eight ranges: infinities in the last, the first, between
    (2, 17, 16), (1, 17, 16),             # nine
    (9, 13, 12),                          # seven
    (5, 40, 39),                          # twenty
])
def test_infinities_of_a_key_range_survive_the_join(dtype, rows, count, at):
    from diffusorrt_amd.kernels import PrefixKVCache

    hq, hkv, block = 28, 4, 64
    n = block * count
    bytes_ = _lib.load().drt_op_sparse_attention_workspace_bytes(rows, hq, hkv, block, count)
    ranges = bytes_ // (rows * hq * 130 * 4)
    print("[case] join", dtype, rows, count, at, "ranges", ranges, flush=True)
    assert ranges > 1 and ranges % 16  # (a range behind the last in a batch of the join)
    rng = np.random.default_rng(rows * count + at)
    k, v = (torch.from_numpy(rng.standard_normal((n, hkv, 128), np.float32)) for _ in range(2))
    clean = v.clone()
    key = block * at + 50
    v[key, :, 3], v[key, :, 4], v[key, :, 5] = float("inf"), -float("inf"), float("nan")
    v[key + 1, :, 6] = 3e38  # beyond fp16: stored as infinity there, a large value in bf16
    cache = PrefixKVCache(1, hkv, n, dtype=dtype)
    cache.store(0, k.cuda(), v.cuda(), 0)
    lists = np.tile(np.arange(count, dtype=np.int32), (rows, hkv, 1))
    lists[3::4, :, at] = -1  # rows that do not list the block
    q = torch.from_numpy(rng.standard_normal((rows, hq, 128), np.float32)).to(TDT[dtype])
    got = cache.sparse_attention(0, q.cuda(), torch.from_numpy(lists).cuda(), block_size=block,
                                 n_keys=n, row_pos0=0, kind="full")
    got = got.double().cpu().numpy().reshape(rows, hq, 128)
    kc, vc = (x.to(TDT[dtype]).double().numpy() for x in (k, clean))
    ends, qd = X.key_ends(rows, n, 0), q.double().numpy()
    out, weight = X.attention(qd, kc, vc, ends, lists, block)
    bound = X.attention_bound(qd, kc, vc, ends, weight, HALF[dtype], n)
    for r in range(rows):
        ok = np.ones(128, bool)
        if r % 4 != 3:
            assert (got[r, :, 3] == np.inf).all() and (got[r, :, 4] == -np.inf).all(), r
            assert np.isnan(got[r, :, 5]).all(), r
            if dtype == "f16":
                assert (got[r, :, 6] == np.inf).all(), r
            ok[3:7] = False
        assert (np.abs(got[r] - out[r]) <= bound[r] * 1.001)[:, ok].all(), r
