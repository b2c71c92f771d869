"""The selection's workspace, at the sizes where each part of its bound applies (no GPU)."""
from __future__ import annotations

import pytest

from diffusorrt_amd import _lib

pytest.importorskip("torch")


@pytest.mark.parametrize("rows,hkv,n_keys,block,want", [
    (32, 8, 32768, 32, 32 * 8 * 1024 * 8),           # all rows at once
    (1 << 20, 8, 1 << 20, 32, 1 << 28),              # as many as 256 MiB hold
    (17, 8, 1 << 23, 32, 1 << 28),                   # 16 rows fill them
    (17, 8, (1 << 23) + 32, 32, 16 * 8 * ((1 << 18) + 1) * 8),  # 16 rows are more
    (16, 8, 1 << 24, 32, 1 << 29),
    (4, 8, 1 << 24, 32, 1 << 27),                    # (no more rows than there are)
])
def test_select_workspace(rows, hkv, n_keys, block, want):
    if not _lib.LIB_PATH.exists():
        from diffusorrt_amd import build
        build.build()
    got = _lib.load().drt_op_select_blocks_workspace_bytes(rows, hkv, n_keys, block)
    assert got == want
    blocks = -(-n_keys // block)
    assert got <= max(1 << 28, 16 * hkv * blocks * 8)
    sums = hkv * -(-n_keys // 32) * 128 * 4
    assert got <= max(1 << 28, sums // 4)
