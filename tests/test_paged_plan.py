"""The paged cache's plan on the CPU: every (row, head, key) that a batch attends to is in one part and
every row in one tile, the places that the lists name lie inside the cache, and what is refused."""
from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from diffusorrt_amd import _lib
from diffusorrt_amd.paged import PagedKVCache
from oracle import paged as P

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")


LARGE = set()  # (many rows, the large kernel is used, parts are joined) of the plans that were looked at


def _cache(pages=64, page_size=64, kv_heads=2):
    return PagedKVCache(1, kv_heads, pages, page_size=page_size, device="cpu")


def _words(batch, at, n, width):
    return batch._list.numpy()[at:at + n * width].reshape(n, width)


def _pieces(batch, large):
    """The parts of a kernel's work-groups: one each, or (large) from its first to the one that says it
    is the last."""
    info, words = batch.info, batch._list.numpy()
    if not large:
        return list(_words(batch, info.small, info.n_small, 16))
    out = []
    for i in words[info.first_large:info.first_large + info.n_large]:
        assert i == len(out)
        while True:
            at = info.large + 16 * len(out)
            out.append(words[at:at + 16])
            if out[-1][10]:
                break
    return out


def _random_batch(seed, many=False):
    rng = random.Random(seed)
    size, kv_heads = rng.choice([32, 64, 256]), rng.choice([16, 32] if many else [1, 2, 4])
    g = rng.choice([1, 2, 7, 40])
    seqs = rng.choice([1, 3, 17])
    kind = rng.choice(["full", "causal", "d2f_hybrid"])
    rows, keys, pos0, prompt = [], [], [], []
    for s in range(seqs):
        n = rng.choice([0, 1, 9, 32, 200])
        k = rng.choice([0, 1, 31, 32, 33, rng.randint(1, 3000)])
        if many and s % 2 == 0:  # enough of them for the large kernel
            n, k = rng.randint(2000, 5000) // g * g // 2 + 300, rng.choice([0, 40, 20000, 70000])
        rows.append(n)
        keys.append(k)
        pos0.append(max(0, k - n) if rng.random() < 0.7 else rng.randint(0, 4000))
        prompt.append(rng.randint(0, 100))
    if not sum(rows):
        rows[0] = 5
    need = [-(-k // size) for k in keys]
    pages = sum(need) + 5
    order = rng.sample(range(pages), pages)
    table = [[order.pop() for _ in range(n)] for n in need]
    block = rng.choice([1, 8, 32, 100])
    cache = _cache(pages, size, kv_heads)
    geometry = (prompt, block) if kind == "d2f_hybrid" else None
    batch = cache.batch(table, keys, rows, heads=kv_heads * g, positions=pos0, kind=kind,
                        mask_geometry=geometry)
    return cache, batch, table, rows, keys, pos0, kind, prompt, block, g


@pytest.mark.parametrize("seed, many", [(i, False) for i in range(40)] +
                         [(i, True) for i in range(100, 130)])
def test_parts_cover_every_row_and_key_once(seed, many):
    cache, batch, table, rows, keys, pos0, kind, prompt, block, g = _random_batch(seed, many)
    info, tpp = batch.info, cache.page_size // 32
    row0 = np.concatenate([[0], np.cumsum(rows)])
    assert batch.rows == sum(rows) == info.rows
    pages = batch._list.numpy()[info.table:info.words]
    joins = _words(batch, info.joins, info.n_joins, 8)
    seen = {}   # (sequence, query vector / 32) -> tile ranges
    slots = set()
    for large in (0, 1):
        for p in _pieces(batch, large):
            r0, nr, p0, nk, pl, vec0, t0, t1, slot, tab = (int(x) for x in p[:10])
            s = [i for i in range(len(rows)) if row0[i] == r0 and rows[i] == nr and rows[i]][0]
            assert (p0, nk) == (pos0[s], keys[s])
            assert pl == (prompt[s] if kind == "d2f_hybrid" else 0)
            need = -(-keys[s] // cache.page_size)
            assert [int(x) for x in pages[tab:tab + need]] == [
                x * cache.kv_heads * tpp for x in table[s][:need]]
            assert 0 <= t0 <= t1 <= -(-keys[s] // 32) and 0 <= vec0 < nr * g
            vecs = nr * g - vec0
            vecs = min(256 if large else 32 << p[11], vecs)
            for sub in range(-(-vecs // 32)):
                seen.setdefault((s, vec0 // 32 + sub), []).append((t0, t1, slot + sub if slot >= 0
                                                                    else -1))
                if slot >= 0:
                    assert slot + sub < info.slots and slot + sub not in slots
                    slots.add(slot + sub)
    assert len(slots) == info.slots
    LARGE.add((many, info.n_large > 0, info.n_large > 0 and info.slots > 0))
    joined = {}
    for r0, vec0, vecs, slot, step, parts, *_ in joins:
        joined[(int(r0), int(vec0))] = (int(vecs), [int(slot) + i * int(step) for i in range(parts)])
    for s, n in enumerate(rows):
        ends = P.key_ends(kind, pos0[s], n, keys[s], prompt[s], block)
        for u in range(-(-n * g // 32)):
            parts = sorted(seen.pop((s, u)))
            last = ends[min(n * g - 1, 32 * u + 31) // g]
            at = 0
            for t0, t1, _ in parts:
                assert t0 == at
                at = t1
            assert at * 32 >= last
            if len(parts) == 1:
                assert parts[0][2] == -1
            else:
                vecs, where = joined.pop((int(row0[s]), 32 * u))
                assert vecs == min(32, n * g - 32 * u)
                assert sorted(x[2] for x in parts) == sorted(where)
    assert not seen and not joined


def test_both_kernels_and_both_cuts_were_planned():
    if len(LARGE) > 1:  # (run with the tests above)
        assert {(False, False, False), (True, True, False), (True, True, True)} <= LARGE


@pytest.mark.parametrize("seed", range(40, 70))
def test_tiles_hold_every_row_once(seed):
    cache, batch, table, rows, keys, pos0, *_ = _random_batch(seed)
    tpp, row, want = cache.page_size // 32, 0, {}
    inside = True
    for s, n in enumerate(rows):
        for i in range(n):
            p = pos0[s] + i
            if p < keys[s]:
                tile = table[s][p // cache.page_size] * cache.kv_heads * tpp + p % cache.page_size // 32
                want[row + i] = (tile, p % 32, p)
            else:
                inside = False
        row += n
    got = {}
    for tile, lo, hi, r, pos, *_ in _words(batch, batch.info.tiles, batch.info.n_tiles, 8):
        assert 0 <= lo < hi <= 32 and 0 <= tile < cache.pages * cache.kv_heads * tpp
        assert (tile // tpp) % cache.kv_heads == 0
        for i in range(hi - lo):
            assert r + i not in got
            got[int(r + i)] = (int(tile), int(lo + i), int(pos + i))
    assert got == want
    assert bool(batch.info.appendable) == inside


def test_rows_of_two_sequences_in_one_tile_are_not_appendable():
    cache = _cache()
    assert cache.batch([[3], [4]], [5, 5], [1, 1], heads=4).info.appendable
    assert not cache.batch([[3], [3]], [5, 7], [1, 1], heads=4).info.appendable
    # a prefix in common is only read
    assert cache.batch([[3, 1], [3, 2]], [70, 70], [1, 1], heads=4).info.appendable


@pytest.mark.parametrize("call, what", [
    (dict(pages=[[64]], keys=[3], rows=[1]), "outside the cache"),
    (dict(pages=[[-1]], keys=[3], rows=[1]), "outside the cache"),
    (dict(pages=[[1, 2]], keys=[129], rows=[1]), "more pages"),
    (dict(pages=[[1], [2, 64]], keys=[3, 65], rows=[1, 1]), "sequence 1"),
    (dict(pages=[[1]], keys=[3], rows=[4]), "from zero on"),
    (dict(pages=[[1]], keys=[3], rows=[0]), "a row at least"),
    (dict(pages=[[1]], keys=[-1], rows=[1]), "from zero on"),
    (dict(pages=[[1]], keys=[3, 4], rows=[1]), "each sequence"),
    (dict(pages=[], keys=[], rows=[]), "a sequence at least"),
    (dict(pages=[[1.5]], keys=[3], rows=[1]), "whole numbers"),
    (dict(pages=[[1]], keys=[2**40], rows=[1]), "32 bits"),
    (dict(pages=[[1]], keys=[3], rows=[1], positions=[2**31 - 1]), "32 bits"),
    (dict(pages=[[1]], keys=[3], rows=[1], heads=3), "multiple"),
    (dict(pages=[[1]], keys=[3], rows=[1], heads=0), "multiple"),
    (dict(pages=[[1]], keys=[3], rows=[1], heads=16386), "16384"),
    (dict(pages=[[1]], keys=[3], rows=[1], heads=4.0), "whole number"),
    (dict(pages=torch.ones(1, 1, dtype=torch.bfloat16), keys=[3], rows=[1]), "whole numbers"),
    (dict(pages=[[1]], keys=torch.ones(1), rows=[1]), "whole numbers"),
    (dict(pages=[1], keys=[3], rows=[1]), "list of page numbers"),
    (dict(pages=np.ones(3, dtype=np.int32), keys=[3], rows=[1]), "sequences, width"),
    (dict(pages=[[1]], keys=[3], rows=[1], heads=2**40), "whole number"),
    (dict(pages=[[1]], keys=[3], rows=[1], kind="d2f_hybrid", mask_geometry=(0,)), "geometry"),
    (dict(pages=[[1]], keys=[3], rows=[1], kind="d2f_hybrid", mask_geometry=(0, 2**40)), "geometry"),
    (dict(pages=[[1]], keys=[3], rows=[1], kind="window"), "mask kind"),
    (dict(pages=[[1]], keys=[3], rows=[1], mask_geometry=(0, 32)), "geometry"),
    (dict(pages=[[1]], keys=[3], rows=[1], kind="d2f_hybrid"), "geometry"),
    (dict(pages=[[1]], keys=[3], rows=[1], kind="d2f_hybrid", mask_geometry=(0, 0)), "geometry"),
    (dict(pages=[[1]], keys=[3], rows=[1], kind="d2f_hybrid", mask_geometry=([1, 2], 8)),
     "each sequence"),
    (dict(pages=[[1]], keys=[3], rows=[1], kind="d2f_hybrid", mask_geometry=([-1], 8)), "geometry"),
    (dict(pages=[[1]], keys=[2**31 - 1], rows=[1]), "too many keys"),
])
def test_bad_batches_are_refused(call, what):
    with pytest.raises(ValueError, match=what):
        _cache().batch(**({"heads": 4} | call))


def test_a_page_is_not_read_behind_a_sequences_keys():
    # (the list may be longer than the keys need, whatever stands there)
    batch = _cache().batch(np.array([[3, -1, 99]], dtype=np.int64), [64], [1], heads=4)
    assert batch.info.words == batch.info.table + 1


def test_caches_that_are_refused():
    for bad in (dict(page_size=48), dict(page_size=16), dict(pages=0), dict(kv_heads=0),
                dict(dtype="i8"), dict(dtype="fp8"), dict(pages=2**31)):
        args = dict(layers=1, kv_heads=2, pages=4, device="cpu") | bad
        with pytest.raises(ValueError):
            PagedKVCache(**args)
    cache = _cache()
    batch = cache.batch([[3]], [5], [1], heads=4)
    with pytest.raises(ValueError, match="GPU"):
        cache.attention(0, None, batch)
    with pytest.raises(ValueError, match="layer"):
        cache.load(1, batch)


def test_more_work_groups_than_a_launch_has_are_refused():
    # 2^32 threads and more: 512 for each sequence's token and K/V head
    n = 2**20
    ones, pages = np.ones(n, dtype=np.int32), np.zeros((n, 1), dtype=np.int32)
    with pytest.raises(ValueError, match="too many rows"):
        _cache(kv_heads=8).batch(pages, ones, ones, heads=8)
    assert _cache(kv_heads=4).batch(pages, ones, ones, heads=4).rows == n
