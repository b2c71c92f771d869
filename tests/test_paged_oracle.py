"""The paged operators' oracle on the CPU: against closed forms and a second way of writing them, and its
attention bound against mistakes planted in it."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import ops as O
from oracle import paged as P


def test_rotation_is_the_references_and_keeps_lengths():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((9, 3, 128))
    pos = np.arange(9) * 37
    f = 1e6 ** (-np.arange(64) / 64)
    y = P.rotate(x, pos, f)
    cos, sin = O.rope_tables(pos, 128, 1e6)
    assert np.allclose(y, O.apply_split_half_rope(x.astype(np.float32), cos, sin), atol=2e-4)
    assert np.allclose((y**2).sum(-1), (x**2).sum(-1))
    # the interleaved layout is the half one of reordered elements
    order = np.concatenate([np.arange(0, 128, 2), np.arange(1, 128, 2)])
    z = P.rotate(x[..., np.argsort(order)], pos, f, layout="interleaved")
    assert np.allclose(z[..., order], y)
    assert np.allclose(P.rotate(y, pos, f, inverse=True), x)
    # products of two turned vectors go by the difference of their positions
    a, b = P.rotate(x, pos, f), P.rotate(x, pos + 5, f)
    c, d = P.rotate(x, pos + 100, f), P.rotate(x, pos + 105, f)
    assert np.allclose((a * b).sum(-1), (c * d).sum(-1))


def test_key_ends():
    assert P.key_ends("full", 3, 2, 9) == [9, 9]
    assert P.key_ends("causal", 3, 3, 5) == [4, 5, 5]
    assert P.key_ends("d2f_hybrid", 2, 5, 20, 4, 8) == [4, 4, 12, 12, 12]
    assert P.key_ends("d2f_hybrid", 0, 2, 3, 4, 8) == [3, 3]
    assert P.key_ends("causal", 0, 2, 0) == [0, 0]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_by_hand_and_planted_mistakes(kind):
    rng = np.random.default_rng(1)
    n, rows = 300, 4
    q, k, v = (rng.standard_normal(s) for s in ((rows, 4, 128), (n, 2, 128), (n, 2, 128)))
    ends = P.key_ends("causal", n - rows, rows, n)
    o, bound = P.attention(q, k, v, ends, kind)
    s = np.einsum("rhd,khd->rhk", q, k.repeat(2, 1)) / np.sqrt(128)
    for r in range(rows):
        s[r, :, ends[r]:] = -np.inf
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    assert np.allclose(o, np.einsum("rhk,khd->rhd", w, v.repeat(2, 1)))
    assert (bound > 0).all() and (bound < 0.02).all()
    # a tile left out, one key too many, the other head's keys, scores off by a twentieth
    wrong = [P.attention(q, np.delete(k, np.s_[64:96], 0), np.delete(v, np.s_[64:96], 0),
                         [e - 32 for e in ends], kind)[0],
             P.attention(q, k, v, [min(n, e + 1) for e in ends], kind)[0][:3],
             P.attention(q, k[:, ::-1], v, ends, kind)[0],
             P.attention(q * 1.05, k, v, ends, kind)[0]]
    for x in wrong:
        assert (np.abs(x - o[:len(x)]) > bound[:len(x)]).any()
    zero, none = P.attention(q, k, v, [0, 1, 0, 2], kind)
    assert (zero[0] == 0).all() and (none[2] == 0).all() and np.allclose(zero[1], v[0].repeat(2, 0))
