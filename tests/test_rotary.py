"""Rotary frequencies and their 64-bit turns on the CPU, and the calls that are refused."""
from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

from diffusorrt_amd.package import rope_linear_factor
from diffusorrt_amd.rotary import _TWO_PI, RotaryPositions, rotary_frequencies


def test_plain_linear_and_ntk():
    f, m = rotary_frequencies(128, 1e6)
    assert m == 1.0 and len(f) == 64 and f[0] == 1.0 and f[63] == pytest.approx(1e6 ** (-126 / 128))
    scaling = {"rope_type": "linear", "factor": 4.0}
    g, m = rotary_frequencies(128, 1e6, scaling)
    assert m == 1.0 and g == [x / rope_linear_factor(scaling) for x in f]
    g, m = rotary_frequencies(128, 1e6, {"type": "ntk", "factor": 8})
    assert m == 1.0 and g[0] == 1.0 and g[63] == pytest.approx(f[63] / 8, rel=1e-14)
    assert all(a / 8 * (1 - 1e-14) <= b <= a for a, b in zip(f, g))


def test_yarn_by_parts():
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    f, _ = rotary_frequencies(128, 1e6)
    g, m = rotary_frequencies(128, 1e6, scaling)
    assert m == pytest.approx(0.1 * math.log(4) + 1)
    for a, b in zip(f, g):
        turns = 32768 * a / (2 * math.pi)
        if turns >= 32:
            assert b == a
        elif turns <= 1:
            assert b == pytest.approx(a / 4, rel=1e-15)
        else:
            keep = (turns - 1) / 31
            assert b == pytest.approx(a * keep + a / 4 * (1 - keep), rel=1e-14)
    assert any(32768 * a / (2 * math.pi) < 1 for a in f) and g == sorted(g, reverse=True)
    _, m = rotary_frequencies(64, 1e4, scaling | {"attention_factor": 1.5, "beta_fast": 16})
    assert m == 1.5


def test_turns_are_the_frequencies_to_64_bits():
    r = RotaryPositions(64, theta=1e4, device="cpu")
    for f, t in zip(r.frequencies, r.turns.tolist()):
        assert abs(Fraction(t, 2**64) - Fraction(f) / _TWO_PI) <= Fraction(1, 2**65)
    assert abs(float(_TWO_PI) - 2 * math.pi) < 1e-15
    # whole turns fall off, backwards ones too
    r = RotaryPositions(8, frequencies=[2 * math.pi * 3, -0.5, 100.0, 0.0], device="cpu")
    t = [x / 2**64 for x in r.turns.tolist()]
    assert abs(t[0]) < 1e-15 and t[1] == pytest.approx(-0.5 / (2 * math.pi))
    assert (t[2] - 100 / (2 * math.pi)) % 1 == pytest.approx(1, abs=1e-12) or \
        (t[2] - 100 / (2 * math.pi)) % 1 < 1e-12
    assert t[3] == 0


@pytest.mark.parametrize("call", [
    dict(dim=0), dict(dim=7), dict(dim=True), dict(dim=2.0), dict(theta=0), dict(theta=math.inf),
    dict(layout="pairs"), dict(scaling="linear"), dict(scaling={"factor": 2.0}),
    dict(scaling={"type": "dynamic", "factor": 2.0}), dict(scaling={"type": "linear"}),
    dict(scaling={"type": "linear", "factor": -1.0}), dict(scaling={"type": "ntk", "factor": "4"}),
    dict(scaling={"type": "linear", "factor": 2.0, "beta_fast": 3}),
    dict(scaling={"type": "yarn", "factor": 2.0}),
    dict(scaling={"type": "yarn", "factor": 2.0, "original_max_position_embeddings": 10,
                  "beta_fast": 1}),
    dict(dim=2, scaling={"type": "ntk", "factor": 2.0}),
    dict(frequencies=[1.0]), dict(frequencies=[math.nan] * 64), dict(magnitude=2.0),
    dict(frequencies=[1.0] * 64, scaling={"type": "linear", "factor": 2.0}),
    dict(frequencies=[1.0] * 64, magnitude=math.inf),
])
def test_bad_rotaries_are_refused(call):
    with pytest.raises(ValueError):
        RotaryPositions(**({"device": "cpu"} | call))


def test_no_rotation_on_the_cpu():
    with pytest.raises(ValueError, match="GPU"):
        RotaryPositions(8, device="cpu").rotate(torch.zeros(1, 1, 8), 0)
