"""What a model's configuration means by its rope_scaling: numbers of published configurations, and the
forms that are refused."""
from __future__ import annotations

import math

import numpy as np
import pytest

from diffusorrt_amd.rotary import RotaryPositions, configured_frequencies, rotary_frequencies

# The frequencies that transformers 5.15.0 gives, in fp32, for dim 128, theta 10^6, {"rope_type": "yarn",
# "factor": 4.0, "original_max_position_embeddings": 32768} (a ramp over pairs 23 to 40), and for dim 64,
# theta 10^4, factor 40, original 4096 (10 to 23).
YARN_128 = [
    1.0, 0.805842221, 0.649381638, 0.523299158, 0.421696514, 0.339820832, 0.273841977, 0.220673397,
    0.177827939, 0.143301263, 0.115478203, 0.0930572003, 0.0749894157, 0.0604296438, 0.0486967526,
    0.0392418988, 0.0316227786, 0.0254829675, 0.0205352511, 0.0165481716, 0.0133352149, 0.0107460786,
    0.00865964312, 0.00697830599, 0.00537532149, 0.0041317381, 0.00316842273, 0.00242342241,
    0.00184827659, 0.00140511245, 0.00106436096, 0.000802959781, 0.000602941145, 0.000450323569,
    0.000334240554, 0.000246258394, 0.000179841154, 0.00012993149, 9.26230132e-05, 6.4903943e-05,
    4.44569851e-05, 3.58253164e-05, 2.88695483e-05, 2.32643015e-05, 1.87473561e-05, 1.51074091e-05,
    1.21741887e-05, 9.81047469e-06, 7.90569356e-06, 6.37074163e-06, 5.13381246e-06, 4.13704265e-06,
    3.33380353e-06, 2.68651957e-06, 2.16491094e-06, 1.74457659e-06, 1.40585337e-06, 1.13289593e-06,
    9.1293532e-07, 7.35681795e-07, 5.92843435e-07, 4.7773824e-07, 3.84981632e-07, 3.10234441e-07]
YARN_64 = [
    1.0, 0.749894202, 0.562341332, 0.421696514, 0.316227764, 0.237137362, 0.177827939, 0.133352146,
    0.100000001, 0.0749894157, 0.0562341288, 0.0390069261, 0.0268793609, 0.0183781441, 0.012447956,
    0.0083345091, 0.00550000044, 0.00356199732, 0.00224936521, 0.00137051346, 0.000790569407,
    0.000414990413, 0.00017782794, 3.3338034e-05, 2.49999994e-05, 1.87473543e-05, 1.40585325e-05,
    1.05424124e-05, 7.90569447e-06, 5.92843435e-06, 4.44569832e-06, 3.33380353e-06]
# A power (2^-23), its inverse, a quotient, the ramp (a difference, a quotient, 1 less it), two products
# and their sum in fp32 (2^-24 each), and nine digits here (2^-30).
FP32 = 2.0**-21


@pytest.mark.parametrize("dim, theta, factor, original, want, magnitude", [
    (128, 1e6, 4.0, 32768, YARN_128, 1.138629436111989),
    (64, 1e4, 40.0, 4096, YARN_64, 1.3688879454113936)])
def test_yarn_of_published_configurations(dim, theta, factor, original, want, magnitude):
    scaling = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": original}
    r = RotaryPositions(dim, theta=theta, scaling=scaling, device="cpu")
    assert r.magnitude == pytest.approx(magnitude, rel=1e-15)
    assert r.frequencies == pytest.approx(want, rel=FP32, abs=0)
    f, m = configured_frequencies(dim, theta, scaling)
    assert (f, m) == (r.frequencies, r.magnitude)
    # (older configurations say "type")
    old = {"type" if k == "rope_type" else k: v for k, v in scaling.items()}
    assert RotaryPositions(dim, theta=theta, scaling=old, device="cpu").frequencies == f


def test_yarns_ramp_is_linear_in_the_pair():
    scaling = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096,
               "beta_fast": 16, "beta_slow": 2.0, "attention_factor": 1.5}
    plain, _ = rotary_frequencies(64, 1e4)
    f, m = configured_frequencies(64, 1e4, scaling)
    low, high = (64 * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(1e4)) for turns in (16, 2))
    low, high = math.floor(low), math.ceil(high)
    assert (low, high, m) == (12, 21, 1.5)
    for i, (a, b) in enumerate(zip(plain, f)):
        scaled = min(1.0, max(0.0, (i - low) / (high - low)))
        assert b == pytest.approx(a * (1 - scaled) + a / 8 * scaled, rel=1e-14)
    assert f[:low + 1] == plain[:low + 1]
    # the paper's, in proportion to the turns, is another: by half of a frequency and more here
    other, _ = rotary_frequencies(64, 1e4, scaling)
    assert max(abs(a / b - 1) for a, b in zip(f, other)) > 0.4


def test_a_ramp_at_one_pair():
    # beta_slow's pair is 8 ln(6 / 2 pi) / (2 ln 10^4) = -0.02, rounded up 0, and beta_fast's held at 0
    plain, _ = rotary_frequencies(8, 1e4)
    f, _ = configured_frequencies(8, 1e4, {"type": "yarn", "factor": 2.0,
                                           "original_max_position_embeddings": 6})
    assert f[0] == plain[0] and f[1:] == [x / 2 for x in plain[1:]]


def test_other_forms_are_the_same_by_both_names():
    for scaling in (None, {"rope_type": "linear", "factor": 3.0}, {"type": "ntk", "factor": 2.5}):
        assert configured_frequencies(96, 5e5, scaling) == rotary_frequencies(96, 5e5, scaling)
        r = RotaryPositions(96, theta=5e5, scaling=scaling, device="cpu")
        assert r.frequencies == rotary_frequencies(96, 5e5, scaling)[0]


@pytest.mark.parametrize("dim, theta, original", [
    (128, 1e6, 4),         # no pair makes one turn
    (128, 1e6, 2.0**60),   # every pair makes more than 32
    (128, 1.0, 4096),      # all pairs make the same number
    (128, 0.5, 4096)])
def test_a_yarn_without_a_ramp_is_refused(dim, theta, original):
    scaling = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": original}
    with pytest.raises(ValueError, match="yarn"):
        configured_frequencies(dim, theta, scaling)
    with pytest.raises(ValueError, match="yarn"):
        RotaryPositions(dim, theta=theta, scaling=scaling, device="cpu")


@pytest.mark.parametrize("frequencies", [configured_frequencies, rotary_frequencies])
@pytest.mark.parametrize("factor", [1.0, 0.5, 1e-5])
def test_yarn_of_no_extension_has_magnitude_one(frequencies, factor):
    scaling = {"type": "yarn", "factor": factor, "original_max_position_embeddings": 4096}
    assert frequencies(128, 1e6, scaling)[1] == 1.0
    assert frequencies(128, 1e6, scaling | {"attention_factor": 0.25})[1] == 0.25
    assert frequencies(128, 1e6, scaling | {"factor": 1 + 2.0**-20})[1] > 1.0


@pytest.mark.parametrize("call", [
    dict(theta=5e-324),                                      # theta^-126/128 is beyond a double
    dict(scaling={"type": "linear", "factor": 1e-320}),      # so is the first pair's 1 / factor
    dict(scaling={"type": "ntk", "factor": 1e308}),          # and the base
    dict(scaling={"type": "ntk", "factor": 5e-324}),         # a base of 0
    dict(scaling={"type": "yarn", "factor": 1e-320, "original_max_position_embeddings": 4096}),
    dict(frequencies=[1.0] * 64, magnitude=1e39),            # infinity in fp32
    dict(scaling={"type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096,
                  "attention_factor": 1e39}),
])
def test_frequencies_and_magnitudes_beyond_their_types_are_refused(call):
    with pytest.raises(ValueError):
        RotaryPositions(**({"device": "cpu"} | call))


def test_numpy_numbers_are_numbers():
    scaling = {"type": "yarn", "factor": np.float32(4), "original_max_position_embeddings": np.int64(4096)}
    r = RotaryPositions(np.int64(64), theta=np.float64(1e4), scaling=scaling, device="cpu")
    assert type(r.dim) is int and r.dim == 64
    assert r.frequencies == configured_frequencies(
        64, 1e4, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})[0]
    own = RotaryPositions(np.int32(4), frequencies=np.array([1.0, 0.5], np.float32), device="cpu")
    assert own.frequencies == [1.0, 0.5]
    for dim in (np.float64(64), np.True_, "64"):
        with pytest.raises(ValueError):
            RotaryPositions(dim, device="cpu")
