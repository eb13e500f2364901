"""Every key of a model's rope scaling is served, known not to matter, or
refused.  The expected values are the definitions' own, pair by pair."""
import math

import pytest
import torch

import epure

YARN = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096}


def yarn(dim, theta, sc, truncate):
    """Frequencies of yarn: pair i turns old * f / 2 pi times within the old
    context; between the (fractional) indices of the pairs that make 32 turns
    and 1 turn the division by the factor sets in linearly.  The indices are
    widened to whole ones unless ``truncate`` is off."""
    old, out = sc["original_max_position_embeddings"], []
    at = [dim / 2 * math.log(old / (2 * math.pi * turns), theta)
          for turns in (sc.get("beta_fast", 32.0), sc.get("beta_slow", 1.0))]
    lo, hi = (math.floor(at[0]), math.ceil(at[1])) if truncate else at
    lo, hi = max(lo, 0), min(hi, dim - 1)
    for i in range(dim // 2):
        f = theta ** (-2 * i / dim)
        t = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        out.append(f * (1 - t) + f / sc["factor"] * t)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("dim,theta", [(64, 150000.0), (128, 1e4), (32, 5e5)])
@pytest.mark.parametrize("truncate", [None, True, False])
def test_yarn_with_and_without_truncation(dim, theta, truncate):
    sc = YARN if truncate is None else {**YARN, "truncate": truncate}
    f, m = epure.rope_frequencies(dim, theta, sc)
    assert torch.allclose(f, yarn(dim, theta, sc, truncate is not False), rtol=1e-12, atol=0.0)
    assert math.isclose(m, 0.1 * math.log(32) + 1)
    other, _ = epure.rope_frequencies(dim, theta, {**YARN, "truncate": truncate is False})
    assert not torch.allclose(f, other, rtol=1e-3, atol=0.0)


@pytest.mark.parametrize("keys,want", [
    ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0),
    ({"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
    ({"mscale": 1.0, "mscale_all_dim": 0.5}, (0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1)),
    ({"mscale": 0.707}, 0.1 * math.log(40) + 1),                # both or none
    ({"mscale": 0.707, "mscale_all_dim": 0}, 0.1 * math.log(40) + 1),
    ({"mscale": 1.0, "mscale_all_dim": 1.0, "attention_factor": 1.25}, 1.25),
    ({"attention_factor": None}, 0.1 * math.log(40) + 1),
    ({"factor": 0.5, "mscale": 1.0, "mscale_all_dim": 0.5}, 1.0)])
def test_yarn_attention_factors(keys, want):
    _, m = epure.rope_frequencies(64, 1e4, {**YARN, "factor": 40.0, **keys})
    assert math.isclose(m, want, rel_tol=1e-12)


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
LINEAR = {"type": "linear", "factor": 2.0}


@pytest.mark.parametrize("base", [YARN, LLAMA3, LINEAR, {"rope_type": "default"}])
@pytest.mark.parametrize("key,value", [("short_factor", [1.0]), ("mrope_section", [16, 24, 24]), ("alpha", 2.0),
                                       ("extrapolation_factor", 1.0)])
def test_keys_that_are_not_served_raise(base, key, value):
    with pytest.raises(ValueError, match=key):
        epure.rope_frequencies(64, 1e4, {**base, key: value})
    epure.rope_frequencies(64, 1e4, {**base, key: None})
    with pytest.raises(ValueError, match=key):
        epure.Rotary(64, 4, scaling={**base, key: value}, device="cpu")


def test_keys_that_a_scaling_does_not_use_are_none_of_its_business():
    for base in (LINEAR, {"rope_type": "default"}):
        a, b = (epure.rope_frequencies(64, 1e4, {**base, **more}) for more in
                ({}, {"original_max_position_embeddings": 4096, "partial_rotary_factor": 0.5, "mscale": 1.0}))
        assert torch.equal(a[0], b[0]) and a[1] == b[1] == 1.0


@pytest.mark.parametrize("base", [YARN, LLAMA3, LINEAR, {"rope_type": "default"}])
def test_theta_in_the_scaling(base):
    """Newer configurations keep rope_theta beside the scaling: taken if no
    other is given, refused if another is."""
    want = epure.rope_frequencies(64, 5e5, base)
    for got in (epure.rope_frequencies(64, scaling={**base, "rope_theta": 5e5}),
                epure.rope_frequencies(64, 5e5, {**base, "rope_theta": 500000})):
        assert torch.equal(got[0], want[0]) and got[1] == want[1]
    with pytest.raises(ValueError, match="theta"):
        epure.rope_frequencies(64, 1e4, {**base, "rope_theta": 5e5})
    assert torch.equal(epure.rope_frequencies(64)[0], epure.rope_frequencies(64, 1e4)[0])
    r = epure.Rotary(64, 20, scaling={**base, "rope_theta": 5e5}, device="cpu")
    assert torch.equal(r.cos, epure.Rotary(64, 20, 5e5, scaling=base, device="cpu").cos)
