"""Frequencies of stretched contexts, with the names that checkpoints' configurations use, against values worked out by hand."""

import math

import pytest
import torch

from miles_amd.kernels.rotary import rotary_frequencies

DEEPSEEK = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1, "mscale": 1.0, "mscale_all_dim": 1.0}
OPEN = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096, "beta_fast": 32.0, "beta_slow": 1.0, "truncate": False}


def _yarn(dim, base, scaling):
    return rotary_frequencies(dim, base, scaling=scaling, device="cpu")


def test_the_ramp_between_fast_and_slow_pairs():
    """64 elements, base 10^4, 4096 positions: 64 ln(4096 / (32 2 pi)) / (2 ln 10^4) = 10.47 and 64 ln(4096 / (2 pi)) / (2 ln 10^4) = 22.51, so that the ramp goes
    from pair 10 to pair 23.  Pair 16 turns 0.01 a position: 0.01 (7 / 13 + 6 / 13 / 40) = 0.0055."""
    f, _ = _yarn(64, 1e4, DEEPSEEK)
    plain = rotary_frequencies(64, 1e4, device="cpu")[0]
    assert abs(f[16].item() - 0.0055) < 1e-16
    assert torch.equal(f[:11], plain[:11]) and torch.allclose(f[23:], plain[23:] / 40, rtol=1e-15, atol=0)
    for pair in range(10, 24):
        slowed = (pair - 10) / 13
        want = 10.0 ** (-pair / 8) * (1 - slowed + slowed / 40)
        assert abs(f[pair].item() - want) < 4e-16 * want, pair


def test_a_ramp_that_is_not_truncated():
    """Where the ends of the ramp are not rounded to whole pairs it is linear in the logarithm of how often a pair turns in the original context:
    all of a pair's speed is kept at 32 turns, none at one."""
    f, scale = _yarn(64, 150000.0, OPEN)
    for pair in range(32):
        speed = 150000.0 ** (-pair / 32)
        kept = min(1.0, max(0.0, math.log(4096 * speed / (2 * math.pi)) / math.log(32)))
        want = speed * (kept + (1 - kept) / 32)
        assert abs(f[pair].item() - want) < 1e-13 * want, pair
    assert abs(scale - (0.1 * math.log(32) + 1)) < 1e-15
    rounded, _ = _yarn(64, 150000.0, {**OPEN, "truncate": True})
    assert (rounded / f - 1).abs().max() > 0.3
    assert torch.equal(rounded, _yarn(64, 150000.0, {k: v for k, v in OPEN.items() if k != "truncate"})[0])


def test_what_cosines_and_sines_are_multiplied_with():
    """0.1 m ln 40 + 1 is 1.3688879454113936 for m = 1 and 1.2608037774058553 for m = 0.707."""
    assert _yarn(64, 1e4, DEEPSEEK)[1] == 1.0
    assert abs(_yarn(64, 1e4, {**DEEPSEEK, "mscale": 0.707})[1] - 1.2608037774058553 / 1.3688879454113936) < 1e-15
    assert abs(_yarn(64, 1e4, {**DEEPSEEK, "mscale_all_dim": 0.707})[1] - 1.3688879454113936 / 1.2608037774058553) < 1e-15
    for none in ({"mscale": None, "mscale_all_dim": None}, {"mscale": 1.0, "mscale_all_dim": 0}, {"mscale": 1.0, "mscale_all_dim": None}):
        assert abs(_yarn(64, 1e4, {**DEEPSEEK, **none})[1] - 1.3688879454113936) < 1e-15
    assert _yarn(64, 1e4, {**DEEPSEEK, "mscale": 0.707, "attention_factor": 1.25})[1] == 1.25
    assert _yarn(64, 1e4, {**DEEPSEEK, "mscale": 0.707, "factor": 1.0})[1] == 1.0
    # one of the two alone is read differently by different programs
    for alone in ({"mscale": 0.707, "mscale_all_dim": None}, {"mscale": None, "mscale_all_dim": 1.0}, {"mscale": 0.5, "mscale_all_dim": 0.0}):
        with pytest.raises(ValueError, match="mscale"):
            _yarn(64, 1e4, {**DEEPSEEK, **alone})


def test_names_that_are_not_known_are_refused():
    for scaling in (DEEPSEEK, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "default"}, {}):
        with pytest.raises(ValueError, match="low_freq_factor"):
            _yarn(64, 1e4, {**scaling, "low_freq_factor": 1.0})
    with pytest.raises(ValueError, match="mscale"):
        _yarn(64, 1e4, {"rope_type": "linear", "factor": 4.0, "mscale": 1.0})
    with pytest.raises(ValueError, match="truncate"):
        _yarn(64, 1e4, {**OPEN, "truncate": "no"})
    # what repeats the arguments has to agree with them
    assert torch.equal(_yarn(64, 1e4, {**DEEPSEEK, "rope_theta": 10000})[0], _yarn(64, 1e4, DEEPSEEK)[0])
    with pytest.raises(ValueError, match="rope_theta"):
        _yarn(64, 1e4, {**DEEPSEEK, "rope_theta": 5e5})
    assert torch.equal(_yarn(64, 1e4, {"rope_type": "default", "partial_rotary_factor": 1.0})[0], rotary_frequencies(64, 1e4, device="cpu")[0])
    with pytest.raises(ValueError, match="partial_rotary_factor"):
        _yarn(64, 1e4, {"rope_type": "default", "partial_rotary_factor": 0.5})
    # a value of None is a name that is not there
    assert torch.equal(_yarn(64, 1e4, {**DEEPSEEK, "low_freq_factor": None, "attention_factor": None})[0], _yarn(64, 1e4, DEEPSEEK)[0])
    for missing in ("factor", "original_max_position_embeddings"):
        with pytest.raises(ValueError, match=missing):
            _yarn(64, 1e4, {k: v for k, v in DEEPSEEK.items() if k != missing})
