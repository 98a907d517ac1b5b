"""Tables of scaled rotary positions against the formulas in 64 bits, pair by pair, and the refusal of what a scaling does not know."""
import math

import pytest

torch = pytest.importorskip("torch")
from kairos_amd.rotary import rotary_frequencies, rotary_table

YARN = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096}


def yarn_by_pair(R, base, factor, original, truncate=True, fast=32.0, slow=1.0):
    """A pair turns original / wavelength times within the original length; the pair that turns n times is i = R ln(original / (2 pi n)) /
    (2 ln base)."""
    ends = [R / 2 * math.log(original / (2 * math.pi * n)) / math.log(base) for n in (fast, slow)]
    if truncate:
        ends = [math.floor(ends[0]), math.ceil(ends[1])]
    out = []
    for i in range(R // 2):
        at = min(max((i - ends[0]) / (ends[1] - ends[0]), 0.0), 1.0)      # 0: kept, 1: divided
        f = base ** (-2.0 * i / R)
        out.append(f * (1 - at) + f / factor * at)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("truncate", [None, True, False])
@pytest.mark.parametrize("R, base, factor, original", [(64, 150000.0, 32.0, 4096), (128, 1000000.0, 4.0, 32768), (64, 10000.0, 40.0, 4096)])
def test_yarn_pair_by_pair(R, base, factor, original, truncate):
    scaling = dict(YARN, factor=factor, original_max_position_embeddings=original, truncate=truncate)
    got, gain = rotary_frequencies(R, base, scaling)
    assert torch.allclose(got, yarn_by_pair(R, base, factor, original, truncate is not False), rtol=1e-12, atol=0)
    assert gain == 0.1 * math.log(factor) + 1.0
    # an end moves by up to one pair of some sixteen: the two forms are per cents apart, so a key that is passed over shows
    assert (yarn_by_pair(R, base, factor, original, True) / yarn_by_pair(R, base, factor, original, False) - 1).abs().max() > 1e-3


@pytest.mark.parametrize("more, gain", [
    ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0),
    ({"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
    ({"mscale": 0.707, "mscale_all_dim": 0.5}, (0.0707 * math.log(32.0) + 1) / (0.05 * math.log(32.0) + 1)),
    ({"mscale": 1.0, "mscale_all_dim": 0.5, "attention_factor": 1.25}, 1.25),
    ({"mscale": None, "mscale_all_dim": None, "attention_factor": None}, 0.1 * math.log(32.0) + 1),
    ({}, 0.1 * math.log(32.0) + 1),
])
def test_yarn_gain(more, gain):
    freq, got = rotary_frequencies(64, 10000.0, dict(YARN, **more))
    assert abs(got - gain) < 1e-14 and torch.equal(freq, rotary_frequencies(64, 10000.0, YARN)[0])
    t = rotary_table(4, 64, 10000.0, dict(YARN, **more), device="cpu")
    assert abs(float(t[0, 0, 0]) - gain) <= gain * 2.0 ** -24


def test_yarn_betas():
    got, _ = rotary_frequencies(64, 10000.0, dict(YARN, beta_fast=16, beta_slow=2))
    assert torch.allclose(got, yarn_by_pair(64, 10000.0, 32.0, 4096, fast=16.0, slow=2.0), rtol=1e-12, atol=0)


def test_the_base_may_stand_in_the_scaling():
    plain, _ = rotary_frequencies(64, 500000.0)
    for scaling in ({"rope_type": "default", "rope_theta": 500000.0}, {"rope_type": "default", "type": "default", "rope_theta": 500000,
                                                                           "partial_rotary_factor": 1.0}):
        assert torch.equal(rotary_frequencies(64, None, scaling)[0], plain)
        assert torch.equal(rotary_frequencies(64, scaling=scaling)[0], plain)
        assert torch.equal(rotary_frequencies(64, 500000.0, scaling)[0], plain)
        with pytest.raises(ValueError, match="rope_theta"):
            rotary_frequencies(64, 10000.0, scaling)
    assert torch.equal(rotary_frequencies(64)[0], rotary_frequencies(64, 10000.0, {"rope_type": "default"})[0])
    yarn = dict(YARN, rope_theta=150000.0)
    assert torch.equal(rotary_frequencies(64, scaling=yarn)[0], rotary_frequencies(64, 150000.0, YARN)[0])


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("bad", [
    dict(YARN, mscale=1.0), dict(YARN, mscale_all_dim=1.0), dict(YARN, mscale=0.0, mscale_all_dim=1.0), dict(YARN, mscale=1.0, mscale_all_dim=0),
    dict(YARN, truncate=0), dict(YARN, beta_fast=1.0, beta_slow=2.0), dict(YARN, beta_slow=0.0), dict(YARN, attention_factor=-1.0),
    dict(YARN, original_max_position_embeddings=None), {"rope_type": "yarn", "factor": 4.0}, {"rope_type": "yarn", "original_max_position_embeddings": 4096},
    dict(YARN, low_freq_factor=1.0), dict(YARN, short_factor=[1.0]), dict(YARN, factor=float("nan")), dict(YARN, factor="4"), dict(YARN, type="linear"),
    dict(YARN, partial_rotary_factor=0.5), {k: v for k, v in LLAMA3.items() if k != "low_freq_factor"}, dict(LLAMA3, high_freq_factor=1.0),
    dict(LLAMA3, beta_fast=32.0), {"rope_type": "linear", "factor": 4.0, "mscale": 1.0}, {"rope_type": "default", "factor": 4.0},
    {"rope_type": "default", "mrope_section": [16, 24, 24]}, {"type": "dynamic", "factor": 2.0}, {"rope_type": "longrope", "factor": 2.0}, {}, {"rope_theta": 10000.0},
])
def test_what_a_scaling_does_not_know_is_refused(bad):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        rotary_frequencies(64, 10000.0, bad)
