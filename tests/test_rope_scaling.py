"""Keys of a model's `rope_scaling` entry that change frequencies or the factor on cosine and sine: taken,
or refused.  Against formulas written out here, in 64 bits."""
import math

import pytest
import torch

from sglang_diffusion_amd.layers.rotary import scaled_inv_freq

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


def ramp_by_hand(rot, base, trained, factor, fast, slow, whole):
    """Pair i keeps the share 1 - (i - first) / (last - first) of its frequency, the rest is divided."""
    at = [rot / 2 * math.log(trained / (2 * math.pi * t), base) for t in (fast, slow)]
    if whole:
        at = [math.floor(at[0]), math.ceil(at[1])]
    first, last = max(at[0], 0), min(at[1], rot - 1)
    out = []
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        share = min(max((i - first) / (last - first), 0.0), 1.0)
        out.append(f * (1 - share) + f / factor * share)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("rot,base", [(64, 10000.0), (128, 500000.0)])
@pytest.mark.parametrize("fast,slow", [(32, 1), (16, 2)])
def test_ends_of_the_ramp(rot, base, fast, slow):
    for more, whole in (({}, True), ({"truncate": True}, True), ({"truncate": False}, False)):
        f, _ = scaled_inv_freq(rot, base, dict(YARN, beta_fast=fast, beta_slow=slow, **more))
        assert torch.allclose(f, ramp_by_hand(rot, base, 4096, 40.0, fast, slow, whole), rtol=1e-12)
    both = [scaled_inv_freq(rot, base, dict(YARN, truncate=t))[0] for t in (True, False)]
    assert not torch.allclose(*both, rtol=1e-4)


def test_factor_on_cosine_and_sine():
    def factor(**more):
        return scaled_inv_freq(64, 10000.0, dict(YARN, **more))[1]

    assert factor() == pytest.approx(0.1 * math.log(40) + 1)
    assert factor(mscale=1.0, mscale_all_dim=1.0) == 1.0
    assert factor(mscale=0.707, mscale_all_dim=1.0) == pytest.approx((0.0707 * math.log(40) + 1) / (0.1 * math.log(40) + 1))
    assert factor(mscale=1.0, mscale_all_dim=0.5) == pytest.approx((0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1))
    assert factor(mscale=1.0, mscale_all_dim=0.5, attention_factor=1.5) == 1.5
    assert factor(attention_factor=None, beta_fast=None) == factor()
    assert scaled_inv_freq(64, 10000.0, dict(YARN, factor=1.0, mscale=2.0, mscale_all_dim=1.0))[1] == 1.0
    for one in ({"mscale": 1.0}, {"mscale_all_dim": 1.0}, {"mscale": 1.0, "mscale_all_dim": 0}):
        with pytest.raises(ValueError, match="mscale"):
            factor(**one)


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default", "factor": 2.0},
    {"rope_type": "linear", "factor": 2.0, "mscale": 1.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192, "truncate": False},
    dict(YARN, low_freq_factor=1.0),
    dict(YARN, rope_theta=10000.0),
    dict(YARN, partial_rotary_factor=0.5),
    {"factor": 2.0},
])
def test_keys_without_a_use_are_refused(scaling):
    with pytest.raises(ValueError, match="does not use"):
        scaled_inv_freq(64, 10000.0, scaling)


def test_types():
    assert torch.equal(scaled_inv_freq(64, scaling={"type": "linear", "factor": 4.0})[0],
                       scaled_inv_freq(64, scaling={"rope_type": "linear", "type": "linear", "factor": 4.0})[0])
    with pytest.raises(ValueError, match="differ"):
        scaled_inv_freq(64, scaling={"rope_type": "linear", "type": "yarn", "factor": 4.0})
    with pytest.raises(ValueError, match="unknown"):
        scaled_inv_freq(64, scaling={"rope_type": "longrope"})
    with pytest.raises(ValueError, match="low_freq_factor"):
        scaled_inv_freq(64, scaling={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
                                     "original_max_position_embeddings": 8192})
    entry = dict(YARN)
    scaled_inv_freq(64, scaling=entry)
    assert entry == YARN                                  # left as it was
