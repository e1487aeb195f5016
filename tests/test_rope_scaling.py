"""What a model's rope scaling may state, and what is refused rather than filled in (CPU only)."""

import math

import pytest

from mla_kv_quant_amd import rotary

YARN = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096}
LONG = {"type": "longrope", "original_max_position_embeddings": 4096, "long_factor": [2.0] * 4, "short_factor": [1.0] * 4}


@pytest.mark.parametrize("scaling,word", [
    (LONG, "factor"),  # the context's factor lies elsewhere in the configuration
    ({k: v for k, v in dict(LONG, factor=4).items() if k != "original_max_position_embeddings"}, "original"),
    (dict(LONG, factor=4, long_mscale=1.2), "long_mscale"), (dict(YARN, finetuned_scale=2.0), "finetuned_scale"),
    (dict(YARN, mscale=0.707), "together"), (dict(YARN, mscale_all_dim=0.707), "together"),
    (dict(YARN, mscale=0.707, mscale_all_dim=0), "together"),
    ({"type": "linear", "factor": 2, "beta_fast": 32}, "beta_fast"), ({"rope_type": "default", "mrope_section": [8, 12]}, "mrope"),
    (dict(YARN, rope_theta=1000000.0), "rope_theta"), ({"factor": 4}, "factor"),
])
def test_entries_that_are_unknown_or_missing(scaling, word):
    with pytest.raises(ValueError, match=word):
        rotary.frequencies(8, scaling=scaling)


def test_entries_that_say_nothing():
    """Missing, None, and what agrees with the base; mscale of one by itself is what it is without."""
    want = rotary.frequencies(64, scaling=YARN)
    for more in ({"mscale": 1.0}, {"mscale": 1}, {"mscale": None, "attention_factor": None, "beta_fast": None},
                 {"rope_theta": 10000.0, "truncate": True}, {"mscale_all_dim": 0}, {"rope_type": "yarn"}):
        assert rotary.frequencies(64, scaling=dict(YARN, **more)) == want
    plain = rotary.frequencies(64)
    assert rotary.frequencies(64, scaling={"rope_type": "default", "rope_theta": 10000.0}) == plain
    assert rotary.frequencies(64, scaling={"type": "linear", "factor": 1, "original_max_position_embeddings": 4096}) == plain
    by = rotary.frequencies(8, scaling=dict(LONG, attention_factor=1.25, long=False))
    assert by[1] == 1.25 and by[0] == rotary.frequencies(8)[0]


def test_a_yarn_ramp_between_numbers_that_are_not_whole():
    """64 ln(4096 / (32 2 pi)) / (2 ln 10000) = 10.4722, 64 ln(4096 / 2 pi) / (2 ln 10000) = 22.5134: pair 15 is slowed by
    (15 - 10.4722) / (22.5134 - 10.4722) of the way, pairs 10 and 23 by nothing and all of it."""
    f = rotary.frequencies(64)[0]
    g = rotary.frequencies(64, scaling=dict(YARN, truncate=False))[0]
    lo, hi = (32 * math.log(4096 / (b * 2 * math.pi)) / math.log(10000) for b in (32, 1))
    assert (lo, hi) == pytest.approx((10.4722, 22.5134), abs=1e-3)
    for i in (0, 10, 11, 15, 22, 23, 31):
        slowed = min(max((i - lo) / (hi - lo), 0), 1)
        assert g[i] / f[i] == pytest.approx(1 - slowed + slowed / 40, rel=1e-12)
    h = rotary.frequencies(64, scaling=YARN)[0]
    assert g[15] != h[15] and g[0] == h[0] and g[31] == h[31]
