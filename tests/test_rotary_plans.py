"""The frequencies of rotary plans, against values worked out from the published formulas in 50 digits."""
import math

import pytest

from kushkash_b200 import rotary_frequencies

PLAIN16 = [10000.0 ** (-i / 8) for i in range(8)]
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}
LONG = {"rope_type": "yarn", "factor": 40, "original_max_position_embeddings": 4096}
# 16 channels, theta 10000.  The pair x that turns b times over 1024 positions is 8 ln(1024 / (2 pi b)) / ln 10000: 1.414 for
# b = 32, 4.424 for b = 1.  Whole ends: 1 and 5; pair i keeps 1 - (i - 1) / 4 of its frequency and a quarter of the rest.
YARN_WHOLE = [1.0, 0.31622776601683794, 0.08125, 0.01976423537605237, 0.004375, 0.0007905694150420948, 0.00025,
              7.905694150420948e-05]
YARN_EXACT = [1.0, 0.31622776601683794, 0.08539863663460479, 0.01912677583148376, 0.0035569715211294347,
              0.0007905694150420948, 0.00025, 7.905694150420948e-05]
# 2048 positions: pairs 0-3 turn more than 4 times over them and stay, pairs 6 and 7 less than once and are divided by 8,
# pairs 4 (3.259 turns) and 5 (1.031) lie between
LLAMA3 = [1.0, 0.31622776601683794, 0.1, 0.03162277660168379, 0.007840188600689215, 0.00042363925004085826, 0.000125,
          3.952847075210474e-05]


@pytest.mark.parametrize("scaling,want,factor", [
    (None, PLAIN16, 1.0),
    ({"rope_type": "default", "rope_theta": 10000}, PLAIN16, 1.0),
    ({"rope_type": "linear", "factor": 8}, [f / 8 for f in PLAIN16], 1.0),
    ({"type": "linear", "factor": 8, "rope_theta": 10000.0, "original_max_position_embeddings": 4096}, [f / 8 for f in PLAIN16], 1.0),
    ({"rope_type": "ntk", "factor": 2.0}, [f * 2 ** (-i / 7) for i, f in enumerate(PLAIN16)], 1.0),
    (YARN, YARN_WHOLE, 0.1 * math.log(4) + 1),
    ({**YARN, "truncate": True, "attention_factor": None}, YARN_WHOLE, 0.1 * math.log(4) + 1),
    ({**YARN, "truncate": False}, YARN_EXACT, 0.1 * math.log(4) + 1),
    ({**YARN, "beta_fast": 32.0, "beta_slow": 1.0, "attention_factor": 1.25}, YARN_WHOLE, 1.25),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
      "original_max_position_embeddings": 2048}, LLAMA3, 1.0)])
def test_frequencies(scaling, want, factor):
    got, f = rotary_frequencies(16, 10000.0, scaling)
    assert got == pytest.approx(want, rel=1e-13) and f == pytest.approx(factor, rel=1e-13)      # (a few roundings of 2^-53)


def test_yarn_of_a_large_ramp():
    """64 channels, theta 150000, 4096 positions stretched 32 times: ends 8.09 and 17.40, not 8 and 18."""
    got, f = rotary_frequencies(64, 150000.0, {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096,
                                               "beta_fast": 32.0, "beta_slow": 1.0, "truncate": False})
    want = [0.10702442147781144, 0.03170569618466377, 0.006794959489732218, 0.0010526021013863348, 3.8308812373753384e-05,
            1.2532569824095001e-05]
    assert got[6:22:3] == pytest.approx(want, rel=1e-13) and f == pytest.approx(0.1 * math.log(32) + 1, rel=1e-13)


@pytest.mark.parametrize("keys,factor", [({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0),
                                         ({"mscale": 0.707, "mscale_all_dim": 1.0}, (0.0707 * math.log(40) + 1) / (0.1 * math.log(40) + 1)),
                                         ({"mscale": 1.0}, 0.1 * math.log(40) + 1), ({"mscale": 1.0, "mscale_all_dim": 0}, 0.1 * math.log(40) + 1),
                                         ({"mscale": 1.0, "mscale_all_dim": 1.0, "attention_factor": 2.0}, 2.0)])
def test_yarn_factor(keys, factor):
    assert rotary_frequencies(64, 10000.0, {**LONG, **keys})[1] == pytest.approx(factor, rel=1e-13)


@pytest.mark.parametrize("scaling", [{**YARN, "long_factor": [1.0]}, {**YARN, "low_freq_factor": 1.0}, {"rope_type": "linear", "factor": 2, "beta_fast": 3},
                                     {"rope_type": "default", "factor": 2.0}, {"rope_type": "linear", "factor": 2, "rope_theta": 500000.0},
                                     {"rope_type": "ntk", "factor": 2, "partial_rotary_factor": 0.5},
                                     {**LONG, "mscale": 0.707}, {**LONG, "mscale_all_dim": 1.0}])
def test_refused_keys(scaling):
    with pytest.raises(ValueError, match="rotary"):
        rotary_frequencies(16, 10000.0, scaling)


@pytest.mark.parametrize("r,theta,scaling", [(128, 500000.0, None), (64, 10000.0, None), (256, 1e6, {"rope_type": "linear", "factor": 3.0}),
                                             (20, 150000.0, {"rope_type": "ntk", "factor": 5.0}), (2, 10000.0, None)])
def test_turns_are_the_nearest_integers(r, theta, scaling):
    """2^64 f / 2 pi in 80 digits, f = theta^(-2i/r): a plan's entry is within half a count (of one turn in 2^64)."""
    import decimal

    import torch

    from kushkash_b200._rotary import make_rotary
    plan = make_rotary(torch.device("cpu"), 256, r, theta, False, scaling)
    with decimal.localcontext(decimal.Context(prec=80)):
        pi = decimal.Decimal("3.1415926535897932384626433832795028841971693993751058209749445923078164062862089986")
        factor = decimal.Decimal(scaling["factor"]) if scaling else 1
        for i, bits in enumerate(plan.turns.tolist()):
            log = -decimal.Decimal(2 * i) / r * decimal.Decimal(theta).ln()
            if scaling and scaling["rope_type"] == "ntk":
                log -= decimal.Decimal(2 * i) / (r - 2) * factor.ln()
            elif scaling:
                log -= factor.ln()
            turns = log.exp() / (2 * pi) * 2 ** 64
            assert abs(bits % 2 ** 64 - turns) <= decimal.Decimal("0.5000001")


def test_refused_values():
    for theta in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="rotary"):
            rotary_frequencies(16, theta)
    for scaling in ({"rope_type": "linear", "factor": math.inf}, {"rope_type": "linear", "factor": -2.0}, {**YARN, "beta_slow": -1},
                    {**YARN, "original_max_position_embeddings": 0}):
        with pytest.raises(ValueError, match="rotary"):
            rotary_frequencies(16, 10000.0, scaling)
