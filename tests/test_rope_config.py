"""Rotation plans from a model's config.json, against numbers written out from the
formulas (no GPU)."""
import math

import pytest

import moe_infer_amd as m


def config(theta=1e7, **scaling):
    return {"head_dim": 256, "partial_rotary_factor": 0.25, "rope_theta": theta,
            "max_position_embeddings": 262144, "rope_scaling": scaling or None}


# yarn by factor 4 of 32 pairs: pairs up to `first` keep their frequency, pairs from `last` on have a
# quarter of it, and those between lie on a straight line over their numbers.  The ends are
# 64 ln(L / (2 pi turns)) / (2 ln theta), down for 32 turns and up for 1:
#   theta 1e7, L 32768     10.11, 16.99
#   theta 1e7, L 262144    14.24, 21.12
#   theta 1e6, L 32768     11.80, 19.82
@pytest.mark.parametrize("theta,rows,first,last", [(1e7, 32768, 10, 17), (1e7, 262144, 14, 22), (1e6, 32768, 11, 20)])
def test_yarn_is_a_ramp_over_the_pairs(theta, rows, first, last):
    r = m.Rope.from_config(config(theta, rope_type="yarn", factor=4.0, original_max_position_embeddings=rows))
    for i, f in enumerate(r.frequencies):
        share = 0.0 if i <= first else 1.0 if i >= last else (i - first) / (last - first)
        assert math.isclose(f, theta ** (-i / 32) * (1 - 0.75 * share), rel_tol=1e-14), i
    assert math.isclose(r.factor, 1.1386294361119891, rel_tol=1e-15)  # 0.1 ln 4 + 1
    same = m.Rope(64, theta, scaling={"type": "yarn", "factor": 4.0, "original_max_position": rows})
    assert same.frequencies == r.frequencies and same.factor == r.factor


def test_yarn_in_numbers():
    """theta 1e6, pair 16: 1e-3 times 1 - 0.75 * 5 / 9."""
    r = m.Rope.from_config(config(1e6, rope_type="yarn", factor=4.0, original_max_position_embeddings=32768))
    assert math.isclose(r.frequencies[16], 5.8333333333333333e-4, rel_tol=1e-14)
    assert r.frequencies[0] == 1.0 and math.isclose(r.frequencies[31], 0.25 * 1e6 ** (-31 / 32), rel_tol=1e-14)


def test_yarn_by_turns_has_a_name_of_its_own():
    """A line in the turns over the first context: pair 16 of theta 1e6 makes 5.2152 of them."""
    r = m.Rope(64, 1e6, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 32768, "ramp": "turns"})
    g = (5.215189175235227 - 1) / 31
    assert math.isclose(r.frequencies[16], 1e-3 * (g + (1 - g) / 4), rel_tol=1e-12)
    for bad in ({"ramp": "rows"}, {"beta_slow": 0.0}, {"original_max_position": 3}):
        with pytest.raises(ValueError):
            m.Rope(64, 1e6, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 32768, **bad})
    with pytest.raises(ValueError):
        m.Rope(64, 1.0, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 32768})
