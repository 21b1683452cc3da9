"""Rotation plans from a model's config.json, against numbers written out from the
formulas (no GPU)."""
import copy
import ctypes
import math
import pickle

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


def test_configs_as_models_have_them():
    """Keys that such configs hold beside those that a type needs."""
    for kind in ("linear", "ntk"):
        r = m.Rope.from_config(config(rope_type=kind, factor=4.0, original_max_position_embeddings=32768))
        assert r.frequencies == m.Rope(64, 1e7, scaling={"type": kind, "factor": 4.0}).frequencies
    # no length of the first context: the config's own (262144)
    r = m.Rope.from_config(config(type="yarn", factor=4.0, beta_fast=32, beta_slow=None))
    assert math.isclose(r.frequencies[18], 1e7 ** (-18 / 32) * 0.625, rel_tol=1e-14)  # half way from 14 to 22
    with pytest.raises(ValueError):
        m.Rope.from_config({"rope_scaling": {"rope_type": "yarn", "factor": 4.0}})
    # ends that are not rounded: 10.1125 and 16.9932 for 32768 rows
    r = m.Rope.from_config(config(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768, truncate=False))
    assert math.isclose(r.frequencies[14], 1e7 ** (-14 / 32) * (1 - 0.75 * (14 - 10.112548975) / 6.880685616), rel_tol=1e-9)
    assert r.frequencies[11] < 1e7 ** (-11 / 32) and r.frequencies[16] > 0.25 * 1e7 ** (-16 / 32)


@pytest.mark.parametrize("keys,factor", [
    ({}, 1.1386294361119891), ({"attention_factor": 1.5}, 1.5), ({"attention_factor": None}, 1.1386294361119891),
    ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0), ({"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
    ({"mscale": 1.0, "mscale_all_dim": 0.5}, 1.1386294361119891 / 1.0693147180559945),  # 0.1 k ln 4 + 1 each
    ({"mscale": 1.0}, 1.1386294361119891), ({"mscale": 1.0, "mscale_all_dim": 0}, 1.1386294361119891),
    ({"mscale": 0.5, "mscale_all_dim": 1.0, "attention_factor": 2.0}, 2.0)])
def test_yarn_factors(keys, factor):
    r = m.Rope.from_config(config(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768, **keys))
    assert math.isclose(r.factor, factor, rel_tol=1e-15)


@pytest.mark.parametrize("keys", [{"rope_type": "longrope", "factor": 4.0}, {"rope_type": "yarn"},
                                  {"rope_type": "yarn", "factor": 4.0, "mscale": 0.5},  # read in two ways
                                  {"rope_type": "yarn", "factor": 4.0, "mscale_all_dim": 0.5},
                                  {"rope_type": "yarn", "factor": 4.0, "short_factor": [1.0]},
                                  {"rope_type": "linear", "factor": 4.0, "beta_fast": 3}])
def test_configs_that_are_refused(keys):
    with pytest.raises(ValueError):
        m.Rope.from_config(config(**keys))


def test_newer_configs_hold_all_of_it_in_one_place():
    """rope_parameters: theta, the rotated part and the scaling."""
    p = {"rope_type": "yarn", "rope_theta": 1e6, "partial_rotary_factor": 0.5, "factor": 4.0,
         "original_max_position_embeddings": 32768}
    for c in ({"head_dim": 256, "rope_parameters": p}, {"text_config": {"head_dim": 256, "rope_parameters": p}}):
        r = m.Rope.from_config(c)
        want = m.Rope(128, 1e6, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 32768})
        assert r.rotary_dim == 128 and r.frequencies == want.frequencies and r.factor == want.factor
    r = m.Rope.from_config({"rope_parameters": {"rope_type": "default", "rope_theta": 1e4}})
    assert r.frequencies == m.Rope(64, 1e4).frequencies
    with pytest.raises(ValueError):  # one for each kind of layer
        m.Rope.from_config({"rope_parameters": {"full_attention": p, "sliding_attention": p}})


def test_a_copied_plan_has_frequencies_of_its_own():
    """What the C entry reads lives as long as the copy, whatever becomes of the original."""
    r = m.Rope(64, 1e6, "interleaved", {"type": "linear", "factor": 2.0})
    for other in (copy.deepcopy(r), copy.copy(r), pickle.loads(pickle.dumps(r))):
        assert other.frequencies == r.frequencies and other.layout == r.layout and other.factor == r.factor
        at, rotary_dim, interleaved, factor = other._args
        assert at == ctypes.addressof(other._f) != ctypes.addressof(r._f)
        assert tuple(other._f) == r.frequencies and (rotary_dim, interleaved, factor) == (64, 1, 1.0)
