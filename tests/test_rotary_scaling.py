"""CPU: the tables of the rotation with every number that a model's configuration may hold for them."""
import math

import pytest
import torch

from sonar_amd.rotary import rotary_cos_sin, rotary_rates

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


def size_of(**more):
    """What cosines and sines are multiplied by: the cosine of the angle 0."""
    return float(rotary_cos_sin(64, 1, scaling={**YARN, **more})[0, 0])


@pytest.mark.parametrize("more,want", [
    (dict(mscale=1.0, mscale_all_dim=1.0), 1.0), (dict(mscale=0.707, mscale_all_dim=1.0), 0.9210423553163399),
    (dict(mscale=1.0, mscale_all_dim=0.5), (0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1)),
    (dict(mscale=0.5, mscale_all_dim=1.0, factor=0.5), 1.0), (dict(mscale=0.5, mscale_all_dim=1.0, attention_factor=0.25), 0.25),
    (dict(mscale=1.0, mscale_all_dim=0), 1.3688879454113936), ({}, 1.3688879454113936)])
def test_size_of_yarn_tables(more, want):
    """Two numbers for the size: their quotient counts.  (Half a step of float32, and that of the test's own number.)"""
    assert abs(size_of(**more) - want) <= 2.0 ** -23 * want


@pytest.mark.parametrize("more", [dict(mscale=0.707), dict(mscale_all_dim=0.707), dict(mscale=0.707, mscale_all_dim=0.0)])
def test_one_of_two_sizes_is_refused(more):
    with pytest.raises(ValueError, match="mscale"):
        size_of(**more)


@pytest.mark.parametrize("truncate,rates", [
    # pairs 8, 9 and 17, 18 lie beside the ends of the line, 8.09 and 17.40; whole ends are 8 and 18
    (False, {0: 1.0, 7: 0.07374456524848938, 8: 0.05081327259540558, 9: 0.031705696135759354, 12: 0.006794959306716919,
             16: 0.0004564839182421565, 17: 0.00012931869423482567, 18: 3.830881178146228e-05, 31: 3.023511396804679e-07}),
    (True, {7: 150000.0 ** (-14 / 64), 8: 150000.0 ** (-16 / 64), 9: 150000.0 ** (-18 / 64) * (0.9 + 0.1 / 32),
            17: 150000.0 ** (-34 / 64) * (0.1 + 0.9 / 32), 18: 150000.0 ** (-36 / 64) / 32})])
def test_ends_of_the_yarn_line(truncate, rates):
    """The numbers for ends that are not rounded are another implementation's, in float32 (each off by a few steps of 2^-23)."""
    got = rotary_rates(64, 150000.0, {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096, "truncate": truncate})
    for pair, want in rates.items():
        assert abs(got[pair] - want) <= 4 * 2.0 ** -23 * want, pair
    ends = [64 * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(150000.0)) for turns in (32, 1)]
    if not truncate:   # and by the definition
        stay = [1 - min(max((i - ends[0]) / (ends[1] - ends[0]), 0), 1) for i in range(32)]
        want = [150000.0 ** (-2 * i / 64) * (s + (1 - s) / 32) for i, s in enumerate(stay)]
        assert torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=1e-13)
    assert 8 < ends[0] < 9 and 17 < ends[1] < 18


LINEAR = {"rope_type": "linear", "factor": 4.0}


@pytest.mark.parametrize("scaling,message", [
    ({**YARN, "beta": 3}, "beta"), ({**LINEAR, "truncate": False}, "truncate"), ({"rope_type": "default", "mrope_section": [8, 12, 12]}, "mrope_section"),
    ({"rope_type": "linear"}, "factor"), ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0}, "original_max"),
    ({"rope_type": "longrope", "short_factor": [1.0]}, "longrope"), ({"factor": 4.0}, "rope_type"), ({**LINEAR, "type": "yarn"}, "type"),
    ({**LINEAR, "rope_theta": 5e5}, "rope_theta"), ({**LINEAR, "factor": 0.0}, "factor")])
def test_what_is_not_known_is_refused(scaling, message):
    for table in (lambda: rotary_rates(64, scaling=scaling), lambda: rotary_cos_sin(64, 3, scaling=scaling)):
        with pytest.raises(ValueError, match=message):
            table()


@pytest.mark.parametrize("scaling", [
    {**LINEAR, "type": "linear"}, {"type": "linear", "factor": 4.0}, {**LINEAR, "rope_theta": 10000.0}, {**LINEAR, "partial_rotary_factor": 0.5},
    {**LINEAR, "original_max_position_embeddings": 4096}, {**LINEAR, "truncate": None}])
def test_what_changes_no_table(scaling):
    assert torch.equal(rotary_cos_sin(64, 9, scaling=scaling), rotary_cos_sin(64, 9, scaling=LINEAR))


def test_numbers_that_are_none_are_absent():
    none = dict.fromkeys(("beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"))
    assert torch.equal(rotary_cos_sin(64, 9, scaling={**YARN, **none}), rotary_cos_sin(64, 9, scaling=YARN))
