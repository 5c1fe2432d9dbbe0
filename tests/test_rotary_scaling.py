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
