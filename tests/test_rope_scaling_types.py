"""Rope scalings that name no type, on the CPU: refused, never taken for none."""

import json

import pytest

from quail_amd.loader import config_from_json
from quail_amd.rotary import RotaryEmbedding, frequencies, scaling_type


def config(**changes):
    with open("tests/golden/qwen3-4b-fp8.config.json") as f:
        return json.load(f) | changes


UNTYPED = [{"factor": 4.0}, {"mrope_section": [16, 24, 24]}, {"rope_theta": 1e6, "factor": 4.0},
           {"rope_type": None, "factor": 4.0}, {"type": "", "original_max_position_embeddings": 32768}]


@pytest.mark.parametrize("scaling", UNTYPED)
def test_a_scaling_without_a_type_is_refused(scaling):
    with pytest.raises(ValueError, match="no rope_type"):
        frequencies(64, 1e6, scaling, 40960)
    with pytest.raises(ValueError, match="no rope_type"):
        RotaryEmbedding(64, scaling=scaling, device="cpu")
    for name in ("rope_scaling", "rope_parameters"):
        with pytest.raises(ValueError, match="no rope_type"):
            config_from_json(config(**{name: scaling}), scaled_rope=True)
    for name, match in (("rope_scaling", "rope_scaling"), ("rope_parameters", "no rope_type")):
        with pytest.raises(ValueError, match=match):
            config_from_json(config(**{name: scaling}))


def test_types_by_either_name():
    assert scaling_type(None) == scaling_type({}) == scaling_type({"rope_theta": 1e4}) == "default"
    assert scaling_type({"rope_type": None, "factor": None, "rope_theta": 1e4}) == "default"
    assert scaling_type({"rope_type": "linear", "factor": 2.0}) == scaling_type({"type": "linear"}) == "linear"
    assert scaling_type({"rope_type": None, "type": "yarn", "factor": 2.0}) == "yarn"
    a, b = (frequencies(64, 1e6, {**kind, "factor": 2.0}) for kind in (dict(type="linear", rope_type=None),
                                                                        dict(rope_type="linear")))
    assert a[0].equal(b[0]) and a[1] == b[1]
    # a type under the older name in rope_parameters
    with pytest.raises(ValueError, match="rope_parameters"):
        config_from_json(config(rope_parameters={"type": "yarn", "factor": 4.0}))


def test_parameters_of_no_scaling_are_read():
    c = config()
    theta = c.pop("rope_theta")
    for rope in ({"rope_theta": theta}, {"rope_type": "default", "rope_theta": theta}):
        for scaled in (False, True):
            got = config_from_json(c | {"rope_parameters": rope}, scaled_rope=scaled)
            assert got.theta == theta and got.max_positions == c["max_position_embeddings"]
