"""Rotary positions on the CPU: frequencies against transformers' own rotary
embeddings, the engine's table, checkpoints with scaled rope, and refusals."""

import json
import math

import pytest
import torch

from quail_amd.loader import config_from_json, load_qwen3_fp8
from quail_amd.model import CONFIGS, build_synthetic
from quail_amd.rotary import RotaryEmbedding, frequencies
from tests.helpers import write_hf_checkpoint

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


def _theirs(d, base, scaling, max_positions):
    from transformers import Qwen3Config
    from transformers.models.qwen3.modeling_qwen3 import Qwen3RotaryEmbedding
    cfg = Qwen3Config(head_dim=d, rope_theta=base, max_position_embeddings=max_positions,
                      hidden_size=256, num_attention_heads=4, rope_scaling=scaling,
                      **({"rope_parameters": {**scaling, "rope_theta": base}} if scaling else {}))
    rot = Qwen3RotaryEmbedding(cfg)
    return rot.inv_freq.double(), rot.attention_scaling


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("base", [10000.0, 1e6])
@pytest.mark.parametrize("scaling", [
    None, YARN, {"rope_type": "linear", "factor": 8.0},
    {"rope_type": "yarn", "factor": 2.5, "original_max_position_embeddings": 4096, "beta_fast": 16,
     "beta_slow": 2, "attention_factor": 1.25},
    {"rope_type": "yarn", "factor": 1.0, "original_max_position_embeddings": 40960}])
def test_frequencies_are_transformers(d, base, scaling):
    want, want_factor = _theirs(d, base, dict(scaling) if scaling else None, 40960)
    got, factor = frequencies(d, base, scaling, 40960)
    # theirs are formed in fp32: a power, a quotient, and with a ramp two products and a sum
    assert float((got / want - 1).abs().max()) <= 2.0 ** -19
    assert factor == pytest.approx(want_factor, rel=1e-12)


def test_cache_rows_are_the_angles_of_far_positions():
    d, rows = 128, 140000
    rot = RotaryEmbedding(d, base=1e6, scaling=YARN, max_positions=rows, dtype=torch.float32,
                          device="cpu")
    inv, factor = frequencies(d, 1e6, YARN)
    cache = rot.cos_sin_cache
    assert cache.shape == (rows, d) and factor == 0.1 * math.log(4.0) + 1
    for p in (0, 1, 40959, 40960, 131071, rows - 1):
        angle = (p * inv)
        want = torch.cat([angle.cos(), angle.sin()]) * factor
        assert float((cache[p].double() - want).abs().max()) <= 2.0 ** -23
    assert rot.cos_sin_cache is cache


def test_cache_of_no_scaling_is_the_checkpoints_table_within_its_angles():
    from oracle.qwen3_ref import rope_cache
    got = RotaryEmbedding(64, base=1e6, max_positions=512, device="cpu").cos_sin_cache
    want = rope_cache(64, 512, 1e6)
    # theirs rounds frequencies and angles (up to 511) to fp32, both a result to bf16
    assert got.dtype == want.dtype
    assert float((got.double() - want.double()).abs().max()) <= 2.0 ** -8 + 512 * 2.0 ** -21


@pytest.mark.parametrize("kw,match", [
    (dict(rotary_dim=63), "even"), (dict(rotary_dim=130), "even"), (dict(rotary_dim=0), "even"),
    (dict(base=1.0), "base"), (dict(base=float("nan")), "base"),
    (dict(scaling={"rope_type": "dynamic", "factor": 2.0}), "rope_type"),
    (dict(scaling={"rope_type": "linear"}), "factor"),
    (dict(scaling={"rope_type": "linear", "factor": 0.5}), "factor"),
    (dict(scaling={"rope_type": "linear", "factor": float("inf")}), "factor"),
    (dict(scaling={"rope_type": "yarn", "factor": 4.0, "mscale": 1.0}), "mscale"),
    (dict(scaling={"rope_type": "yarn", "factor": 4.0, "truncate": False}), "truncate"),
    (dict(scaling={"rope_type": "yarn", "factor": 4.0, "beta_fast": 1, "beta_slow": 2}), "beta"),
    (dict(scaling={"rope_type": "yarn", "factor": 4.0}, max_positions=None), "original_max"),
    (dict(inv_freq=[1.0] * 3), "inv_freq"), (dict(inv_freq=[1.0] * 64, scaling=YARN), "both"),
    (dict(dtype=torch.float16), "bf16 or fp32")])
def test_modules_that_are_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        RotaryEmbedding(128, device="cpu", **kw)


@pytest.mark.parametrize("kw", [dict(rotary_dim=64), dict(interleaved=True)])
def test_the_engines_table_is_refused_for_other_layouts(kw):
    with pytest.raises(ValueError, match="half pairs"):
        RotaryEmbedding(128, device="cpu", **kw).cos_sin_cache


def _rows(n=3, heads=2, d=64, dtype=torch.bfloat16):
    return torch.zeros(n, heads * d, dtype=dtype)


@pytest.mark.parametrize("positions", [torch.zeros(4, dtype=torch.int64), torch.zeros(3, dtype=torch.int32),
                                       torch.zeros(6, dtype=torch.int64)[::2],
                                       torch.zeros(3, 1, dtype=torch.int64)])
def test_positions_that_are_refused(positions):
    with pytest.raises(ValueError, match="positions"):
        RotaryEmbedding(64, device="cpu")(positions, _rows())


@pytest.mark.parametrize("q,k,out,match", [
    (_rows(dtype=torch.float64), None, None, "float64"),
    (_rows(), _rows(dtype=torch.float16), None, "float16"),
    (torch.zeros(3, 100, dtype=torch.bfloat16), None, None, "contiguous heads"),
    (torch.zeros(3, 2, 128, dtype=torch.bfloat16)[..., ::2], None, None, "contiguous heads"),
    (torch.zeros(3, 4, 64, dtype=torch.bfloat16)[:, ::2], None, None, "contiguous heads"),
    (torch.zeros(3, 0, dtype=torch.bfloat16), None, None, "contiguous heads"),
    (_rows(), _rows(2), None, "contiguous heads"),
    (_rows(1).expand(3, -1), None, None, "overlap"),
    (_rows(), None, _rows(2), "out of"), (_rows(), None, _rows(dtype=torch.float32), "out of"),
    (_rows(), None, None, "one GPU")])
def test_rows_that_are_refused(q, k, out, match):
    with pytest.raises(ValueError, match=match):
        RotaryEmbedding(64, device="cpu")(torch.zeros(3, dtype=torch.int64), q, k, out=out)


def _checkpoint(tmp_path, **changes):
    cfg = CONFIGS["tiny"]
    path = write_hf_checkpoint(build_synthetic(cfg, seed=3, device="cpu"), cfg, tmp_path / "c")
    config = json.loads((path / "config.json").read_text())
    config.update(changes)
    (path / "config.json").write_text(json.dumps(config))
    return path


def test_scaled_checkpoints_load_where_they_are_asked_for(tmp_path):
    path = _checkpoint(tmp_path, rope_scaling={"type": "yarn", "factor": 4.0}, max_position_embeddings=4096)
    with pytest.raises(ValueError, match="rope_scaling"):
        load_qwen3_fp8(path, device="cpu")
    model = load_qwen3_fp8(path, device="cpu", scaled_rope=True)
    rotary = model.model.layers[0].self_attn.rotary_emb
    want, factor = frequencies(64, CONFIGS["tiny"].theta, YARN | {"original_max_position_embeddings": 4096})
    assert torch.equal(rotary.inv_freq, want) and rotary.factor == factor
    assert rotary.cos_sin_cache.shape == (16384, 64) and model.config.max_positions == 16384


def test_checkpoints_of_no_scaling_load_the_same_with_scaled_rope(tmp_path):
    path = _checkpoint(tmp_path)
    a, b = (load_qwen3_fp8(path, device="cpu", scaled_rope=s) for s in (False, True))
    assert a.config == b.config
    assert torch.equal(*(m.model.layers[0].self_attn.rotary_emb.cos_sin_cache for m in (a, b)))


def test_positions_not_named_are_the_checkpoints_own(tmp_path):
    path = _checkpoint(tmp_path, max_position_embeddings=4096, rope_scaling={
        "type": "yarn", "factor": 4.0, "original_max_position_embeddings": None})
    rotary = load_qwen3_fp8(path, device="cpu", scaled_rope=True).model.layers[0].self_attn.rotary_emb
    want, _ = frequencies(64, CONFIGS["tiny"].theta, YARN | {"original_max_position_embeddings": 4096})
    assert torch.equal(rotary.inv_freq, want) and rotary.max_positions == 16384


def test_unknown_scalings_are_refused(tmp_path):
    path = _checkpoint(tmp_path, rope_scaling={"rope_type": "dynamic", "factor": 4.0})
    with pytest.raises(ValueError, match="rope_type"):
        load_qwen3_fp8(path, device="cpu", scaled_rope=True)


def test_scaled_config_reads_rope_parameters():
    with open("tests/golden/qwen3-4b-fp8.config.json") as f:
        config = json.load(f)
    theta = config.pop("rope_theta")
    config["rope_parameters"] = YARN | {"rope_theta": theta}
    cfg = config_from_json(config, scaled_rope=True)
    assert cfg.max_positions == 131072 and cfg.theta == theta
