"""Rotary tables and the loader's reading of a config against transformers' own module (the
installed transformers, fp32 on the CPU)."""
from __future__ import annotations

import math

import pytest
import torch

M = pytest.importorskip("transformers.models.qwen3_omni_moe.modeling_qwen3_omni_moe")

# What fp32 costs the module's table, relative: the exponent's rounding (2^-25 ln theta, at most
# 2^-21), the power and quotients (2^-22), and the blend's share, off by 2^-22, of up to
# scale - 1 <= 31 times the slowed frequency (2^-17).  Another rule is off by 2^-7 and more.
FP32 = 2.0 ** -16


def theirs(rope, head_dim=128, theta=1e6, **kw):
    """The module for a config with these rope parameters."""
    from transformers.models.qwen3_omni_moe.configuration_qwen3_omni_moe import (
        Qwen3OmniMoeTextConfig,
    )

    return M.Qwen3OmniMoeThinkerTextRotaryEmbedding(Qwen3OmniMoeTextConfig(
        hidden_size=128, num_attention_heads=2, num_key_value_heads=1, head_dim=head_dim,
        rope_scaling=dict(rope), rope_theta=theta, num_hidden_layers=1, num_experts=4,
        num_experts_per_tok=2, moe_intermediate_size=32, intermediate_size=64, **kw))


def close(ours, module):
    torch.testing.assert_close(ours.inv_freq.double(), module.inv_freq.double(), rtol=FP32, atol=0)
    assert math.isclose(ours.factor, module.attention_scaling, rel_tol=2.0 ** -22)


@pytest.mark.parametrize("dims,theta,scale,trained,kw", [
    (128, 1e6, 4.0, 32768, {}), (128, 1e4, 8.0, 4096, {}), (64, 1e4, 16.0, 2048, {}),
    (128, 1e6, 1.0, 32768, {}), (128, 1e6, 2.0, 262144, {"slow": 2.0, "fast": 16.0}),
    (128, 1e6, 4.0, 32768, {"whole": False}), (32, 500.0, 32.0, 100, {}),
    (128, 100.0, 4.0, 1000000, {}), (256, 1e6, 4.0, 20, {}), (128, 1e6, 4.0, 32768,
                                                             {"factor": 1.25})])
def test_scaled_tables_are_those_of_checkpoints(pkg, dims, theta, scale, trained, kw):
    rope = {"rope_type": "yarn", "factor": scale, "original_max_position_embeddings": trained}
    for ours, name in (("slow", "beta_slow"), ("fast", "beta_fast"), ("whole", "truncate"),
                       ("factor", "attention_factor")):
        if ours in kw:
            rope[name] = kw[ours]
    close(pkg.Rotary.scaled(dims, theta, scale, trained, blend="pairs", **kw),
          theirs(rope, dims, theta))
    if scale > 1 and (dims, theta) == (128, 1e6):  # the paper's text is another table
        other = pkg.Rotary.scaled(dims, theta, scale, trained, **{**kw, "whole": True})
        want = theirs(rope, dims, theta).inv_freq
        assert ((other.inv_freq - want).abs() > 2.0 ** -7 * want).any()


def test_divided_positions(pkg):
    close(pkg.Rotary.scaled(128, 1e6, 4.0), theirs({"rope_type": "linear", "factor": 4.0}))


def test_scaled_refuses(pkg):
    for kw, match in ((dict(blend="both"), "blend"), (dict(slow=0.0), "slow"),
                      (dict(scale=math.nan), "scale"),
                      (dict(blend="pairs", trained=2), "no pair")):
        a = {**dict(scale=4.0, trained=4096), **kw}
        with pytest.raises(RuntimeError, match=match):
            pkg.Rotary.scaled(64, 1e4, a.pop("scale"), a.pop("trained"), **a)


CONFIGS = [
    {"rope_type": "default"}, {"type": "default"}, {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
    {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 2.0},  # trained for max_position_embeddings
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768,
     "attention_factor": 1.5, "beta_fast": 16.0, "beta_slow": 2.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768,
     "mscale": 0.7, "mscale_all_dim": 1.0, "truncate": False},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768,
     "mscale": 0.7, "attention_factor": None, "beta_fast": None}]


@pytest.mark.parametrize("rope", CONFIGS)
@pytest.mark.parametrize("where", ["rope_scaling", "rope_parameters"])
def test_loader_builds_the_config_s_table(pkg, rope, where):
    from qwen3_omni_duplex_amd.loader import thinker_rotary

    tc = {"rope_theta": 1e6, "max_position_embeddings": 65536, where: rope}
    close(thinker_rotary(tc, 128), theirs(rope, max_position_embeddings=65536))
    axes = {"mrope_section": [24, 20, 20], "mrope_interleaved": True}
    with_axes = thinker_rotary({**tc, where: {**rope, **axes}}, 128)
    assert with_axes.axes == pkg.interleaved_axes([24, 20, 20])
    close(with_axes, theirs(rope, max_position_embeddings=65536))


@pytest.mark.parametrize("rope", [
    {"rope_type": "dynamic", "factor": 4.0}, {"rope_type": "llama3", "factor": 8.0},
    {"type": "longrope", "factor": 4.0}, {"rope_type": "linear"}, {"rope_type": "yarn"},
    {"rope_type": "yarn", "factor": 4.0}, {"rope_type": "linear", "factor": 2.0,
                                           "partial_rotary_factor": 0.5}])
def test_loader_refuses_other_tables(pkg, rope):
    """A rotation that is not built is refused, not replaced by the plain one."""
    from qwen3_omni_duplex_amd.loader import thinker_rotary

    with pytest.raises((NotImplementedError, ValueError), match="rotary"):
        thinker_rotary({"rope_theta": 1e6, "rope_scaling": rope}, 128)


@pytest.mark.parametrize("context", [{}, {"window": 64}, {"kv_dtype": torch.int8}])
def test_a_scaled_table_needs_pages(pkg, tmp_path, context):
    """The other caches' entries turn by the plain table: a config with another one is refused
    before a weight is read, a default one is not."""
    import json

    from qwen3_omni_duplex_amd import loader

    def layer(rope):
        tc = {"num_attention_heads": 8, "num_key_value_heads": 2, "hidden_size": 1024,
              "head_dim": 128, "rope_theta": 1e6, "rope_scaling": rope}
        (tmp_path / "config.json").write_text(json.dumps({"text_config": tc}))
        (tmp_path / "model.safetensors.index.json").write_text('{"weight_map": {}}')
        return loader.load_thinker_layer(loader.Checkpoint(tmp_path), 0, "cpu", **context)

    with pytest.raises(NotImplementedError, match="pages"):
        layer({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768})
    for rope in ({"rope_type": "default"}, {"type": "mrope", "mrope_section": [24, 20, 20]}, None):
        with pytest.raises(KeyError):  # the first weight
            layer(rope)


def angles(module, p):
    """The angle of each pair that the module turns tokens at p [3, T] by, modulo a turn."""
    cos, sin = module(torch.zeros(1, p.shape[1], 128), p[:, None])
    return torch.atan2(sin[0], cos[0])[:, :cos.shape[-1] // 2]


@pytest.mark.parametrize("rope", [
    {"rope_type": "default", "mrope_section": [24, 20, 20], "mrope_interleaved": True},
    {"rope_type": "default", "mrope_section": [24, 20, 20]},
    {"rope_type": "default", "mrope_section": [32, 16, 16], "mrope_interleaved": False},
    {"rope_type": "default"}, {}])
def test_axes_of_a_config(pkg, rope, monkeypatch):
    """Which position each pair turns by, found from the module's angles: with a flag or without,
    and by the default sections where there are none.  The loader's path gives these axes."""
    from qwen3_omni_duplex_amd import loader

    module = theirs(rope or {"rope_type": "default"})
    far = torch.tensor([[0], [0], [0]])
    axes = [None] * 64
    for a in range(3):
        p = far.clone()
        p[a] = 1
        for i in (angles(module, p)[0] != 0).nonzero()[:, 0].tolist():
            assert axes[i] is None
            axes[i] = a
    tc = {"num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 128, "rope_theta": 1e6,
          "rope_scaling": rope}

    class Config:
        def text_config(self):
            return tc

        def tensor(self, name):
            return torch.zeros(1)

    seen = {}
    monkeypatch.setattr(loader, "load_attention", lambda *a, **kw: {"qkv": None, "o": None})
    monkeypatch.setattr(loader, "ThinkerAttention", lambda *a, **kw: seen.update(kw))
    monkeypatch.setattr(loader, "load_moe_layer", lambda *a, **kw: None)
    monkeypatch.setattr(loader, "ThinkerDecoderLayer", lambda *a: None)
    loader.load_thinker_layer(Config(), 0, "cpu", pages=4)
    assert seen["rotary"].axes == tuple(axes)


def test_mrope_is_the_default_table(pkg):
    from qwen3_omni_duplex_amd.loader import thinker_rotary

    r = thinker_rotary({"rope_theta": 1e6, "rope_scaling": {"type": "mrope",
                                                            "mrope_section": [24, 20, 20]}}, 128)
    close(r, theirs({"rope_type": "default"}))
    assert r.axes == pkg.interleaved_axes([24, 20, 20])
