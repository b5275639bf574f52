"""The axes of a multimodal rotary embedding against transformers' own module (the installed
transformers, fp32 on the CPU), and the loader's reading of a config."""
from __future__ import annotations

import pytest
import torch

from tests.test_thinker_ref import _module

pytest.importorskip("transformers.models.qwen3_omni_moe.modeling_qwen3_omni_moe")


def test_axes_match_transformers(pkg):
    """Positions that differ along the three axes: each pair's angle is its axis' position times
    its frequency."""
    *_, rot = _module(hd=16, nh=2, nkv=1, hidden=128)
    axes = pkg.interleaved_axes([3, 3, 2])
    f = pkg.rope_inv_freq(16, 1e6)
    assert len(axes) == 8 and torch.equal(f, rot.inv_freq)
    p = torch.tensor([[5, 9, 100, 0], [40, 2, 77, 3], [1, 8, 3000, 11]])
    cos, sin = rot(torch.zeros(1, 4, 128), p[:, None])
    a = torch.stack([p[axis] for axis in axes], -1).float() * f
    a = torch.cat([a, a], -1)
    torch.testing.assert_close(cos[0], a.cos(), rtol=0, atol=1e-6)
    torch.testing.assert_close(sin[0], a.sin(), rtol=0, atol=1e-6)


def test_axes_of_the_thinker(pkg):
    axes = pkg.interleaved_axes([24, 20, 20])
    assert len(axes) == 64 and [axes.count(a) for a in (0, 1, 2)] == [24, 20, 20]
    assert axes[:6] == (0, 1, 2, 0, 1, 2) and axes[60:] == (0, 0, 0, 0)
    assert pkg.interleaved_axes([4]) == (0, 0, 0, 0)


def test_loader_reads_the_rotary_embedding(pkg):
    from qwen3_omni_duplex_amd.loader import thinker_rotary

    tc = {"rope_theta": 1e6, "rope_scaling": {"mrope_section": [24, 20, 20],
                                              "mrope_interleaved": True}}
    r = thinker_rotary(tc, 128)
    assert r.axes == pkg.interleaved_axes([24, 20, 20]) and r.layout == "half"
    assert torch.equal(r.inv_freq, pkg.rope_inv_freq(128, 1e6))
    assert thinker_rotary({"rope_theta": 1e4}, 128).axes is None
    assert thinker_rotary({"rope_theta": 1e4, "rope_scaling": {"mrope_section": [2, 1, 1]}},
                          128).axes is None
