"""Module plumbing of the selective state space layer and of the residual block, without a GPU."""

from __future__ import annotations

import pytest
import torch

from spear_b200.nn.block import MixerBlock
from spear_b200.nn.phalanx import Phalanx
from spear_b200.nn.ssm import SelectiveSSM


def test_construction_and_state_dict(tmp_path):
    torch.manual_seed(1)
    a = SelectiveSSM(dim=40, state_size=8, width=3, dtype=torch.bfloat16)
    assert (a.inner, a.rank) == (80, 3)
    assert sorted(a.state_dict()) == ["A_log", "D", "conv_bias", "conv_weight", "dt_bias", "dt_proj.weight", "in_proj.weight",
                                      "out_proj.weight", "x_proj.weight"]
    assert a.A_log.dtype == a.D.dtype == a.dt_bias.dtype == torch.float32 and a.conv_weight.dtype == torch.bfloat16
    size = torch.nn.functional.softplus(a.dt_bias)
    assert (size > 0.9e-3).all() and (size < 1.1e-1).all()
    torch.save(a.state_dict(), tmp_path / "a.pt")
    b = SelectiveSSM(dim=40, state_size=8, width=3, dtype=torch.bfloat16)
    b.load_state_dict(torch.load(tmp_path / "a.pt"))
    assert all(torch.equal(u, v) for u, v in zip(a.state_dict().values(), b.state_dict().values()))
    s = a.empty_state(2)
    assert s.conv.shape == (2, 2, 80) and s.ssm.shape == (2, 80, 8) and s.ssm.dtype == torch.float32
    c = s.clone_detached()
    assert c.ssm.data_ptr() != s.ssm.data_ptr()


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=8, expand=0), dict(dim=8, state_size=0), dict(dim=8, state_size=65),
                                dict(dim=8, width=1), dict(dim=8, width=5), dict(dim=8, dt_min=0.0), dict(dim=8, dt_min=1.0, dt_max=0.1)])
def test_refused_arguments(kw):
    with pytest.raises(ValueError):
        SelectiveSSM(**kw)


def test_needs_a_gpu_and_checks_shapes():
    layer = SelectiveSSM(dim=16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer(torch.randn(1, 4, 16))
    for bad in (torch.randn(4, 16), torch.randn(1, 4, 17)):
        with pytest.raises(ValueError, match="SelectiveSSM takes"):
            layer(bad)
    with pytest.raises(ValueError, match="step takes"):
        layer.step(torch.randn(1, 1, 16), layer.empty_state(1))
    block = MixerBlock(Phalanx(dim=64, length=32, dtype=torch.bfloat16), 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        block(torch.randn(1, 32, 64))
    with pytest.raises(ValueError, match="MixerBlock takes"):
        block(torch.randn(1, 32, 65))


def test_public_names():
    import spear_b200
    from spear_b200 import ops

    assert spear_b200.SelectiveSSM is SelectiveSSM and spear_b200.MixerBlock is MixerBlock
    for name in ("rms_norm", "rms_norm_8bit", "causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step"):
        assert callable(getattr(ops, name))


@pytest.mark.parametrize("built,cast", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float16)])
def test_a_cast_layer_works_in_its_new_type(built, cast):
    layer = SelectiveSSM(dim=16, dtype=built).to(cast)
    assert layer.dtype == cast and layer.empty_state(2).conv.dtype == cast and layer.empty_state(2).ssm.dtype == torch.float32
    for given in (built, cast):  # past the projections, up to the first operator
        with pytest.raises(RuntimeError, match="no CPU path"):
            layer(torch.randn(1, 4, 16, dtype=given))
        with pytest.raises(RuntimeError, match="no CPU path"):
            layer.step(torch.randn(1, 16, dtype=given), layer.empty_state(1))


def test_a_mixer_that_cannot_stream_is_named_before_anything_runs():
    block = MixerBlock(Phalanx(dim=64, length=32, dtype=torch.bfloat16), 64)
    with pytest.raises(TypeError, match="Phalanx has no prefill"):
        block.prefill(torch.randn(1, 32, 64))
    with pytest.raises(TypeError, match="Phalanx has no step"):
        block.step(torch.randn(1, 64), None, None)
