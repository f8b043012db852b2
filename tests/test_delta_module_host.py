"""DynamicDeltaRule's and DynamicDeltaStack's parameters and states, and what DynamicLinearAttention keeps, without a GPU."""

import pytest
import torch

from linattn import DynamicDeltaRule, DynamicDeltaStack, DynamicLinearAttention


def test_sizes_are_checked():
    for cls in (DynamicDeltaRule, DynamicLinearAttention):
        with pytest.raises(ValueError):
            cls(100, 3, 7, 4)
        with pytest.raises(ValueError):
            cls(128, 4, 6, 4)  # R + 1 is no power of two
        with pytest.raises(ValueError):
            cls(1024, 2, 7, 4)  # 512 channels a head


def test_parameters_and_states():
    m = DynamicDeltaStack(64, 2, 3, 7, 4).to(torch.bfloat16)
    states = m.new_state(5)
    assert len(states) == 3 and all(s.attn.shape == (5, 2, 32, 32) and s.attn.dtype == torch.float32 for s in states)
    assert all(s.conv.shape == (5, 3, 192) and s.conv.dtype == torch.bfloat16 for s in states)
    layer = m.layers[0]
    lam, beta = layer._gates(torch.zeros(2, 3, 64, dtype=torch.bfloat16))
    assert lam.shape == beta.shape == (2, 3, 2) and lam.dtype == torch.bfloat16
    assert (lam < 0).all() and (beta == 0.5).all()


def test_linear_attentions_parameters_are_as_they_were():
    torch.manual_seed(0)
    m = DynamicLinearAttention(64, 2, 7, 4)
    assert list(m.state_dict()) == ["norm_weight", "norm_bias", "c_attn.weight", "conv.proj_out", "conv.proj_out_bias",
                                    "conv.proj_in.weight", "c_gate.weight", "c_proj.weight"]
