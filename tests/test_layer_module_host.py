"""DynamicLinearAttention's parameters, decays and states under the usual set-ups, without a GPU."""

import copy

import pytest
import torch

from linattn import DynamicLinearAttention


@pytest.fixture
def bf16_default():
    torch.set_default_dtype(torch.bfloat16)
    yield
    torch.set_default_dtype(torch.float32)


def test_states_are_float32_under_another_default_dtype(bf16_default):
    m = DynamicLinearAttention(64, 2, 7, 4)
    state = m.new_state(3)
    assert state.attn.dtype == torch.float32 and m.log_decay.dtype == torch.float32
    assert state.conv.dtype == m.c_attn.weight.dtype == torch.bfloat16
