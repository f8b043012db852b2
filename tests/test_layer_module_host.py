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


def test_decays_of_a_layer_built_on_meta():
    """to_empty gives every buffer the memory's old contents; the decays are no state of a checkpoint."""
    want = DynamicLinearAttention(96, 3, 7, 4)
    with torch.device("meta"):
        m = DynamicLinearAttention(96, 3, 7, 4)
    assert m.log_decay.is_meta
    big = torch.full((4096,), 3.7e37)  # so that fresh memory is not zero by chance
    del big
    m = m.to_empty(device="cpu")
    m.load_state_dict(want.state_dict())
    assert torch.equal(m.log_decay, want.log_decay) and "log_decay" not in m.state_dict()
    half = m.to(torch.bfloat16)
    assert half.log_decay.dtype == torch.float32 and torch.equal(half.log_decay, want.log_decay)


def test_decays_follow_the_module():
    m = DynamicLinearAttention(96, 3, 7, 4)
    want = m.log_decay.clone()
    for move in (lambda t: t.half(), lambda t: t.double(), lambda t: t.float(), lambda t: copy.deepcopy(t),
                 lambda t: t.to(torch.bfloat16)):
        m = move(m)
        assert m.log_decay.dtype == torch.float32 and torch.equal(m.log_decay, want)
    assert m.to("meta").log_decay.is_meta


def test_head_dims_past_the_operator_are_refused_when_built():
    with pytest.raises(ValueError):
        DynamicLinearAttention(1024, 2, 7, 4)  # 512 channels a head
    assert DynamicLinearAttention(512, 2, 7, 4).head_dim == 256
