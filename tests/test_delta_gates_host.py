"""The type in which DynamicDeltaRule passes its gates on, without a GPU."""

import pytest
import torch

from linattn import DynamicDeltaRule, DynamicDeltaStack

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF])
def test_float32_gates_keep_their_bits(dtype):
    torch.manual_seed(0)
    layer = DynamicDeltaRule(64, 4, 7, 4, gates=F32).to(dtype)
    x = torch.randn(2, 50, 64).to(dtype)
    lam, beta = (t.detach() for t in layer._gates(x))
    assert lam.dtype == beta.dtype == F32 and lam.shape == beta.shape == (2, 50, 4)
    # from the projections as they are: exp, softplus, sigmoid and two products in float32, each within 4 units of 2^-23
    u, w = layer.c_decay(x).double() + layer.decay_bias.double(), layer.c_beta(x).double()
    want = -torch.exp(layer.log_rate.double()) * torch.log1p(torch.exp(u)), 1 / (1 + torch.exp(-w))
    for a, b in zip((lam, beta), want):
        assert ((a.double() - b).abs() <= 20 * 2.0**-23 * b.abs()).all()
    layer.gates = None
    assert all(torch.equal(a, b.to(dtype)) for a, b in zip(layer._gates(x), (lam, beta)))


def test_types_are_checked():
    for bad in (BF, HF, torch.float64):
        with pytest.raises(ValueError):
            DynamicDeltaRule(64, 4, 7, 4, gates=bad)
    stack = DynamicDeltaStack(64, 4, 2, 7, 4, gates=F32)
    assert all(layer.gates == F32 for layer in stack.layers)
    assert list(stack.state_dict()) == list(DynamicDeltaStack(64, 4, 2, 7, 4).state_dict())
