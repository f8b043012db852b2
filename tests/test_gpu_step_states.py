"""What the single-token operators do to their states as autograd sees it, through the native binding and without it."""

import pytest
import torch

from helpers import gen, randn
from linattn import DynamicLinearAttention, linear_attention, linear_attention_step
from lowrank import lowrank_dynamic_convolution_step

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    from dynconv import _capi

    _capi.load()
    if request.param == "python":
        monkeypatch.setattr(_capi, "binding", None)
    elif _capi.binding is None:
        pytest.skip("no native binding")


def _attention(g, B=2, H=3, T=40, K=32):
    q, k, v = (randn(g, B, H, T, K).to(DEV) for _ in range(3))
    return q, k, v, torch.full((H,), -0.1, device=DEV), randn(g, B, H, K, K).to(DEV)


def _conv(g, N=3, D=64, R=8, W=4):
    return (randn(g, N, D).to(DEV), randn(g, N, R).to(DEV), randn(g, R, W * D).to(DEV),
            randn(g, N, W - 1, D).to(DEV))


def test_a_step_makes_the_backward_of_what_saved_its_state_raise(path):
    """As torch's own in-place operations do: a gradient of the old state from the new one's values would be wrong."""
    q, k, v, lam, S = _attention(gen(1))
    q.requires_grad_()
    o = linear_attention(q, k, v, lam, initial_state=S)
    with torch.no_grad():
        linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lam, S)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    x, z, U, state = _conv(gen(2))
    w = torch.ones_like(state, requires_grad=True)
    y = (state * w).sum()
    lowrank_dynamic_convolution_step(x, z, U, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_layer_that_steps_on_before_its_backward_raises(path):
    torch.manual_seed(0)
    m = DynamicLinearAttention(64, 2, 7, 4).to(DEV)
    x = randn(gen(3), 2, 9, 64).to(DEV)
    with torch.no_grad():
        _, state = m(x, return_state=True)
    out = m(x, state)
    m.step(x[:, 0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_states_of_inference_mode_are_taken(path):
    q, k, v, lam, _ = _attention(gen(4))
    x, z, U, _ = _conv(gen(5))
    with torch.inference_mode():
        S, state = torch.zeros(2, 3, 32, 32, device=DEV), torch.zeros(3, 3, 64, device=DEV)
        inside = linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lam, S)
        lowrank_dynamic_convolution_step(x, z, U, state)
    with torch.no_grad():  # and outside of it, which torch's in-place operations refuse
        S2 = torch.zeros(2, 3, 32, 32, device=DEV)
        assert torch.equal(linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lam, S2), inside)
        assert torch.equal(S, S2)
        linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lam, S)
        lowrank_dynamic_convolution_step(x, z, U, state)


def test_a_forward_mode_tangent_is_refused(path):
    """The steps have none: taken for a plain tensor, a dual tensor would lose it."""
    fw = torch.autograd.forward_ad
    q, k, v, lam, S = _attention(gen(6))
    args = [q[:, :, 0], k[:, :, 0], v[:, :, 0], lam, S]
    before = S.clone()
    x, z, U, state = _conv(gen(7))
    conv, past = [x, z, U, state], state.clone()
    with torch.no_grad(), fw.dual_level():
        for i in range(5):
            dual = [fw.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
            with pytest.raises(AssertionError):
                linear_attention_step(*dual)
        for i in range(4):
            dual = [fw.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(conv)]
            with pytest.raises(AssertionError):
                lowrank_dynamic_convolution_step(*dual)
        assert torch.equal(S, before) and torch.equal(state, past)
        linear_attention_step(*args)
        lowrank_dynamic_convolution_step(*conv)
    with torch.no_grad(), pytest.raises((AssertionError, RuntimeError)):
        torch.func.jvp(lambda t: linear_attention_step(t, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
