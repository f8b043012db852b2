"""What linear_attention keeps for its backward, through the native binding and without it."""

import pytest
import torch

from helpers import gen, randn
from linattn import linear_attention

pytestmark = pytest.mark.gpu

DEV = "cuda"
B, H, T, K = 1, 2, 3000, 64


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    from dynconv import _capi

    _capi.load()
    if request.param == "python":
        monkeypatch.setattr(_capi, "binding", None)
    elif _capi.binding is None:
        pytest.skip("no native binding")


def _leaves(seed):
    g = gen(seed)
    return [randn(g, B, H, T, K).to(torch.bfloat16).to(DEV).requires_grad_() for _ in range(3)]


def _states_bytes():
    from dynconv import _capi

    n = _capi.load().dc_linear_attention_ws_bytes(B, H, T, K, K, _capi.dtype_code(torch.bfloat16), 0)
    assert n > 0, "several segments"
    return n


def test_the_segments_states_go_with_the_saved_tensors(path):
    """Freed by the backward, though the output and its node live on."""
    leaves = _leaves(1)
    lam = torch.full((H,), -0.01, device=DEV)
    o = linear_attention(*leaves, lam)
    do = torch.ones_like(o)
    torch.autograd.grad(o, leaves, do, retain_graph=True)
    held = torch.cuda.memory_allocated()
    torch.autograd.grad(o, leaves, do)
    assert o.grad_fn is not None and held - torch.cuda.memory_allocated() >= _states_bytes()
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(o, leaves, do)


def test_saved_tensor_hooks_see_them(path):
    leaves = _leaves(2)
    lam = torch.full((H,), -0.01, device=DEV)
    do = randn(gen(3), B, H, T, K).to(torch.bfloat16).to(DEV)
    want = torch.autograd.grad(linear_attention(*leaves, lam), leaves, do)
    sizes = []

    def pack(t):
        sizes.append(t.numel() * t.element_size())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
        o = linear_attention(*leaves, lam)
    assert _states_bytes() in sizes
    for a, b in zip(torch.autograd.grad(o, leaves, do), want):
        assert torch.equal(a, b)
