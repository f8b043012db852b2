"""DynamicDeltaStack's norms are the framework's own, the first one too (bounds: test_gpu_residual_norm.py)."""

import pytest
import torch

from helpers import gen, randn
from linattn import DynamicDeltaStack
from oracle.layer import residual_norm_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def no_library_norm(monkeypatch):
    def refuse(*args, **kw):
        raise AssertionError("a library's norm")

    for owner in (torch.nn.functional, torch):
        monkeypatch.setattr(owner, "rms_norm", refuse)


@pytest.mark.parametrize("dtype,stream", [(F32, None), (BF, None), (BF, F32)])
def test_training_and_steps(dtype, stream, no_library_norm):
    torch.manual_seed(0)
    m = DynamicDeltaStack(128, 4, 2, 7, 4, stream=stream).to(DEV).to(dtype)
    x = randn(gen(1), 2, 9, 128).to(DEV).to(dtype).requires_grad_()
    y = m(x)
    y.sum().backward()
    assert torch.isfinite(x.grad).all() and m.weight.grad[0].abs().max() > 0
    with torch.no_grad():
        assert torch.isfinite(m.step(x[:, 0].detach(), m.new_state(2))).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("strided", [False, True])
def test_the_first_norm(dtype, strided, no_library_norm):
    """A stack of no layers is its first norm: y and the gradients of x and the weight against float64."""
    m = DynamicDeltaStack(96, 4, 0, 7, 4, stream=F32).to(DEV).to(dtype)
    with torch.no_grad():
        m.weight.copy_(1 + 0.1 * randn(gen(2), 1, 96))
    x, dy = randn(gen(3), 3, 7, 96, scale=3.0).to(dtype), randn(gen(4), 3, 7, 96).to(dtype)
    leaf = x.to(DEV)
    if strided:
        leaf = torch.cat([leaf, leaf], -1)[..., :96]
    leaf = leaf.detach().requires_grad_()
    y = m(leaf)
    dx, dw = torch.autograd.grad(y, (leaf, m.weight), dy.to(DEV))
    r, w = x.double().requires_grad_(), m.weight.detach().double().cpu()[0].requires_grad_()
    want = residual_norm_ref(r, r.detach(), w, scale=0.0, eps=m.eps)[0]
    rx, rw = torch.autograd.grad(want, (r, w), dy.double())
    # float32 sums of 96 or 21 terms, a row's factor, and the results' rounding (dx: of the stream's part and of its sum with 0)
    u = 2.0**-8 if dtype == BF else 2.0**-24
    for a, b in ((y.detach(), want.detach()), (dx, rx), (dw[0], rw)):
        assert a.dtype == dtype and (a.double().cpu() - b).norm() <= (2 * u + 2.0**-18) * b.norm()
