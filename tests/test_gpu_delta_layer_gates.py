"""DynamicDeltaRule and DynamicDeltaStack with their gates in float32 around 16-bit activations (bounds:
test_gpu_delta_layers.py)."""

import pytest
import torch

from helpers import gen, randn
from linattn import DynamicDeltaRule, DynamicDeltaStack
from test_gpu_delta_layers import BF, DEV, F32, _layer_ref, _stack_ref

pytestmark = pytest.mark.gpu


def _model(kind, dtype):
    torch.manual_seed(0)
    m = (DynamicDeltaRule(128, 4, 7, 4, gates=F32) if kind == "layer" else DynamicDeltaStack(128, 4, 2, 7, 4, gates=F32)).to(DEV)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith("proj_out"):
                p.normal_(0, 0.2)
            elif name.endswith("decay_bias"):
                p.normal_(0.5, 0.1)
    return m.to(dtype)


@pytest.mark.parametrize("kind,roundings", [("layer", 6), ("stack", 12)])
def test_training(kind, roundings):
    m = _model(kind, BF)
    x = randn(gen(1), 2, 150, 128).to(BF)
    leaf = x.to(DEV).requires_grad_()
    out = m(leaf)
    ref = _layer_ref(m, x.double())[0] if kind == "layer" else _stack_ref(m, x.double())
    assert out.dtype == BF and (out.detach().double().cpu() - ref).norm() <= roundings * 2.0**-8 * ref.norm()
    out.backward(randn(gen(2), *out.shape).to(DEV).to(BF))
    for name, p in [("x", leaf), *m.named_parameters()]:
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name


@pytest.mark.parametrize("kind", ["layer", "stack"])
def test_the_rule_is_given_float32_gates(kind, monkeypatch):
    from dynconv import modules

    seen = []

    def note(f):
        def call(q, k, v, log_decay, beta, *args, **kw):
            seen.append((q.dtype, log_decay.dtype, beta.dtype))
            return f(q, k, v, log_decay, beta, *args, **kw)
        return call

    for name in ("gated_delta_rule", "gated_delta_rule_step"):
        monkeypatch.setattr(modules, name, note(getattr(modules, name)))
    m = _model(kind, BF)
    x = randn(gen(3), 2, 5, 128).to(DEV).to(BF)
    with torch.no_grad():
        out, state = m(x[:, :4], return_state=True)
        last = m.step(x[:, 4], state)
        whole = m(x)
    assert set(seen) == {(BF, F32, F32)}
    # the same tokens whole and one by one, each way rounded as the reference's bounds count
    n = 6 if kind == "layer" else 12
    assert (torch.cat([out, last[:, None]], 1) - whole).double().norm() <= 2 * n * 2.0**-8 * whole.double().norm()
