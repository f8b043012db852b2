"""gated_delta_rule's dbeta at tokens whose beta is zero or next to it, under gradients of a loss that is a mean over many
tokens (bounds: test_gpu_delta_rule.py, here over those tokens alone)."""

import pytest
import torch

from linattn import gated_delta_rule
from oracle.layer import gated_delta_rule_chunked
from test_gpu_delta_rule import BF, DEV, F32, HF, NAMES, UO, _compare, _inputs, _rounding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [(2, 1, 2, 100, 64, 48), (1, 2, 2, 130, 128, 128), (9, 16, 16, 20, 128, 128), (1, 1, 1, 40, 100, 20)])
@pytest.mark.parametrize("small", [0.0, 2.0**-45])
@pytest.mark.parametrize("dtype,gdtype", [(BF, BF), (BF, F32), (HF, F32), (F32, F32)])
def test_dbeta(size, small, dtype, gdtype):
    B, Hk, H, T, K, V = size
    print(f"[delta small beta] {size} {dtype} {gdtype} beta {small}", flush=True)
    (q, k, v, lam, beta, do), S0, _ = _inputs(*size, dtype, gdtype, True, 13)
    few = torch.rand(B, H, T, generator=torch.Generator().manual_seed(T)) < 0.2
    few[..., 0] = few[..., -1] = True
    beta = torch.where(few, torch.full_like(beta, small), beta)
    do = (do.float() * 2.0**-25 if dtype != HF else do.float() * 2.0**-10).to(dtype)
    args = (q, k, v, lam, beta, K**-0.5, do, S0, None, None, True)
    exact = gated_delta_rule_chunked(*args)[1][4]
    r, u_r = _rounding(dtype, gdtype == F32)
    rounded = gated_delta_rule_chunked(*args, dtype=F32, r=r)[1][4]
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam, beta)]
    out = gated_delta_rule(*leaves, initial_state=S0.to(DEV), normalize=True)
    got = torch.autograd.grad(out, leaves, do.to(DEV))[4]
    rest = [None] * 6
    _compare([*rest, got.cpu()[few], None], [*rest, exact[few], None], [*rest, rounded[few], None], dict.fromkeys(NAMES, gdtype), u_r)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_token_is_written(dtype):
    """beta of zero throughout: the state only decays, and o reads it."""
    (q, k, v, lam, beta, _), S0, _ = _inputs(2, 2, 2, 100, 64, 64, dtype, F32, True, 14)
    lam = lam.clamp(min=-0.05)
    args = [t.to(DEV) for t in (q, k, v, lam, torch.zeros_like(beta))]
    o, S = gated_delta_rule(*args, initial_state=S0.to(DEV), return_state=True, normalize=True)
    G = torch.exp(lam.double().cumsum(-1))
    unit = lambda t: t.double() / torch.sqrt((t.double()**2).sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    eo, eS = 64**-0.5 * G[..., None] * (unit(q) @ S0.double()), G[..., -1][..., None, None] * S0.double()
    # two chunks of 64 or four of 32, each a factor and a product of the state in float32 or as good: 2^-20
    assert (o.double().cpu() - eo).norm() <= (UO[dtype] + 2.0**-20) * eo.norm()
    assert (S.double().cpu() - eS).norm() <= 2.0**-20 * eS.norm()
