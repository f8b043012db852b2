"""gated_delta_rule in bf16 training without float32 results is as good as its results' own rounding.

Bounds.  e is the error of the exact result rounded once to bf16, ||round(b) - b||.  Before that rounding the kernels' operands
are off by 2^-16 of themselves where they are two bf16 parts (T, P, X, Z, Y, the pairs' gradients), by up to 2^-12 (a half of 11
bits) where they come through memory (S, dS, Z), a sixteenth of a rounding to bf16, and by a rounding to bf16 in dX, which is dv.
An operand's errors are independent, and a sum over it takes them on as it does its values: a result is off by about the operand's
share of itself.

  o, dv     16-bit operands alone: e and 2^-14 of the result
  dq        S, Z and what comes of them: 3 (e / 16) with a factor of 2 for terms that cancel, e sqrt(1 + (6/16)^2) < 1.1 e
  dk, dlog  the same and dX in one of two or more terms, about half of e: e sqrt(1 + (6/16)^2 + 1/4) < 1.25 e
  dbeta     the same with dX in one of three terms of k.W, up to 0.7 of e: e sqrt(1 + (6/16)^2 + 1/2) < 1.3 e (a product with dX
            itself would take its rounding in full, 1.5 e)
"""

import pytest
import torch

from helpers import gen, randn
from linattn import gated_delta_rule
from oracle.layer import gated_delta_rule_chunked

pytestmark = pytest.mark.gpu

DEV, BF = "cuda", torch.bfloat16
FACTORS = dict(o=1.0, dq=1.1, dk=1.25, dv=1.0, dlog_decay=1.25, dbeta=1.3)


def _inputs(B, Hk, H, T, K, V):
    g = gen(T + K)
    q, k = (randn(g, B, Hk, T, K) + 0.5 * randn(g, Hk, 1, K) for _ in range(2))
    lam = -torch.log1p(torch.exp(randn(g, B, H, T))) * torch.exp2(-9 * torch.rand(1, H, 1, generator=g))
    beta = torch.sigmoid(randn(g, B, H, T))
    return [t.to(BF) for t in (q, k, randn(g, B, H, T, V), lam, beta, randn(g, B, H, T, V))]


def _run(q, k, v, lam, beta, do):
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam, beta)]
    o = gated_delta_rule(*leaves, normalize=True)
    got = [o.detach(), *torch.autograd.grad(o, leaves, do.to(DEV))]
    (eo, _), eg = gated_delta_rule_chunked(q, k, v, lam, beta, q.shape[-1]**-0.5, do, None, None, None, True)
    return dict(zip(FACTORS, zip((t.double().cpu() for t in got), (eo, *eg))))


@pytest.mark.parametrize("size", [(1, 2, 2, 1024, 128, 128), (2, 1, 2, 700, 64, 96), (1, 1, 2, 500, 256, 256), (4, 16, 16, 100, 128, 64),
                                  (1, 2, 2, 600, 100, 72)])
def test_one_rounding(size):
    for name, (a, b) in _run(*_inputs(*size)).items():
        e = (b.to(BF).double() - b).norm()
        print(f"  {size} {name}: {((a - b).norm() / e).item():.3f} roundings", flush=True)
        assert (a - b).norm() <= FACTORS[name] * e + 2.0**-14 * b.norm(), name


def test_columns_of_any_size():
    """Columns of v from 2^-40 to 2^40, with gradients the other way round: states' columns and their gradients' too."""
    q, k, v, lam, beta, do = _inputs(1, 2, 2, 400, 128, 128)
    by = torch.exp2(torch.linspace(-40, 40, 128).round())
    for name, (a, b) in _run(q, k, (v.float() * by).to(BF), lam, beta, (do.float() / by).to(BF)).items():
        if name in ("o", "dv"):
            s = by.double() if name == "o" else 1 / by.double()
            a, b = a / s, b / s
            e = (b.to(BF).double() - b).flatten(0, -2).norm(dim=0)
            assert ((a - b).flatten(0, -2).norm(dim=0) <= e + 2.0**-14 * b.flatten(0, -2).norm(dim=0)).all(), name
        else:
            e = (b.to(BF).double() - b).norm()
            assert (a - b).norm() <= FACTORS[name] * e + 2.0**-14 * b.norm(), name


@pytest.mark.parametrize("flags", [1, 5])
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_the_backward_leaves_the_forwards_workspace_alone(flags, dtype):
    """Kept states or not, in segments or whole: a backward can be called again, on another stream too."""
    from dynconv.delta import _GatedDeltaRuleFn as Fn
    from test_gpu_rule_states import _Ctx

    for size in ((1, 2, 2, 700, 128, 128), (9, 16, 16, 70, 64, 64)):
        q, k, v, lam, beta, do = (t.to(dtype).to(DEV) for t in _inputs(*size))
        ctx = _Ctx(*[True] * 6)
        Fn.forward(ctx, q, k, v, lam, beta, None, None, size[4]**-0.5, 1e-6, flags, False)
        before = ctx.saved_tensors[-1].clone()
        first = Fn.backward(ctx, do)[:5]
        assert torch.equal(ctx.saved_tensors[-1], before)
        assert all(torch.equal(a, b) for a, b in zip(first, Fn.backward(ctx, do)))
