"""The restatements of the gated delta rule (oracle/layer.py) with normed rows and an eps of zero or close to it: rows that are
no tokens, behind a partial chunk or past a length, have no norm to divide by."""

import pytest
import torch

from oracle.layer import gated_delta_rule_chunked, gated_delta_rule_ref
from test_oracle_delta import F64, _inputs


@pytest.mark.parametrize("eps", [0.0, 1e-12])
@pytest.mark.parametrize("T,lens", [(1, None), (7, None), (9, [9, 4]), (16, [0, 11])])
def test_chunks_are_the_recurrence(T, lens, eps):
    B = 1 if lens is None else 2
    q, k, v, lam, beta, S0 = _inputs(B, 1, 2, T, 4, 3, seed=T)
    do, dS = torch.randn(B, 2, T, 3, dtype=F64), torch.randn(B, 2, 4, 3, dtype=F64)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, lam, beta, S0)]
    out = gated_delta_rule_ref(*leaves[:5], 0.7, leaves[5], lens, True, eps)
    grads = torch.autograd.grad(out, leaves, (do, dS))
    got, dgot = gated_delta_rule_chunked(q, k, v, lam, beta, 0.7, do, S0, dS, lens, True, eps, chunk=8)
    for a, b in zip((*got, *dgot), (*out, *grads)):
        assert torch.isfinite(b).all()
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-10)
