"""The float64 restatements of the gated delta rule and the residual norm (oracle/layer.py): hand-computed values, the chunked
formulas against the recurrence and its autograd gradients, and gradients against differences."""

import pytest
import torch

from oracle.layer import gated_delta_rule_chunked, gated_delta_rule_ref, linear_attention_ref, residual_norm_ref

F64 = torch.float64


def _inputs(B, Hk, H, T, K, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    lam = -torch.rand(B, H, T, generator=g, dtype=F64)
    return n(B, Hk, T, K), n(B, Hk, T, K), n(B, H, T, V), lam, torch.rand(B, H, T, generator=g, dtype=F64), n(B, H, K, V)


def test_by_hand():
    one = torch.ones(1, 1, 2, 1, dtype=F64)
    half = torch.full((1, 1, 2), 0.5, dtype=F64)
    # S_0 = 1/2 (v = 1), then S' = S/2 = 1/4, u = (1 - 1/4) / 2 = 3/8, S_1 = 5/8
    o, S = gated_delta_rule_ref(one, one, one, torch.log(half), half, 2.0)
    assert torch.allclose(o.flatten(), torch.tensor([1.0, 1.25], dtype=F64)) and abs(S.item() - 0.625) < 1e-15


def test_a_full_correction_stores_the_value():
    q, k, v, _, _, S0 = _inputs(1, 2, 2, 5, 4, 3)
    k = k / k.norm(dim=-1, keepdim=True)
    zero = torch.zeros(1, 2, 5, dtype=F64)
    o, _ = gated_delta_rule_ref(k, k, v, zero, zero + 1, 1.0, S0)
    assert torch.allclose(o, v)  # read back with its own key


def test_orthogonal_keys_are_linear_attention():
    q, _, v, _, _, _ = _inputs(1, 1, 1, 6, 6, 3)
    k = torch.eye(6, dtype=F64)[None, None]
    lam = torch.tensor([-0.3], dtype=F64)
    o, S = gated_delta_rule_ref(q, k, v, lam[:, None, None].expand(1, 1, 6), torch.ones(1, 1, 6, dtype=F64), 0.5)
    ro, rS = linear_attention_ref(q, k, v, lam, 0.5)
    assert torch.allclose(o, ro) and torch.allclose(S, rS)


@pytest.mark.parametrize("B,Hk,H,T,K,V,lens,normalize", [
    (2, 1, 1, 9, 4, 3, None, False), (2, 2, 4, 21, 5, 6, [21, 13], True), (3, 1, 2, 16, 3, 4, [0, 1, 16], True)])
def test_chunks_are_the_recurrence(B, Hk, H, T, K, V, lens, normalize):
    q, k, v, lam, beta, S0 = _inputs(B, Hk, H, T, K, V, seed=T)
    beta[0, 0, 0] = 0.0
    if T > 5:
        lam[-1, -1, 4] = -float("inf")
    if not normalize:
        k = k / k.norm(dim=-1, keepdim=True)
    do, dS = torch.randn(B, H, T, V, dtype=F64), torch.randn(B, H, K, V, dtype=F64)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, lam, beta, S0)]
    out = gated_delta_rule_ref(*leaves[:5], 0.7, leaves[5], lens, normalize)
    grads = torch.autograd.grad(out, leaves, (do, dS))
    got, dgot = gated_delta_rule_chunked(q, k, v, lam, beta, 0.7, do, S0, dS, lens, normalize, chunk=8)
    for a, b in zip((*got, *dgot), (*out, *grads)):
        # a decay of minus infinity has a gradient of 0 in the formula and in its limit, 0 * inf in autograd's exp
        b = torch.nan_to_num(b.detach(), nan=0.0)
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-10)


def test_gradients_against_differences():
    q, k, v, lam, beta, S0 = _inputs(1, 1, 2, 4, 3, 2, seed=3)
    f = lambda *t: gated_delta_rule_ref(*t[:5], 0.7, t[5], None, True)  # noqa: E731
    assert torch.autograd.gradcheck(f, [t.requires_grad_() for t in (q, k, v, lam, beta, S0)])


def test_residual_norm_by_hand():
    x, b = torch.tensor([[3.0, 1.0]], dtype=F64), torch.tensor([[3.0, 4.0]], dtype=F64)
    y, h = residual_norm_ref(x, b, scale=2.0, eps=0.0)
    rms = (12.5) ** 0.5
    assert torch.allclose(h, torch.tensor([[3 + 6 / rms, 1 + 8 / rms]], dtype=F64))
    assert torch.allclose((y * y).mean(), torch.ones((), dtype=F64))
    y1, h1 = residual_norm_ref(x, b, gate=torch.zeros_like(b), activation="sigmoid", eps=0.0)
    assert torch.allclose(h1, x + b / rms / 2)
    assert torch.allclose(residual_norm_ref(x, b, gate=torch.zeros_like(b), activation="silu")[1], x)


def test_residual_norm_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    ts = [torch.randn(*s, generator=g, dtype=F64).requires_grad_() for s in ((2, 5), (2, 5), (5,), (5,), (2, 5), (5,))]
    for act in ("silu", "sigmoid", None):
        assert torch.autograd.gradcheck(lambda *t: residual_norm_ref(*t[:5], act, t[5]), ts)
