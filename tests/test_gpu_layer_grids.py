"""Calls whose workgroups pass what one launch counts (2^32 work-items along an axis): taken in several launches."""

import pytest
import torch

from helpers import gen
from linattn import group_norm, linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def _free(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of GPU memory")


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def test_a_step_of_many_heads():
    """2^24 + 2^9 heads of one channel: one workgroup of 256 threads each."""
    _free(8)
    B, H = (1 << 15) + 1, 1 << 9
    print(f"[grids] step B{B} H{H}", flush=True)
    q, k, v, S = (_randn(i, B, H, 1) for i in range(4))
    lam = -torch.rand(H, generator=gen(0)).to(DEV)
    state = S[..., None].clone()
    with torch.no_grad():
        o = linear_attention_step(q, k, v, lam, state, scale=0.5)
    want = torch.exp(lam)[:, None] * S + k * v
    torch.testing.assert_close(state[..., 0], want, rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(o, 0.5 * q * want, rtol=1e-6, atol=1e-6)


def test_whole_sequences_of_many_heads():
    """Three passes of 12.6 million workgroups of 128 threads in the backward, and one token each."""
    _free(16)
    B, H = 12300, 1 << 10
    print(f"[grids] sequences B{B} H{H}", flush=True)
    q, k, v, do = (_randn(i, B, H, 1, 1).to(BF) for i in range(4))
    lam = torch.zeros(H, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = linear_attention(*leaves, lam, scale=1.0)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    q, k, v, do = (t.detach().float() for t in (q, k, v, do))
    # a score is rounded to bf16, and the output: 2^-7 of a product of three factors
    for got, want in ((o, q * k * v), (dq, do * v * k), (dk, do * v * q), (dv, q * k * do)):
        assert ((got.detach().float() - want).abs() <= 2.0**-7 * want.abs() + 1e-30).all()


def test_a_norm_of_many_groups():
    """2^30 + 128 channels in groups of two: 64 channels to a wavefront."""
    _free(32)
    D = (1 << 30) + 128
    print(f"[grids] norm D{D}", flush=True)
    x = _randn(5, 1, D).to(BF)
    y = group_norm(x, D // 2, activation=None, eps=1e-5)
    for part in (slice(0, 4096), slice(D // 2, D // 2 + 4096), slice(D - 4096, D)):
        r = x[0, part].double().view(-1, 2)
        want = ((r - r.mean(1, keepdim=True)) / torch.sqrt(r.var(1, unbiased=False, keepdim=True) + 1e-5)).view(-1)
        torch.testing.assert_close(y[0, part].double(), want, rtol=2.0**-8, atol=2.0**-8)
