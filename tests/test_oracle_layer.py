"""What pins oracle/layer.py: hand-computed values, a second formulation, gradcheck (CPU)."""

import math

import torch

import helpers  # noqa: F401  (sets sys.path)
from helpers import gen, randn
from oracle.layer import group_norm_ref, linear_attention_ref, lowrank_step_ref
from oracle.reference_cpu import lowrank_dynamic_convolution_ref


def test_linear_attention_by_hand():
    # one head of one channel: S = 1*2 = 2, then 0.5*2 + 3*5 = 16; o = 0.5 * q S
    q, k, v = (torch.tensor(t).view(1, 1, 2, 1) for t in ([7.0, 11.0], [1.0, 3.0], [2.0, 5.0]))
    o, S = linear_attention_ref(q, k, v, torch.tensor([math.log(0.5)], dtype=torch.float64), 0.5)
    torch.testing.assert_close(o.flatten(), torch.tensor([7.0, 88.0], dtype=torch.float64))
    torch.testing.assert_close(S.flatten(), torch.tensor([16.0], dtype=torch.float64))


def test_linear_attention_against_all_pairs():
    g = gen(1)
    B, H, T, K, V = 2, 3, 9, 4, 5
    q, k, v = (randn(g, B, H, T, n).double() for n in (K, K, V))
    S0, lam = randn(g, B, H, K, V).double(), -torch.rand(H, generator=g).double()
    lens = [9, 4]
    o, S = linear_attention_ref(q, k, v, lam, 0.3, S0, lens)
    for b in range(B):
        for h in range(H):
            n = lens[b]
            for t in range(T):
                want = torch.zeros(V, dtype=torch.float64)
                if t < n:
                    want = 0.3 * torch.exp(lam[h] * (t + 1)) * (q[b, h, t] @ S0[b, h])
                    for j in range(t + 1):
                        want = want + 0.3 * torch.exp(lam[h] * (t - j)) * (q[b, h, t] @ k[b, h, j]) * v[b, h, j]
                torch.testing.assert_close(o[b, h, t], want)
            want = torch.exp(lam[h] * n) * S0[b, h]
            for j in range(n):
                want = want + torch.exp(lam[h] * (n - 1 - j)) * torch.outer(k[b, h, j], v[b, h, j])
            torch.testing.assert_close(S[b, h], want)


def test_linear_attention_ignores_rows_past_the_length():
    g = gen(2)
    q, k, v = (randn(g, 2, 1, 6, 3).double() for _ in range(3))
    for t in (q, k, v):
        t[0, :, 2:] = math.nan
        t[1] = math.inf
    o, S = linear_attention_ref(q, k, v, torch.tensor([-0.1]), 1.0, None, [2, 0])
    assert torch.isfinite(o).all() and torch.isfinite(S).all()
    assert (o[0, :, 2:] == 0).all() and (o[1] == 0).all() and (S[1] == 0).all()


def test_gradcheck():
    g = gen(3)
    q, k, v, S0 = (randn(g, *s).double().requires_grad_() for s in ((1, 2, 4, 3), (1, 2, 4, 3), (1, 2, 4, 2), (1, 2, 3, 2)))
    lam = torch.tensor([-0.2, 0.0])
    assert torch.autograd.gradcheck(lambda *a: linear_attention_ref(*a[:3], lam, 0.5, a[3], [3]), (q, k, v, S0))
    x, w, b, gate = (randn(g, *s).double().requires_grad_() for s in ((2, 3, 8), (8,), (8,), (2, 3, 8)))
    assert torch.autograd.gradcheck(lambda *a: group_norm_ref(a[0], 2, a[1], a[2], a[3]), (x, w, b, gate))
    assert torch.autograd.gradcheck(lambda *a: group_norm_ref(a[0], 4, a[1], a[2]), (x, w, b))


def test_group_norm_by_hand():
    # two groups of two channels: (1, 3) and (5, 5); weight 2, bias 1, no activation
    x = torch.tensor([[1.0, 3.0, 5.0, 5.0]])
    y = group_norm_ref(x, 2, torch.full((4,), 2.0), torch.ones(4), activation=None, eps=0.0001)
    r = 1 / math.sqrt(1.0001)
    torch.testing.assert_close(y, torch.tensor([[1 - 2 * r, 1 + 2 * r, 1.0, 1.0]], dtype=torch.float64))
    s = group_norm_ref(x, 2, torch.full((4,), 2.0), torch.ones(4), eps=0.0001)
    torch.testing.assert_close(s, y * torch.sigmoid(y))


def test_lowrank_step_is_a_row_of_the_whole_sequence():
    g = gen(4)
    N, T, D, R, W = 2, 6, 5, 3, 4
    x, z, U, sw = randn(g, N, T, D), randn(g, N, T, R), randn(g, R, W * D), randn(g, W, D)
    whole = lowrank_dynamic_convolution_ref(x.double(), z.double(), U.double(), sw.double(), residual=True)
    state = torch.zeros(N, W - 1, D)
    for t in range(T):
        y, state = lowrank_step_ref(x[:, t], z[:, t], U, state, sw, True)
        torch.testing.assert_close(y, whole[:, t])
