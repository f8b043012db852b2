"""linear_attention in fp16 on values of every size that the type holds, against float64 recurrences (oracle/layer.py).

Bounds, on the norm of a difference (of a whole tensor, of one token's row or of one column), with E, N and f as in
test_gpu_linear_attention.py:

    ||a - b|| <= ||fp16(b) - b|| + c u ||E|| + f (||E|| + ||b||)

The first term is the output's own rounding, on fp16's subnormal grid too.  A factor that is rounded to fp16 moves by at
most u = 2^-11 of itself, with a standard deviation below u / sqrt(3) of it, so the norm of what that does to many outputs
is below u ||E||: c = 1 for a tensor, 2 for one row or column of at least 64.  There is no term for a factor's own smallest
step: operands are held where the type has all of its bits.  States and their gradients are float32, from products whose
one factor has 22 bits: c u = 2^-22 and no rounding of the output.
"""

import pytest
import torch

from helpers import gen, randn
from linattn import linear_attention
from oracle.layer import linear_attention_ref
from test_gpu_linear_attention import _check, _norms

pytestmark = pytest.mark.gpu

DEV = "cuda"
HF, F32 = torch.float16, torch.float32
u, u2 = 2.0**-11, 2.0**-22


def _bounds(q, k, v, lam, s_in, so, skv, lens, rev):
    """(E, what the state's error is measured by, f) of one pass."""
    fE, fS, f = _norms(q, k, v, lam, s_in, so, skv, lens, rev, F32)
    return fE / f, fS / f, f


def _compare(a, b, E, f, name, c=1.0, dim=None):
    """The bound above; dim: over this axis of [B, H, T, channels] alone."""
    a = a.detach().double().cpu()
    assert a.isfinite().all(), f"{name}: not finite"

    def norm(t):
        return t.norm() if dim is None else t.norm(dim=dim)
    bound = norm(b.to(HF).double() - b) + c * u * norm(E) + f * (norm(E) + norm(b)) + 1e-300
    ratio = (norm(a - b) / bound).max().item()
    assert ratio <= 1, f"{name}: {ratio:.3g} times the bound (off by {((a - b).norm() / b.norm()).item():.3g})"


def _compare_state(a, b, S, f, name):
    a = a.detach().double().cpu()
    ratio = ((a - b).norm() / ((u2 + f) * S.norm() + 1e-300)).item()
    assert ratio <= 1, f"{name}: {ratio:.3g} times the bound (off by {((a - b).norm() / b.norm()).item():.3g})"


def _run(q, k, v, do, lam, scale, S0=None, dS=None):
    """Forward and backward, and the same in float64: dicts of o, state, dq, dk, dv, dinitial."""
    T = q.shape[2]
    names = ["q", "k", "v"] + (["initial"] if S0 is not None else [])
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)] + ([S0.to(DEV).requires_grad_()] if S0 is not None else [])
    o, S = linear_attention(*leaves[:3], lam.to(DEV), scale=scale, initial_state=leaves[3] if S0 is not None else None,
                            return_state=True)
    grads = torch.autograd.grad((o, S) if dS is not None else o, leaves,
                                (do.to(DEV), dS.to(DEV)) if dS is not None else do.to(DEV))
    ref = [t.double().requires_grad_() for t in (q, k, v)] + ([S0.double().requires_grad_()] if S0 is not None else [])
    ro, rS = linear_attention_ref(*ref[:3], lam, scale, ref[3] if S0 is not None else None, None)
    rg = torch.autograd.grad((ro, rS), ref, (do.double(), torch.zeros_like(rS) if dS is None else dS.double()))
    got = dict(o=o, state=S, **{"d" + n: g for n, g in zip(names, grads)})
    want = dict(o=ro.detach(), state=rS.detach(), **{"d" + n: g for n, g in zip(names, rg)})
    n = [T] * q.shape[0]
    Eo, So, f = _bounds(q, k, v, lam, S0, scale, 1.0, n, False)
    Eq, _, _ = _bounds(do, v, k, lam, None if S0 is None else S0.transpose(2, 3), scale, 1.0, n, False)
    Ek, _, _ = _bounds(v, do, q, lam, None if dS is None else dS.transpose(2, 3), 1.0, scale, n, True)
    Ev, Sv, _ = _bounds(k, q, do, lam, dS, 1.0, scale, n, True)
    return got, want, dict(o=Eo, dq=Eq, dk=Ek, dv=Ev, state=So, dinitial=Sv), f


LAM = torch.tensor([-(2.0**-8), -(2.0**-5), 0.0])


# ----------------------------------------------------------------------- scores
@pytest.mark.parametrize("rest", [1.0, 0.1, 0.01, 0.001])
def test_a_large_score_leaves_the_other_tokens_their_digits(rest):
    """Two tokens whose scores are near or past the type's end, each in a block of 32 with others that are not."""
    g = gen(40)
    B, H, T, K = 1, 3, 64, 64
    q, k, v = rest * randn(g, B, H, T, K), 4 * randn(g, B, H, T, K), randn(g, B, H, T, K)
    for t in (9, 40):
        q[:, :, t] = randn(g, B, H, K) * (1e4 if rest < 1 else 1e3)
    q, k, v, do = (t.to(HF) for t in (q, k, 0.01 * v, randn(g, B, H, T, K)))
    scores = (q.double() @ k.double().transpose(2, 3)).abs() * K**-0.5
    assert scores[:, :, 40].max() > 32768 * (1 if rest < 1 else 0.1)
    got, want, E, f = _run(q, k, v, do, LAM, K**-0.5)
    _compare(got["o"], want["o"], E["o"], f, "o, by token", c=2, dim=-1)
    # the same of k's scores in the backward: one token's v
    v2 = randn(g, B, H, T, K)
    v2[:, :, 20] *= 1e4
    got, want, E, f = _run(q.clamp(-0.01, 0.01), k * 0.01, v2.to(HF), do * rest, LAM, K**-0.5)
    _compare(got["dk"], want["dk"], E["dk"], f, "dk, by token", c=2, dim=-1)


@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-5])
def test_small_scores(size):
    """One chunk, whose dk and dq are products of scores of do and v."""
    g = gen(41)
    q, k, v, do = (randn(g, 2, 3, 64, 64) for _ in range(4))
    got, want, E, f = _run(*(t.to(HF) for t in (q, k, v, size * do)), LAM, 64**-0.5)
    for name in ("o", "dq", "dk"):
        _compare(got[name], want[name], E[name], f, name)
        _compare(got[name], want[name], E[name], f, f"{name}, by token", c=2, dim=-1)


# ------------------------------------------------------------------- states
@pytest.mark.parametrize("q_size,lo,hi", [(1e3, -6, 0), (3e-3, -0.5, 5.5)], ids=["small", "large"])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 128), (200, 72), (33, 31)])
def test_columns_of_the_state_of_many_sizes(K, V, q_size, lo, hi):
    """o = q S for a state whose columns lie anywhere from below fp16's bits to past its end, 2^20 apart."""
    g = gen(42 + K)
    B, H, T = 1, 3, 64
    sizes = 10.0 ** torch.linspace(lo, hi, V)[torch.randperm(V, generator=g)]
    S0 = randn(g, B, H, K, V) * sizes
    q, k, v, do = q_size * randn(g, B, H, T, K), randn(g, B, H, T, K), torch.zeros(B, H, T, V), randn(g, B, H, T, V)
    got, want, E, f = _run(*(t.to(HF) for t in (q, k, v, do)), LAM, K**-0.5, S0, torch.zeros_like(S0))
    assert want["o"].abs().max() < 65504
    _compare(got["o"], want["o"], E["o"], f, "o, by column", c=2, dim=-2)
    # dk = dS v: dS of all sizes by its rows, which are dk's channels
    rows = 10.0 ** torch.linspace(lo, hi, K)[:, None]
    got, want, E, f = _run(*(t.to(HF) for t in (q, k, q_size * do, 0 * do)), LAM, K**-0.5, torch.zeros_like(S0),
                           randn(g, B, H, K, V) * rows)
    assert want["dk"].abs().max() < 65504
    _compare(got["dk"], want["dk"], E["dk"], f, "dk, by column", c=2, dim=-2)


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("T", [40, 300, 1500])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 128), (200, 40), (100, 100)])
def test_small_gradients(K, V, T, size):
    """o's gradient as it is without a loss scale: every gradient, and the initial state's in float32."""
    g = gen(43 + K)
    B, H = 1, 3
    q, k, v, do = (randn(g, B, H, T, c) for c in (K, K, V, V))
    S0, dS = randn(g, B, H, K, V), size * randn(g, B, H, K, V)
    got, want, E, f = _run(*(t.to(HF) for t in (q, k, v, size * do)), LAM, K**-0.5, S0, dS)
    for name in ("o", "dq", "dk", "dv"):
        _compare(got[name], want[name], E[name], f, name)
    _compare_state(got["state"], want["state"], E["state"], f, "state")
    _compare_state(got["dinitial"], want["dinitial"], E["dinitial"], f, "dinitial")


@pytest.mark.parametrize("size", [1e-3, 1e-5])
@pytest.mark.parametrize("T", [40, 300, 1500])
def test_small_values(T, size):
    """v small, and some of its columns smaller still: o, and the state by column, which is float32."""
    g = gen(44)
    B, H, K, V = 2, 3, 64, 96
    q, k, v, do = (randn(g, B, H, T, c) for c in (K, K, V, V))
    sizes = torch.where(torch.arange(V) % 3 == 0, size, 1.0)
    got, want, E, f = _run(*(t.to(HF) for t in (q, k, v * size, do)), LAM, K**-0.5)
    _compare(got["o"], want["o"], E["o"], f, "o")
    _compare(got["dq"], want["dq"], E["dq"], f, "dq")
    _compare_state(got["state"], want["state"], E["state"], f, "state")
    got, want, E, f = _run(*(t.to(HF) for t in (q, k, v * sizes, do)), LAM, K**-0.5)
    _compare(got["o"], want["o"], E["o"], f, "o, by column", c=2, dim=-2)
    for n in range(0, V, 7):
        _compare_state(got["state"][..., n], want["state"][..., n], E["state"][..., n], f, f"state, column {n}")


@pytest.mark.parametrize("T", [40, 300, 1500])
@pytest.mark.parametrize("scale", [4.0, 300.0, -4.0])
def test_scaled_values_past_the_type(T, scale):
    """A scale above one and a loss-scaled gradient: their product passes the type, the gradients do not."""
    g = gen(45)
    B, H, K = 1, 3, 64
    q, k, v, do = (randn(g, B, H, T, K) for _ in range(4))
    small = 0.02 * abs(4.0 / scale) ** 0.5 * min(1.0, (300 / T) ** 0.5)
    q, k, v, do = (t.to(HF) for t in (small * q, small * k, small * 1e-2 * v, (2e4 * do).clamp(-6e4, 6e4)))
    assert do.double().abs().max() * abs(scale) > 2 * 65504
    got, want, E, f = _run(q, k, v, do, LAM, scale, torch.zeros(B, H, K, K), torch.zeros(B, H, K, K))
    for name in ("o", "dq", "dk", "dv"):
        assert want[name].abs().max() < 65504
        _compare(got[name], want[name], E[name], f, name)
    _compare_state(got["dinitial"], want["dinitial"], E["dinitial"], f, "dinitial")


def test_values_and_decays_far_apart():
    """Chunks whose values are far larger or smaller than those before, under decays that leave either, and zeros."""
    g = gen(46)
    B, H, T, K = 1, 4, 512, 64
    lam = torch.tensor([0.0, -0.01, -0.7, -float("inf")])
    q, k, v, do = (randn(g, B, H, T, K) for _ in range(4))
    sizes = torch.tensor([1e-4, 1e3, 0.0, 1e-2, 1.0, 3e-5, 1e2, 0.0]).repeat_interleave(64)[:, None]
    got, want, E, f = _run(*(t.to(HF) for t in (q, k, v * sizes, do)), lam, K**-0.5)
    _compare(got["o"], want["o"], E["o"], f, "o, by token", c=2, dim=-1)
    for h in range(H):
        _compare_state(got["state"][:, h], want["state"][:, h], E["state"][:, h], f, f"state of head {h}")


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 130, 300])
def test_lengths(T):
    _check(2, 3, T, 64, 64, HF)
