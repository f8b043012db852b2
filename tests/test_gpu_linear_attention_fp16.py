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


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 130, 300])
def test_lengths(T):
    _check(2, 3, T, 64, 64, HF)
