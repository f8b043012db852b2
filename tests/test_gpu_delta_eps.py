"""gated_delta_rule with normed rows and an eps of zero or close to it, or rows far longer than one: what lies behind a partial
chunk, or past a length, has no part in anything (bounds: test_gpu_delta_rule.py).

One token without a state before it has a dlog_decay of zero, which leaves no relative bound.  The kernel forms it as q.dq - k.dk
with dq = p k and dk = p q of the same p = scale b (do.v) / (|q| |k|).  Each of the two sums has K terms p q_d k_d, each rounded
twice (dq, and its product with q) and then in a sum of up to 16 steps (4 terms of a lane for each of 4 blocks of channels at
most, 2 exchanges and 2 additions of wavefronts): within 20 roundings of 2^-24 of sum |p q_d k_d| <= scale b |do.v|, as the rows
are no longer than 1 then.  do.v of K products in parts enters both alike.  Together 40 2^-24 < 2^-18 of scale b |do| |v|."""

import pytest
import torch

from linattn import gated_delta_rule
from oracle.layer import gated_delta_rule_chunked
from test_gpu_delta_rule import BF, DEV, F32, HF, NAMES, _compare, _inputs, _rounding

pytestmark = pytest.mark.gpu


def _check(size, dtype, eps, state, lens=None, long=1.0):
    B, Hk, H, T, K, V = size
    print(f"[delta eps] {size} {dtype} eps={eps} state={state} {lens} rows {long} times as long", flush=True)
    (q, k, v, lam, beta, do), S0, dS = _inputs(*size, dtype, dtype, True, 12)
    q, k = ((t * long).to(dtype) for t in (q, k))
    s0, ds = (S0, dS) if state else (None, None)
    args, before = (q, k, v, lam, beta, K**-0.5, do, s0, ds, lens, True, eps), []
    (eo, eS), eg = gated_delta_rule_chunked(*args, before=before)
    r, u_r = _rounding(dtype, state)
    (ro, rS), rg = gated_delta_rule_chunked(*args, dtype=F32, r=r)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam, beta, S0)[:6 if state else 5]]
    ld = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = gated_delta_rule(*leaves[:5], initial_state=leaves[5] if state else None, lengths=ld, return_state=state, normalize=True,
                           eps=eps)
    grads = torch.autograd.grad(out, leaves, (do.to(DEV), dS.to(DEV)) if state else do.to(DEV))
    got = [*(out if state else (out, None)), *grads, *([] if state else [None])]
    if T == 1 and not state:
        most = K**-0.5 * beta[:, :, 0].double().abs() * (do[:, :, 0].double().norm(dim=-1) * v[:, :, 0].double().norm(dim=-1))
        assert (got[5][:, :, 0].double().cpu().abs() <= 2.0**-18 * most).all()
        got[5] = None
    dt = dict.fromkeys(NAMES, dtype) | dict(state=F32, dinitial=F32)
    _compare(got, (eo, eS, *eg), (ro, rS, *rg), dt, u_r, before)


SIZES = [((1, 1, 1, 1, 64, 64), None), ((2, 2, 4, 65, 64, 64), [65, 1]), ((2, 1, 2, 33, 128, 128), [33, 17]), ((1, 1, 1, 70, 100, 40), None),
         ((9, 16, 16, 20, 128, 128), None), ((1, 2, 2, 700, 128, 128), None), ((1, 1, 1, 66, 256, 64), None)]


@pytest.mark.parametrize("size,lens", SIZES)
@pytest.mark.parametrize("eps", [0.0, 1e-12])
@pytest.mark.parametrize("dtype,state", [(BF, False), (BF, True), (HF, False), (HF, True), (F32, True)])
def test_small_eps(size, lens, eps, dtype, state):
    _check(size, dtype, eps, state, lens)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", [(1, 1, 1, 65, 64, 64), (1, 2, 2, 97, 128, 128)])
def test_long_rows(size, dtype):
    _check(size, dtype, 1e-6, True, long=1024.0)
