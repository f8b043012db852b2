"""gated_delta_rule's states kept for the backward, and workgroups past two to a CU (bounds: test_gpu_delta_rule.py)."""

import pytest
import torch

from test_gpu_delta_rule import BF, DEV, F32, HF, _check, _inputs

pytestmark = pytest.mark.gpu


class _Ctx:
    def __init__(self, *needs):
        self.needs_input_grad = needs

    def set_materialize_grads(self, value):
        pass

    def save_for_backward(self, *tensors):
        self.saved_tensors = tensors


@pytest.mark.parametrize("size", [(1, 2, 4, 700, 128, 128), (2, 2, 2, 3000, 128, 64), (1, 16, 16, 300, 64, 96), (1, 1, 2, 200, 250, 250)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_kept_states_are_those_of_the_backward(size, dtype):
    """The backward from the forward's states, from its triangular systems alone, and from nothing but the inputs."""
    from dynconv.delta import _GatedDeltaRuleFn as Fn

    B, Hk, H, T, K, V = size
    tensors, s0, _ = _inputs(*size, dtype, dtype, True, 5)
    q, k, v, lam, beta, do, s0 = (t.to(DEV) for t in (*tensors, s0))
    lens = torch.tensor([T - 70] * B, dtype=torch.int32, device=DEV)
    seen = []
    for flags in (5, 1):
        ctx = _Ctx(*[True] * 6)
        o = Fn.forward(ctx, q, k, v, lam, beta, s0, lens, K**-0.5, 1e-6, flags, False)
        seen.append((o, *Fn.backward(ctx, do)[:6]))
        ctx.saved_tensors = ctx.saved_tensors[:-1] + (None,)
        seen.append((o, *Fn.backward(ctx, do)[:6]))
    assert all(torch.isfinite(t).all() for t in seen[0])
    for other in seen[1:]:
        for name, a, b in zip(("o", "dq", "dk", "dv", "dlog_decay", "dbeta", "dinitial"), seen[0], other):
            assert torch.equal(a, b), name


@pytest.mark.parametrize("size", [(3, 48, 48, 70, 128, 128), (2, 8, 16, 1300, 128, 128), (1, 24, 24, 1000, 128, 120)])
@pytest.mark.parametrize("state", [False, True])
def test_workgroups_past_two_to_a_cu(size, state):
    """bf16 with float32 results at 128 channels: more than 512 workgroups, of chains and of segments."""
    _check(*size, BF, "fp32", state=state, lens=[size[3] - 35 * b for b in range(size[0])])
