"""DynamicLinearAttention: the convolutions, linear attention, the norm and their single-token forms run together.

In float32 the pieces of a sequence are the same sums in other orders: outputs agree to 1e-4 of the largest (a chain of
five products whose float32 sums are good to about 1e-6 each, a norm that divides by a deviation of about 1)."""

import pytest
import torch

from helpers import gen, max_rel, randn
from linattn import DynamicLinearAttention
from oracle.layer import group_norm_ref, linear_attention_ref
from oracle.reference_cpu import lowrank_dynamic_convolution_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _layer(D=128, H=4, R=7, W=4, dtype=torch.float32):
    torch.manual_seed(0)
    m = DynamicLinearAttention(D, H, R, W)
    with torch.no_grad():
        m.conv.proj_out.normal_(0, 0.2)
        m.norm_weight.normal_(1, 0.1)
        m.norm_bias.normal_(0, 0.1)
    return m.to(device=DEV, dtype=dtype)


def _ref(m, x, lens=None):
    """The layer in float64 on the CPU, whole sequences."""
    p = {k: v.detach().double().cpu() for k, v in m.named_parameters()}
    B, T, D = x.shape
    H, R, hd = m.heads, m.conv.R, m.head_dim
    qkv = x @ p["c_attn.weight"].t()
    z = x @ p["conv.proj_in.weight"].t()
    heads = []
    for g in range(3):
        y = lowrank_dynamic_convolution_ref(qkv[..., g * D:(g + 1) * D].contiguous(), z[..., g * R:(g + 1) * R].contiguous(),
                                            p["conv.proj_out"][g], p["conv.proj_out_bias"][g], residual=True)
        heads.append(y.view(B, T, H, hd).transpose(1, 2))
    o, S = linear_attention_ref(*heads, m.log_decay.cpu(), hd**-0.5, None, lens)
    y = group_norm_ref(o.transpose(1, 2).reshape(B, T, D), H, p["norm_weight"], p["norm_bias"],
                       x @ p["c_gate.weight"].t(), "silu", m.eps)
    return y @ p["c_proj.weight"].t(), S


def test_forward_against_float64():
    m = _layer()
    x = randn(gen(1), 2, 150, 128)
    out, state = m(x.to(DEV), return_state=True)
    ref, S = _ref(m, x.double())
    assert max_rel(out, ref) < 1e-4 and max_rel(state.attn, S) < 1e-4


def test_prompt_in_pieces_then_tokens():
    m = _layer()
    B, T = 3, 140
    x = randn(gen(2), B, T, 128).to(DEV)
    with torch.no_grad():
        whole = m(x)
        a, state = m(x[:, :2], return_state=True)          # shorter than the filters
        b, state = m(x[:, 2:100], state=state, return_state=True)
        parts = [a, b] + [m.step(x[:, t], state)[:, None] for t in range(100, T)]
    assert max_rel(torch.cat(parts, 1), whole) < 1e-4


def test_ragged_prompts_into_a_cache():
    """Prompts of different lengths, padded with NaN, then tokens from rows of a larger cache."""
    m = _layer()
    lens, T = [70, 0, 1, 33], 70
    x = randn(gen(3), 4, T + 2, 128).to(DEV)
    padded = x[:, :T].clone()
    for b, n in enumerate(lens):
        padded[b, n:] = float("nan")
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    slots = torch.tensor([5, 0, 3, 6], dtype=torch.int32, device=DEV)
    cache = m.new_state(7)
    with torch.no_grad():
        out, state = m(padded, lengths=n, return_state=True)
        cache.conv[slots.long()] = state.conv
        cache.attn[slots.long()] = state.attn
        idle = cache.attn[1].clone()
        steps = []
        for i in range(2):
            token = torch.stack([x[b, m_ + i] for b, m_ in enumerate(lens)])
            steps.append(m.step(token, cache, slots=slots))
        for b, k in enumerate(lens):
            want = m(x[b:b + 1, :k + 2])[0]
            assert max_rel(torch.cat([out[b, :k], steps[0][b:b + 1], steps[1][b:b + 1]]), want) < 1e-4
    assert torch.equal(cache.attn[1], idle)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_training_reaches_every_parameter(dtype):
    m = _layer(dtype=dtype)
    assert m.log_decay.dtype == torch.float32
    x = randn(gen(4), 2, 100, 128).to(DEV).to(dtype).requires_grad_()
    out = m(x)
    dout = randn(gen(5), *out.shape)
    out.backward(dout.to(DEV).to(dtype))
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name
    if dtype == torch.float32:
        r = x.detach().double().cpu().requires_grad_()
        (want,) = torch.autograd.grad(_ref(m, r)[0], r, dout.double())
        assert max_rel(x.grad, want) < 1e-4


def test_sizes_are_checked():
    with pytest.raises(ValueError):
        DynamicLinearAttention(100, 3, 7, 4)
    with pytest.raises(ValueError):
        DynamicLinearAttention(128, 4, 6, 4)  # R + 1 is no power of two
