"""DynamicDeltaRule and DynamicDeltaStack: the convolutions, the gated delta rule, the norms and their single-token forms run
together.

In float32 the pieces of a sequence are the same sums in other orders: outputs agree to 1e-4 of the largest (a chain of
five products a layer whose float32 sums are good to about 1e-6 each, norms that divide by deviations of about 1).  In bf16
each of the chain's tensors is rounded to 2^-8 of itself: outputs of one layer agree to 6 roundings, 6 * 2^-8, of the largest
in the norm, of two layers on the residual stream to twice that."""

import pytest
import torch

from helpers import gen, max_rel, randn
from linattn import DynamicDeltaRule, DynamicDeltaStack
from oracle.layer import gated_delta_rule_ref, group_norm_ref, residual_norm_ref
from oracle.reference_cpu import lowrank_dynamic_convolution_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _model(kind, D=128, H=4, R=7, W=4, dtype=F32, stream=None):
    torch.manual_seed(0)
    m = DynamicDeltaRule(D, H, R, W) if kind == "layer" else DynamicDeltaStack(D, H, 2, R, W, stream=stream)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith("proj_out"):
                p.normal_(0, 0.2)
            elif "weight" in name and p.dim() == (1 if kind == "layer" else p.dim()) and "c_" not in name and "proj_in" not in name:
                p.normal_(1, 0.1)
            elif name.endswith(("bias", "scale")):
                p.normal_(0.5, 0.1)
    return m.to(device=DEV, dtype=dtype)


def _layer_ref(m, x, lens=None):
    """The layer in float64 on the CPU, whole sequences."""
    p = {k: v.detach().double().cpu() for k, v in m.named_parameters()}
    B, T, D = x.shape
    H, R, hd = m.heads, m.conv.R, m.head_dim
    qkv, z = x @ p["c_attn.weight"].t(), x @ p["conv.proj_in.weight"].t()
    heads = []
    for g in range(3):
        y = lowrank_dynamic_convolution_ref(qkv[..., g * D:(g + 1) * D].contiguous(), z[..., g * R:(g + 1) * R].contiguous(),
                                            p["conv.proj_out"][g], p["conv.proj_out_bias"][g], residual=True)
        heads.append(y.view(B, T, H, hd).transpose(1, 2))
    rate = torch.exp(p["log_rate"])
    lam = -rate * torch.log1p(torch.exp(x @ p["c_decay.weight"].t() + p["decay_bias"]))
    beta = 1 / (1 + torch.exp(-(x @ p["c_beta.weight"].t())))
    o, S = gated_delta_rule_ref(*heads, lam.transpose(1, 2), beta.transpose(1, 2), hd**-0.5, None, lens, True)
    y = group_norm_ref(o.transpose(1, 2).reshape(B, T, D), H, p["norm_weight"], p["norm_bias"], x @ p["c_gate.weight"].t(), "silu",
                       m.eps)
    return y @ p["c_proj.weight"].t(), S


def _stack_ref(m, x):
    p = {k: v.detach().double().cpu() for k, v in m.named_parameters()}
    h = x
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + m.eps) * p["weight"][0]
    for i, layer in enumerate(m.layers):
        y, h = residual_norm_ref(h, _layer_ref(layer, y)[0], p["weight"][i + 1], p["branch_weight"][i], None, None, p["scale"][i], m.eps)
    return y


def test_forward_against_float64():
    m = _model("layer")
    x = randn(gen(1), 2, 150, 128)
    out, state = m(x.to(DEV), return_state=True)
    ref, S = _layer_ref(m, x.double())
    assert max_rel(out, ref) < 1e-4 and max_rel(state.attn, S) < 1e-4
    m = _model("stack")
    assert max_rel(m(x.to(DEV)), _stack_ref(m, x.double())) < 2e-4


@pytest.mark.parametrize("stream", [None, F32])
def test_bf16_against_float64(stream):
    x = randn(gen(6), 2, 150, 128).to(BF)
    m = _model("stack", dtype=BF, stream=stream)
    out, ref = m(x.to(DEV)), _stack_ref(m, x.double())
    assert out.dtype == BF
    assert (out.double().cpu() - ref).norm() <= 12 * 2.0**-8 * ref.norm()


@pytest.mark.parametrize("kind", ["layer", "stack"])
def test_prompt_in_pieces_then_tokens(kind):
    m = _model(kind)
    B, T = 3, 140
    x = randn(gen(2), B, T, 128).to(DEV)
    with torch.no_grad():
        whole = m(x)
        a, state = m(x[:, :2], return_state=True)          # shorter than the filters
        b, state = m(x[:, 2:100], state, return_state=True)
        parts = [a, b] + [m.step(x[:, t], state)[:, None] for t in range(100, T)]
    assert max_rel(torch.cat(parts, 1), whole) < 2e-4


def test_ragged_prompts_into_a_cache():
    """Prompts of different lengths, padded with NaN, then tokens from rows of a larger cache."""
    m = _model("stack")
    lens, T = [70, 0, 1, 33], 70
    x = randn(gen(3), 4, T + 2, 128).to(DEV)
    padded = x[:, :T].clone()
    for b, n in enumerate(lens):
        padded[b, n:] = float("nan")
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    slots = torch.tensor([5, 0, 3, 6], dtype=torch.int32, device=DEV)
    cache = m.new_state(7)
    with torch.no_grad():
        out, states = m(padded, lengths=n, return_state=True)
        for c, s in zip(cache, states):
            c.conv[slots.long()] = s.conv
            c.attn[slots.long()] = s.attn
        idle = cache[1].attn[1].clone()
        steps = []
        for i in range(2):
            token = torch.stack([x[b, m_ + i] for b, m_ in enumerate(lens)])
            steps.append(m.step(token, cache, slots=slots))
        for b, k in enumerate(lens):
            want = m(x[b:b + 1, :k + 2])[0]
            assert max_rel(torch.cat([out[b, :k], steps[0][b:b + 1], steps[1][b:b + 1]]), want) < 2e-4
    assert torch.equal(cache[1].attn[1], idle)


@pytest.mark.parametrize("kind", ["layer", "stack"])
@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_training_reaches_every_parameter(kind, dtype):
    m = _model(kind, dtype=dtype)
    x = randn(gen(4), 2, 100, 128).to(DEV).to(dtype).requires_grad_()
    out = m(x)
    dout = randn(gen(5), *out.shape)
    out.backward(dout.to(DEV).to(dtype))
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name
    if dtype == F32:
        r = x.detach().double().cpu().requires_grad_()
        ref = _layer_ref(m, r)[0] if kind == "layer" else _stack_ref(m, r)
        (want,) = torch.autograd.grad(ref, r, dout.double())
        assert max_rel(x.grad, want) < 4e-4


def test_captured_decoding():
    """A step of the stack recorded once and replayed moves the states as eager steps do."""
    m = _model("stack", dtype=BF)
    x = randn(gen(7), 6, 3, 128).to(BF).to(DEV)
    a, b, warm = (m.new_state(3) for _ in range(3))
    static = x[0].clone()
    m.step(static, warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.step(static, a)
    for t in range(6):
        static.copy_(x[t])
        graph.replay()
        want = m.step(x[t], b)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert all(torch.equal(p, q) for s, r in zip(a, b) for p, q in zip(s, r))
