"""What linear_attention keeps for its backward, through the native binding and without it."""

import pytest
import torch

from helpers import gen, randn
from linattn import linear_attention

pytestmark = pytest.mark.gpu

DEV = "cuda"
B, H, T, K = 1, 2, 3000, 64


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    from dynconv import _capi

    _capi.load()
    if request.param == "python":
        monkeypatch.setattr(_capi, "binding", None)
    elif _capi.binding is None:
        pytest.skip("no native binding")


def _leaves(seed):
    g = gen(seed)
    return [randn(g, B, H, T, K).to(torch.bfloat16).to(DEV).requires_grad_() for _ in range(3)]


def _states_bytes():
    from dynconv import _capi

    n = _capi.load().dc_linear_attention_ws_bytes(B, H, T, K, K, _capi.dtype_code(torch.bfloat16), 0)
    assert n > 0, "several segments"
    return n


def test_the_segments_states_go_with_the_saved_tensors(path):
    """Freed by the backward, though the output and its node live on."""
    leaves = _leaves(1)
    lam = torch.full((H,), -0.01, device=DEV)
    o = linear_attention(*leaves, lam)
    do = torch.ones_like(o)
    torch.autograd.grad(o, leaves, do, retain_graph=True)
    held = torch.cuda.memory_allocated()
    torch.autograd.grad(o, leaves, do)
    assert o.grad_fn is not None and held - torch.cuda.memory_allocated() >= _states_bytes()
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(o, leaves, do)


def test_saved_tensor_hooks_see_them(path):
    leaves = _leaves(2)
    lam = torch.full((H,), -0.01, device=DEV)
    do = randn(gen(3), B, H, T, K).to(torch.bfloat16).to(DEV)
    want = torch.autograd.grad(linear_attention(*leaves, lam), leaves, do)
    sizes = []

    def pack(t):
        sizes.append(t.numel() * t.element_size())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
        o = linear_attention(*leaves, lam)
    assert _states_bytes() in sizes
    for a, b in zip(torch.autograd.grad(o, leaves, do), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("given", [True, False], ids=["forward's workspace", "own states"])
def test_the_backward_stays_within_its_workspace(given):
    """The C entry with and without the forward's workspace: equal gradients, and nothing written past either size."""
    from dynconv import _capi

    lib = _capi.load()
    q, k, v = (t.detach() for t in _leaves(4))
    do = randn(gen(5), B, H, T, K).to(torch.bfloat16).to(DEV)
    lam = torch.full((H,), -0.01, device=DEV)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(linear_attention(*leaves, lam), leaves, do)
    o, grads = torch.empty_like(q), [torch.empty_like(t) for t in (q, k, v)]
    dtype, st = _capi.dtype_code(q.dtype), _capi.int64_array(q.stride()[:3])

    def room(which):
        n = lib.dc_linear_attention_ws_bytes(B, H, T, K, K, dtype, which)
        return torch.full((n + 4096,), 77, dtype=torch.uint8, device=DEV), n

    ws, n = room(0)
    args = [x for t in (q, k, v) for x in (_capi.ptr(t), st)]
    _capi.check(lib.dc_linear_attention_fwd(*args, _capi.ptr(lam), None, None, _capi.ptr(o), st, None, _capi.ptr(ws), n, B,
                                            H, T, K, K, K**-0.5, dtype, _capi.stream_of(q)), "forward")
    kept = ws.clone()
    bws, m = room(2 if given else 1)
    out = [x for t in grads for x in (_capi.ptr(t), st)]
    _capi.check(lib.dc_linear_attention_bwd(*args, _capi.ptr(lam), None, None, _capi.ptr(do), st, None, *out, None,
                                            _capi.ptr(ws) if given else None, _capi.ptr(bws), m, B, H, T, K, K, K**-0.5,
                                            dtype, _capi.stream_of(q)), "backward")
    assert (ws[n:] == 77).all() and (bws[m:] == 77).all() and torch.equal(ws, kept)
    for a, b in zip(grads, want):
        assert torch.equal(a, b)
