"""group_norm against float64 (oracle/layer.py), forward and gradients.

Everything between the inputs and the outputs is float32, so an entry is off by the rounding to its type (r: 2^-8
bf16, 2^-11 fp16, 2^-23 fp32) and by float32 roundings of the terms it is made of.  Those are bounded by 2^-18 of the
terms' magnitudes: the statistics' sums and the hardware exponential are good to about 2^-21 of theirs, and x - mean to
2^-23 (|x| + |mean|), whose share grows with |mean| rstd.
"""

import pytest
import torch

from helpers import gen, randn
from linattn import group_norm
from oracle.layer import group_norm_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
R = {BF: 2.0**-8, HF: 2.0**-11, F32: 2.0**-23}


def _close(a, b, terms, dtype, name):
    bound = R[dtype] * b.abs() + 2.0**-18 * terms + (2.0**-25 if dtype == HF else 1e-30)
    ratio = ((a.detach().double().cpu() - b).abs() / bound).nan_to_num(nan=float("inf"))
    assert ratio.max() <= 1, f"{name}: {ratio.max().item():.3g} times the bound at {int(ratio.argmax())}"


def _check(shape, groups, dtype, pdtype=None, weight=True, bias=True, gate=True, act="silu", mean=0.0, scale=2.0,
           eps=1e-5, seed=0):
    print(f"[group_norm] {shape} groups {groups} {dtype} weight={weight} bias={bias} gate={gate} {act}", flush=True)
    pdtype = pdtype or dtype
    g = gen(seed + shape[-1])
    D = shape[-1]
    x = (mean + scale * randn(g, *shape)).to(dtype)
    w = (1 + 0.3 * randn(g, D)).to(pdtype) if weight else None
    b = (0.3 * randn(g, D)).to(pdtype) if bias else None
    gt = (2 * randn(g, *shape)).to(dtype) if gate else None
    dy = randn(g, *shape).to(dtype)
    dev = [None if t is None else t.to(DEV).requires_grad_() for t in (x, w, b, gt)]
    y = group_norm(dev[0], groups, weight=dev[1], bias=dev[2], gate=dev[3], activation=act, eps=eps)
    wanted = [t for t in dev if t is not None]
    grads = iter(torch.autograd.grad(y, wanted, dy.to(DEV)))
    ref = [None if t is None else t.double().requires_grad_() for t in (x, w, b, gt)]
    ry = group_norm_ref(ref[0], groups, ref[1], ref[2], ref[3], act, eps)
    rg = iter(torch.autograd.grad(ry, [t for t in ref if t is not None], dy.double()))

    with torch.no_grad():
        rows = x.double().reshape(-1, groups, D // groups)
        mu = rows.mean(-1, keepdim=True)
        rstd = 1 / torch.sqrt(((rows - mu) ** 2).mean(-1, keepdim=True) + eps)
        grow = (1 + mu.abs() * rstd)  # digits that x - mean loses

        def per(t):
            return t.reshape(-1, groups, D // groups)

        xh = (rows - mu) * rstd
        ww = per((torch.ones(D) if w is None else w).double().expand(shape))
        bb = per((torch.zeros(D) if b is None else b).double().expand(shape))
        u = xh * ww + bb
        U = (xh.abs() + grow - 1) * ww.abs() + bb.abs() + 2.0**-3 * ww.abs()
        a = u if gt is None else per(gt.double())
        fac = (1 + a.abs()) * (1 if gt is None else 1 + a.abs())
        _close(y, ry, (U * fac).reshape(shape), dtype, "y")
        d = per(dy.double()).abs()
        du = d * fac * (1 + U)
        duw = du * ww.abs()
        dx = rstd * grow * (duw + duw.mean(-1, keepdim=True) + xh.abs() * (duw * xh.abs()).mean(-1, keepdim=True))
        _close(next(grads), next(rg), dx.reshape(shape), dtype, "dx")
        n = tuple(range(len(shape) - 1))
        if weight:
            _close(next(grads), next(rg), (du * (xh.abs() + grow)).reshape(shape).sum(n), pdtype, "dweight")
        if bias:
            _close(next(grads), next(rg), du.reshape(shape).sum(n), pdtype, "dbias")
        if gate:
            _close(next(grads), next(rg), (d * U * fac).reshape(shape), dtype, "dgate")


# group sizes: one channel, odd, off the pieces, several pieces a lane, the largest
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D,groups", [(5, 5), (21, 3), (64, 8), (100, 1), (1000, 10), (2048, 16), (600, 1), (4096, 1),
                                      (1030, 2), (4095, 1), (4094, 1), (8192, 2), (512, 512), (130, 13)])
def test_group_sizes(D, groups, dtype):
    _check((2, 9, D), groups, dtype)


@pytest.mark.parametrize("gate", [False, True], ids=["", "gate"])
@pytest.mark.parametrize("act", ["silu", None])
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
def test_forms(gate, act, weight, bias):
    _check((3, 17, 256), 4, BF, weight=weight, bias=bias, gate=gate, act=act, seed=3)


@pytest.mark.parametrize("shape", [(1, 64), (64,), (1, 1, 1, 64), (2, 3001, 128), (20000, 64)])
def test_rows(shape):
    _check(shape, 4, HF, seed=4)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_float32_parameters(dtype):
    _check((2, 50, 384), 3, dtype, pdtype=F32, seed=5)


def test_means_far_from_zero_and_flat_groups():
    _check((2, 30, 256), 2, F32, mean=300.0, scale=0.5, seed=6)
    x = torch.full((3, 4, 64), 7.0, device=DEV)  # variance 0: u = bias
    b = torch.randn(64, device=DEV)
    y = group_norm(x, 8, bias=b, activation=None)
    assert torch.equal(y, b.expand(3, 4, 64))


def test_large_gates():
    """exp overflows in the sigmoid of a very negative gate: the output is 0, not NaN."""
    x = torch.randn(4, 64, device=DEV)
    gate = torch.full((4, 64), -1e4, device=DEV, requires_grad=True)
    y = group_norm(x, 2, gate=gate)
    (d,) = torch.autograd.grad(y, gate, torch.ones_like(y))
    assert (y == 0).all() and (d == 0).all()


def test_unaligned_rows():
    """x whose rows start off the 16-byte pieces: the same values from smaller pieces."""
    base = torch.randn(6 * 64 + 8, device=DEV).to(BF)
    for off in (1, 2, 4):
        x = base[off:off + 6 * 64].view(6, 64)
        assert torch.equal(group_norm(x, 4), group_norm(x.clone(), 4))


def test_same_gradients_again():
    g = gen(8)
    x, dy = randn(g, 3000, 512).to(BF).to(DEV).requires_grad_(), randn(g, 3000, 512).to(BF).to(DEV)
    w, b = torch.ones(512, device=DEV, requires_grad=True), torch.zeros(512, device=DEV, requires_grad=True)
    runs = [torch.autograd.grad(group_norm(x, 4, weight=w, bias=b), (x, w, b), dy) for _ in range(2)]
    for p, q in zip(*runs):
        assert torch.equal(p, q)


def test_no_rows():
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = group_norm(x, 4, weight=w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and (dw == 0).all()


def test_graph():
    x, dy = torch.empty(500, 256, dtype=BF, device=DEV), torch.empty(500, 256, dtype=BF, device=DEV)
    w = torch.randn(256, device=DEV)

    def step():
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        y = group_norm(leaves[0], 2, weight=leaves[1])
        return [y, *torch.autograd.grad(y, leaves, dy)]

    def fill(seed):
        g = gen(seed)
        x.copy_(randn(g, *x.shape))
        dy.copy_(randn(g, *x.shape))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2, 3):
        fill(seed)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_native_binding_and_python_functions_agree(monkeypatch):
    from dynconv import _capi

    _capi.load()
    if _capi.binding is None:
        pytest.skip("no native binding")
    g = gen(9)
    x, gate, dy = (randn(g, 30, 128).to(BF).to(DEV) for _ in range(3))
    w, b = torch.randn(128, device=DEV), torch.randn(128, device=DEV)

    def run():
        leaves = [t.detach().requires_grad_() for t in (x, w, b, gate)]
        y = group_norm(leaves[0], 4, leaves[1], leaves[2], leaves[3])
        z = group_norm(leaves[0], 4, activation=None, eps=1e-3)
        return [y, z, *torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(z, leaves[:1], dy)], y.grad_fn.name()

    a, name = run()
    monkeypatch.setattr(_capi, "binding", None)
    c, other = run()
    assert name != other and all(torch.equal(p, q) for p, q in zip(a, c))


def test_refusals():
    x = torch.randn(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    bad = [
        lambda: group_norm(x.cpu(), 4),
        lambda: group_norm(x.t(), 4),
        lambda: group_norm(x.double(), 4),
        lambda: group_norm(x, 3),
        lambda: group_norm(x, 0),
        lambda: group_norm(torch.randn(2, 4097, device=DEV), 1),
        lambda: group_norm(x, 4, weight=w[:32]),
        lambda: group_norm(x, 4, weight=w.half()),
        lambda: group_norm(x.half(), 4, weight=w.half(), bias=w),
        lambda: group_norm(x, 4, weight=w.cpu()),
        lambda: group_norm(x, 4, gate=x[:2]),
        lambda: group_norm(x, 4, gate=x.half()),
        lambda: group_norm(x, 4, activation="relu"),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError):
            f()
            pytest.fail(f"call {i} was taken")
