"""lowrank_dynamic_convolution_step(_grouped) against float64 (oracle/layer.py) and the whole-sequence operator.

The step's products and sums are float32 on the inputs' values, so an output is off by its rounding (2^-8 bf16, 2^-11
fp16, 2^-24 fp32) and by 2^-20 of the magnitudes of its W (R + 1) + 1 terms; the state moves whole."""

import pytest
import torch

from helpers import gen, randn
from lowrank import (lowrank_dynamic_convolution, lowrank_dynamic_convolution_step,
                     lowrank_dynamic_convolution_step_grouped)
from oracle.layer import lowrank_step_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(g, G, N, D, R, W, static, rows, dtype):
    x = randn(g, N, G * D).to(dtype)
    z = [randn(g, N, R).to(dtype) for _ in range(G)]
    U = [randn(g, R, W * D, scale=(R * W) ** -0.5).to(dtype) for _ in range(G)]
    sw = [randn(g, W, D, scale=0.4).to(dtype) for _ in range(G)] if static else None
    return x, z, U, sw, randn(g, rows, W - 1, G * D).to(dtype)


def _dev(t):
    return None if t is None else [a.to(DEV) for a in t] if isinstance(t, list) else t.to(DEV)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("G,N,D,R,W,static,residual", [
    (1, 1, 256, 16, 4, False, True), (3, 8, 256, 15, 4, True, True), (2, 9, 130, 7, 3, True, False),
    (4, 3, 65, 1, 1, True, True), (1, 21, 33, 8, 2, False, False), (3, 17, 512, 31, 4, True, True),
    (1, 5, 200, 64, 16, False, True), (2, 40, 128, 127, 9, True, True), (1, 300, 64, 4, 5, False, True),
    (1, 33, 136, 256, 2, False, True), (2, 70, 128, 63, 3, True, True)])
def test_step(G, N, D, R, W, static, residual, dtype):
    print(f"[step] G{G} N{N} D{D} R{R} W{W} static={static} {dtype}", flush=True)
    g = gen(G + N + D + W)
    rows = N + 3
    x, z, U, sw, state = _inputs(g, G, N, D, R, W, static, rows, dtype)
    ids = torch.randperm(rows, generator=g)[:N]
    if N > 2:
        ids[1], ids[N - 1] = -1, rows  # take no part
    free = [r for r in range(rows) if r not in ids.tolist()]
    state[free] = float("nan")
    before = state.clone()
    dstate = state.to(DEV)
    ys = lowrank_dynamic_convolution_step_grouped(_dev(x), _dev(z), _dev(U), dstate, static_w=_dev(sw),
                                                  residual=residual, slots=ids.to(torch.int32).to(DEV))
    dstate = dstate.cpu()
    assert torch.isnan(dstate[free]).all() if W > 1 and free else True
    live = [n for n in range(N) if 0 <= ids[n] < rows]
    rnd = {BF: 2.0**-8, HF: 2.0**-11, F32: 2.0**-24}[dtype]
    for h in range(G):
        c = slice(h * D, (h + 1) * D)
        s = before[ids[live]][..., c]
        args = (x[live][:, c], z[h][live], U[h], s, None if sw is None else sw[h], residual)
        y, new = lowrank_step_ref(*args)
        terms, _ = lowrank_step_ref(*[t.abs() if isinstance(t, torch.Tensor) else t for t in args])
        got = ys[h].double().cpu()
        assert ((got[live] - y).abs() <= 1.01 * rnd * y.abs() + 2.0**-20 * terms + (2.0**-25 if dtype == HF else 0)).all()
        assert torch.equal(dstate[ids[live]][..., c].double(), new)
        out = [n for n in range(N) if n not in live]
        assert (got[out] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("R,W,static", [(15, 4, True), (8, 1, False), (31, 5, True), (63, 9, True), (128, 3, False),
                                        (256, 2, False)])
def test_many_workgroups(R, W, static, dtype):
    """Sizes past those that split the taps over a workgroup's wavefronts."""
    N, D = (300, 2568) if dtype == F32 else (70, 2824)
    test_step(1, N, D, R, W, static, True, dtype)


@pytest.mark.parametrize("D", [128, 33, 8448])
def test_sequences_that_take_no_part_may_hold_anything(D):
    g = gen(30)
    x, z, U, _, state = _inputs(g, 1, 5, D, 8, 3, False, 5, BF)
    x[2], z[0][2], x[4], z[0][4] = float("nan"), float("nan"), float("inf"), float("inf")
    ids = torch.tensor([0, 1, -1, 3, 5], dtype=torch.int32, device=DEV)
    y, = lowrank_dynamic_convolution_step_grouped(_dev(x), _dev(z), _dev(U), _dev(state), slots=ids)
    assert (y[[2, 4]] == 0).all() and y.isfinite().all()


def test_steps_follow_the_whole_sequence():
    g = gen(31)
    N, T, D, R, W = 3, 11, 96, 7, 4
    x, z = randn(g, N, T, D).to(DEV), randn(g, N, T, R).to(DEV)
    U, sw = randn(g, R, W * D, scale=0.2).to(DEV), randn(g, W, D).to(DEV)
    whole = lowrank_dynamic_convolution(x, z, U, static_w=sw, residual=True)
    state = torch.zeros(N, W - 1, D, device=DEV)
    for t in range(T):
        y = lowrank_dynamic_convolution_step(x[:, t].contiguous(), z[:, t].contiguous(), U, state, static_w=sw, residual=True)
        torch.testing.assert_close(y, whole[:, t], rtol=1e-5, atol=1e-5)
    assert torch.equal(state, x[:, T - W + 1:])


def test_step_in_a_cache_past_32_bits():
    rows, D, W = 70000, 4096, 4
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 6 GiB of GPU memory")
    x, z, U, sw, first = (_dev(t) for t in _inputs(gen(36), 3, 3, D, 7, W, True, 3, BF))
    state = torch.empty(rows, W - 1, 3 * D, dtype=BF, device=DEV)
    ids = torch.tensor([rows - 1, 60000, 2], dtype=torch.int32, device=DEV)
    state[ids.long()] = first
    small = first.clone()
    a = lowrank_dynamic_convolution_step_grouped(x, z, U, state, static_w=sw, slots=ids)
    b = lowrank_dynamic_convolution_step_grouped(x, z, U, small, static_w=sw)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(state[ids.long()], small)


def test_wide_rows_and_unaligned_tensors():
    """x as columns of a wider tensor, and starting off the pairs: the values of contiguous ones."""
    g = gen(32)
    x, z, U, sw, state = (_dev(t) for t in _inputs(g, 2, 6, 64, 7, 4, True, 6, BF))
    want_state = state.clone()
    want = lowrank_dynamic_convolution_step_grouped(x, z, U, want_state, static_w=sw)
    for off in (2, 3):
        wide = torch.full((6, 160), float("nan"), dtype=BF, device=DEV)
        wide[:, off:off + 128] = x
        s = state.clone()
        got = lowrank_dynamic_convolution_step_grouped(wide[:, off:off + 128], z, U, s, static_w=sw)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(s, want_state)


def test_graph():
    x, z, U, sw, state = (_dev(t) for t in _inputs(gen(33), 3, 4, 64, 15, 4, True, 4, BF))

    def step():
        return lowrank_dynamic_convolution_step_grouped(x, z, U, state, static_w=sw, residual=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2, 3):
        new, first = randn(gen(seed), *x.shape).to(BF).to(DEV), state.clone()
        x.copy_(new)
        want, end = [y.clone() for y in step()], state.clone()
        state.copy_(first)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(state, end)


def test_native_binding_and_python_function_agree(monkeypatch):
    from dynconv import _capi

    _capi.load()
    x, z, U, sw, state = (_dev(t) for t in _inputs(gen(35), 2, 6, 64, 7, 4, True, 9, HF))
    ids = torch.tensor([8, 1, -1, 3, 0, 5], dtype=torch.int32, device=DEV)

    def run():
        s = state.clone()
        return [*lowrank_dynamic_convolution_step_grouped(x, z, U, s, static_w=sw, residual=True, slots=ids), s]

    a = run()
    monkeypatch.setattr(_capi, "binding", None)
    assert all(torch.equal(p, q) for p, q in zip(a, run()))


def test_refusals():
    x, z, U, sw, state = (_dev(t) for t in _inputs(gen(34), 2, 3, 64, 7, 4, True, 3, BF))
    step = lowrank_dynamic_convolution_step_grouped
    bad = [
        lambda: step(x.cpu(), z, U, state, sw),
        lambda: step(x[:, :127], z, U, state, sw),
        lambda: step(x, z[:1], U, state, sw),
        lambda: step(x, z, U, state, None),           # rank 7 without a static filter
        lambda: step(x, z, U, state[:, :2].contiguous(), sw),
        lambda: step(x, z, U, state[:2], sw),         # more sequences than rows
        lambda: step(x, z, U, state.float(), sw),
        lambda: step(x, z, U, state.transpose(0, 1), sw),
        lambda: step(x, [t[:2] for t in z], U, state, sw),
        lambda: step(x, z, [t[:, :100].contiguous() for t in U], state, sw),
        lambda: step(x, z, U, state, [t[:2] for t in sw]),
        lambda: step(x, z, U, state, sw, slots=torch.zeros(2, dtype=torch.int32, device=DEV)),
        lambda: step(x.clone().requires_grad_(), z, U, state, sw),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError):
            f()
            pytest.fail(f"call {i} was taken")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [128, 33, 25088])
def test_sequences_that_take_no_part_are_zero_whatever_the_filters_hold(D, dtype):
    x, z, U, sw, state = _inputs(gen(37), 1, 5, D, 7, 3, True, 5, dtype)
    U[0][3] = float("inf")
    U[0][5, ::2] = float("nan")
    sw[0][1] = float("-inf")
    before = state.clone()
    ids = torch.tensor([0, 1, -1, 3, 5], dtype=torch.int32, device=DEV)
    dstate = _dev(state)
    y, = lowrank_dynamic_convolution_step_grouped(_dev(x), _dev(z), _dev(U), dstate, static_w=_dev(sw), slots=ids)
    assert (y[[2, 4]] == 0).all() and not y[[0, 1, 3]].isfinite().any()
    assert torch.equal(dstate[[2, 4]].cpu(), before[[2, 4]])
