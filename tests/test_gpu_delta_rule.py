"""gated_delta_rule and gated_delta_rule_step against float64 (oracle/layer.py).

Bounds.  The operands of the kernels' products are rounded: bf16 once (u_r = 2^-8 of each, or better), fp16 in two bf16 parts
(2^-16), float32 and 16 bits with float32 results as float32 (2^-24, and float32 sums of up to 256 + 64 terms in chains of
chunks).
What these roundings take a result away from its float64 value depends on how far its terms cancel, so it is computed: err_r is
the error of gated_delta_rule_chunked in float32 with the same operands rounded the same way.  The kernel's roundings are
others of the same kind and number (other sums, other orders), independent and many, so their norm comes out alike: within a
factor of 3 in the norm over a tensor and of 4 in the largest norm of a row, above a floor of one rounding of an operand and
one of the result, of u_r and u_o (2^-8 bf16, 2^-11 fp16, 2^-24 float32) of everything, and 2^-18 in float32 sums:

    |a - b| <= 3 |err_r| + (u_o + u_r + 2^-18) |b| + 2^-25 sqrt(n) in fp16, whose steps end at 2^-24

With normed rows dq and dk are n (dt - t (t . dt)), the part across the row t of the gradient dt of the normed row.  Where dt lies
along t (always, with one channel) nothing is left of it but the float32 roundings of its parts: t to 3 roundings (the sum of
squares, its root, the product), twice in t (t . dt), the sum of K products in it, and the difference, under 16 2^-24 = 2^-20 of
n dt; that much of n dt is allowed besides.
"""

import pytest
import torch

from helpers import gen, randn
from linattn import gated_delta_rule, gated_delta_rule_step
from oracle.layer import gated_delta_rule_chunked, gated_delta_rule_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
UO = {BF: 2.0**-8, HF: 2.0**-11, F32: 2.0**-24}
NAMES = ("o", "state", "dq", "dk", "dv", "dlog_decay", "dbeta", "dinitial")


def _two_parts(t):
    hi = t.to(BF).to(t.dtype)
    return hi + (t - hi).to(BF).to(t.dtype)


def _rounding(dtype, wide):
    if dtype == F32 or wide:
        return (lambda t: t), 2.0**-24
    return (_two_parts, 2.0**-16) if dtype == HF else ((lambda t: t.to(BF).to(t.dtype)), 2.0**-8)


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    from dynconv import _capi

    _capi.load()
    if request.param == "python":
        monkeypatch.setattr(_capi, "binding", None)
    elif _capi.binding is None:
        pytest.skip("no native binding")


def _layout(t, layout):
    if layout == "token":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "slice":  # columns of a wider, oddly aligned tensor
        B, H, T, c = t.shape
        wide = torch.full((B, T, H * c + 7), float("nan"), dtype=t.dtype, device=t.device)
        wide[..., 3:3 + H * c] = t.transpose(1, 2).reshape(B, T, H * c)
        return wide[..., 3:3 + H * c].view(B, T, H, c).transpose(1, 2)
    return t


def _inputs(B, Hk, H, T, K, V, dtype, gdtype, normalize, seed):
    g = gen(seed + 31 * T + K)
    q, k = randn(g, B, Hk, T, K) + 0.5 * randn(g, Hk, 1, K), randn(g, B, Hk, T, K) + 0.5 * randn(g, Hk, 1, K)
    if not normalize:
        q, k = (t / t.norm(dim=-1, keepdim=True) for t in (q, k))
    lam = -torch.rand(B, H, T, generator=g) * torch.exp2(-8 * torch.rand(1, H, 1, generator=g))
    beta = torch.sigmoid(randn(g, B, H, T))
    if T > 3:
        beta[:, 0, 1] = 0.0
        beta[:, -1, 2] = 1.0
        lam[:, -1, 2] = -float("inf")
        lam[:, 0, 3] = 0.0
    v, do = randn(g, B, H, T, V), randn(g, B, H, T, V)
    return [t.to(dtype) for t in (q, k, v)] + [t.to(gdtype) for t in (lam, beta)] + [do.to(dtype)], randn(g, B, H, K, V), randn(
        g, B, H, K, V)


def _compare(got, exact, rounded, dtypes, u_r, before=None):
    along = dict(zip(("dq", "dk"), before or ()))
    for name, a, b, e in zip(NAMES, got, exact, rounded):
        if a is None or a.numel() == 0:
            continue
        a, e = a.detach().double().cpu(), e.double() - b
        assert a.shape == b.shape, name
        assert torch.isfinite(a).all(), f"{name}: not finite at {int((~torch.isfinite(a)).flatten().int().argmax())}"
        u = UO[dtypes[name]] + u_r + 2.0**-18
        floor = 2.0**-25 if dtypes[name] == HF else 1e-300
        d = a - b
        across = 2.0**-20 * along[name].norm() if name in along else 0.0
        off, most = d.norm(), 3 * e.norm() + u * b.norm() + floor * a.numel()**0.5 + across
        print(f"  {name}: {off / b.norm().clamp(min=1e-300):.2e} off, bound {most / b.norm().clamp(min=1e-300):.2e}", flush=True)
        assert off <= most, f"{name}: {off / most:.3g} times the bound"
        row = (lambda t: t.norm(dim=-1).max()) if a.dim() == 4 else (lambda t: t.abs().max())
        most = 4 * row(e) + 2 * u * row(b) + 2 * floor * a.shape[-1]**0.5 + 2 * across
        assert row(d) <= most, f"{name}: a row {row(d) / most:.3g} times the bound"


def _check(B, Hk, H, T, K, V, dtype, gates="same", layout="head", lens=None, state=True, normalize=True, seed=0, train=True):
    gdtype = dtype if gates == "same" else F32
    print(f"[delta] B{B} Hk{Hk} H{H} T{T} K{K} V{V} {dtype} {gdtype} {layout} {lens} state={state} normalize={normalize}", flush=True)
    (q, k, v, lam, beta, do), S0, dS = _inputs(B, Hk, H, T, K, V, dtype, gdtype, normalize, seed)
    scale = K**-0.5
    s0, ds = (S0, dS) if state else (None, None)
    args = (q, k, v, lam, beta, scale, do, s0, ds, lens, normalize)
    before = [] if normalize else None
    exact = gated_delta_rule_chunked(*args, before=before)
    wide = state or gdtype == F32
    r, u_r = _rounding(dtype, wide)
    rounded = gated_delta_rule_chunked(*args, dtype=F32, r=r)

    def put(t):
        t = t.clone()
        if lens is not None:
            for b, m in enumerate(lens):
                t[b, :, m:] = float("nan")
                if t.dim() == 4:
                    t[b, :, m:, ::2] = float("inf")
        return _layout(t.to(DEV), layout) if t.dim() == 4 else t.to(DEV)

    leaves = [put(t).detach().requires_grad_(train) for t in (q, k, v)]
    # gates as a projection gives them, token by token
    leaves += [put(t).transpose(1, 2).contiguous().transpose(1, 2).detach().requires_grad_(train) for t in (lam, beta)]
    if state:
        leaves.append(S0.to(DEV).requires_grad_(train))
    ld = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = gated_delta_rule(*leaves[:5], initial_state=leaves[5] if state else None, lengths=ld, return_state=state,
                           normalize=normalize)
    o = out[0] if state else out
    assert o.transpose(1, 2).is_contiguous() and o.dtype == dtype
    grads = torch.autograd.grad(out, leaves, (put(do), dS.to(DEV)) if state else put(do)) if train else (None,) * 6
    got = [o, out[1] if state else None, *grads, *([] if state else [None])]
    dt = dict.fromkeys(NAMES, dtype) | dict(state=F32, dinitial=F32, dlog_decay=gdtype, dbeta=gdtype)
    (eo, eS), eg = exact
    (ro, rS), rg = rounded
    _compare(got, (eo, eS, *eg), (ro, rS, *rg), dt, u_r, before)
    if lens is not None:
        for t in [o, *grads[:5]] if train else [o]:
            for b, m in enumerate(lens):
                assert (t[b, :, m:] == 0).all()


SIZES = [(1, 1, 1, 1, 1, 1), (1, 2, 2, 2, 3, 5), (2, 1, 2, 15, 16, 16), (1, 1, 1, 16, 33, 65), (1, 2, 4, 17, 64, 64),
         (2, 1, 1, 63, 100, 100), (1, 1, 1, 64, 128, 128), (1, 1, 3, 65, 64, 128), (1, 2, 2, 130, 128, 64),
         (1, 1, 1, 200, 256, 64), (1, 1, 1, 129, 64, 256), (1, 1, 2, 70, 256, 256), (1, 1, 1, 96, 192, 17)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_sizes(size, dtype):
    _check(*size, dtype)


@pytest.mark.parametrize("dtype,gates", [(BF, "same"), (BF, "fp32"), (HF, "same"), (HF, "fp32"), (F32, "same")])
@pytest.mark.parametrize("state,normalize", [(False, True), (False, False), (True, False)])
def test_types_without_states(dtype, gates, state, normalize):
    _check(2, 2, 4, 150, 64, 64, dtype, gates, state=state, normalize=normalize, layout="token")


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["head", "token", "slice"])
@pytest.mark.parametrize("lens", [[0, 1, 150], [64, 150, 128], [63, 65, 0]])
def test_lengths(dtype, layout, lens):
    """Rows past the lengths hold infinities and NaN."""
    _check(3, 1, 2, 150, 64, 48, dtype, layout=layout, lens=lens, state=lens[0] == 0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_heads_and_chunks(dtype):
    _check(3, 5, 10, 700, 64, 64, dtype, "same", "token", state=False)
    _check(1, 2, 2, 1537, 100, 100, dtype, "fp32", "token", state=True)


@pytest.mark.parametrize("size", [(1, 2, 2, 700, 128, 128), (3, 30, 30, 70, 128, 128), (2, 1, 1, 1100, 128, 64), (1, 4, 8, 400, 128, 96),
                                  (9, 16, 16, 20, 128, 128), (1, 1, 1, 3000, 64, 64), (2, 1, 2, 500, 256, 128)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_without_float32_results(size, dtype):
    """Tokens in segments, and workgroups of two and of four wavefronts."""
    _check(*size, dtype, state=False, lens=[size[3] - 7 * b for b in range(size[0])] if size[0] > 1 else None)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_forward_alone(dtype):
    _check(2, 2, 4, 100, 128, 128, dtype, train=False, state=False)
    _check(2, 2, 4, 100, 128, 128, dtype, train=False, state=True)


def test_no_tokens():
    S0 = torch.randn(2, 3, 8, 4, device=DEV)
    q, v = torch.randn(2, 3, 0, 8, device=DEV), torch.randn(2, 3, 0, 4, device=DEV)
    g = torch.randn(2, 3, 0, device=DEV)
    o, S = gated_delta_rule(q, q, v, g, g, initial_state=S0, return_state=True)
    assert o.shape == (2, 3, 0, 4) and torch.equal(S, S0)
    q, v, g, S0 = (t.requires_grad_() for t in (q, v, g, S0))
    _, S = gated_delta_rule(q, q, v, g, g, initial_state=S0, return_state=True)
    (d,) = torch.autograd.grad(S, S0, S0.detach())
    assert torch.equal(d, S0)


def test_an_output_that_the_loss_does_not_reach(path):
    (q, k, v, lam, beta, do), S0, dS = _inputs(1, 1, 1, 70, 32, 32, F32, F32, True, 0)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam, beta, S0)]
    for which in (0, 1):
        out = gated_delta_rule(*leaves[:5], initial_state=leaves[5], return_state=True, normalize=True)
        got = torch.autograd.grad(out[which], leaves, (do, dS)[which].to(DEV))
        zero = [do, dS]
        zero[1 - which] = torch.zeros_like(zero[1 - which])
        _, want = gated_delta_rule_chunked(q, k, v, lam, beta, 32**-0.5, zero[0], S0, zero[1], None, True)
        _, near = gated_delta_rule_chunked(q, k, v, lam, beta, 32**-0.5, zero[0], S0, zero[1], None, True, dtype=F32)
        _compare([None, None, *got], [None, None, *want], [None, None, *near], dict.fromkeys(NAMES, F32), 2.0**-24)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_one_gradient_alone(dtype, path):
    """Inputs without a gradient change nothing of the others' (bf16 in float32 results where those are asked for alone)."""
    (q, k, v, lam, beta, do), S0, _ = _inputs(1, 1, 2, 90, 32, 32, dtype, dtype, True, 11)
    ts = [t.to(DEV) for t in (q, k, v, lam, beta, S0)]
    for i in range(6):
        one = [t.clone().requires_grad_(j == i or (j == 5 and i != 5)) for j, t in enumerate(ts)]
        full = [t.clone().requires_grad_() for t in ts]
        f = lambda ls: gated_delta_rule(*ls[:5], initial_state=ls[5], normalize=True)  # noqa: E731
        (got,), (want,) = torch.autograd.grad(f(one), one[i], do.to(DEV)), torch.autograd.grad(f(full), full[i], do.to(DEV))
        assert torch.equal(got, want)


def test_expanded_inputs_and_views():
    """Heads and batches that are expanded views: their gradients are sums, by autograd."""
    (q, k, v, lam, beta, do), _, _ = _inputs(2, 2, 2, 80, 32, 32, F32, F32, False, 1)
    q1, k1, b1 = q[:, :1], k[:1], beta[:, :, :1]
    leaves = [t.to(DEV).requires_grad_() for t in (q1, k1, v, lam, b1)]
    full = [leaves[0].expand_as(q), leaves[1].expand_as(k), leaves[2], leaves[3], leaves[4].expand_as(beta)]
    got = torch.autograd.grad(gated_delta_rule(*full), leaves, do.to(DEV))
    args = (q1.expand_as(q), k1.expand_as(k), v, lam, b1.expand_as(beta), 32**-0.5, do)
    sums = (lambda g: (g[0].sum(1, True), g[1].sum(0, True), g[2], g[3], g[4].sum(2, True)))
    want, near = (sums(gated_delta_rule_chunked(*args, dtype=d)[1]) for d in (F64, F32))
    _compare([None, None, *got], [None, None, *want], [None, None, *near], dict.fromkeys(NAMES, F32), 2.0**-24)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_pieces_are_the_whole(dtype):
    """A sequence in pieces, its state handed on, and the last tokens one by one."""
    (q, k, v, lam, beta, _), S0, _ = _inputs(2, 2, 4, 150, 64, 32, dtype, F32, True, 2)
    args = [t.to(DEV) for t in (q, k, v, lam, beta)]
    with torch.no_grad():
        whole, last = gated_delta_rule(*args, initial_state=S0.to(DEV), return_state=True, normalize=True)
        S, rows = S0.to(DEV), []
        for a in (slice(0, 70), slice(70, 71), slice(71, 148)):
            o, S = gated_delta_rule(*(t[:, :, a] for t in args), initial_state=S, return_state=True, normalize=True)
            rows.append(o)
        for t in (148, 149):
            rows.append(gated_delta_rule_step(*(x[:, :, t] for x in args), S, normalize=True)[:, :, None])
    exact = gated_delta_rule_ref(q, k, v, lam, beta, 64**-0.5, S0, None, True)
    # the operands of all in two parts (or float32), carried through 150 tokens: 2^-16 of each, with the results' own rounding
    u = UO[dtype] + (2.0**-13 if dtype == BF else 2.0**-18)
    for a in (whole, torch.cat(rows, 2)):
        assert (a.double().cpu() - exact[0]).norm() <= u * exact[0].norm()
    u = 2.0**-14 if dtype == BF else 2.0**-18
    for a in (last, S):
        assert (a.double().cpu() - exact[1]).norm() <= u * exact[1].norm()


def test_runs_repeat_bit_by_bit():
    (q, k, v, lam, beta, do), S0, dS = _inputs(2, 2, 4, 300, 128, 128, BF, F32, True, 3)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam, beta, S0)]

    def once():
        out = gated_delta_rule(*leaves[:5], initial_state=leaves[5], return_state=True, normalize=True)
        return [*out, *torch.autograd.grad(out, leaves, (do.to(DEV), dS.to(DEV)))]

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_another_stream_and_two_calls_at_once():
    (q, k, v, lam, beta, do), _, _ = _inputs(1, 2, 2, 300, 64, 64, BF, BF, True, 4)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam, beta)]
    dod = do.to(DEV)
    want = torch.autograd.grad(gated_delta_rule(*leaves, normalize=True), leaves, dod)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(gated_delta_rule(*leaves, normalize=True), leaves, dod))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("state", [False, True])
def test_captured_training_step(state, path):
    """Forward and backward recorded once, replayed on new inputs with eager work between."""
    sets = [_inputs(2, 1, 2, 130, 64, 64, BF, F32 if state else BF, True, s) for s in range(3)]
    static = [t.to(DEV).requires_grad_() for t in sets[0][0][:5]]
    dod = sets[0][0][5].to(DEV)

    def step(leaves, d):
        out = gated_delta_rule(*leaves, return_state=state, normalize=True)
        o = out[0] if state else out
        return [o.detach(), *torch.autograd.grad(o, leaves, d)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, dod)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rec = step(static, dod)
    for ts, _, _ in sets * 2:
        with torch.no_grad():
            for a, b in zip(static, ts[:5]):
                a.copy_(b)
            dod.copy_(ts[5])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in rec]
        want = step([t.detach().clone().requires_grad_() for t in static], dod.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ single tokens
STEP_SIZES = [(1, 1, 1, 1, 1), (3, 1, 2, 32, 32), (2, 2, 2, 33, 65), (4, 2, 4, 64, 128), (2, 1, 1, 100, 100), (2, 3, 3, 128, 128),
              (1, 1, 2, 256, 64), (2, 1, 1, 200, 256)]


def _step_bounds(S, k, q, v, lam, beta, scale, u_o):
    """float64 results and bounds of their float32 errors: K products in each sum, 2^-24 of each term's magnitude in the
    worst case for its own rounding and for each of log2 K + 8 sums on its way (u and S enter the following sums)."""
    K = k.shape[-1]
    f = 2.0**-24 * (K**0.5 + 12)
    a = torch.exp(lam)[..., None, None]
    D = a * S
    kS, mag = (k[..., None] * D).sum(2), (k[..., None] * D).abs().sum(2)
    u = beta[..., None] * (v - kS)
    du = f * beta.abs()[..., None] * (v.abs() + mag)
    S2 = D + k[..., None] * u[:, :, None]
    dS = f * (D.abs() + (k[..., None] * u[:, :, None]).abs()) + k.abs()[..., None] * du[:, :, None]
    o = scale * (q[..., None] * S2).sum(2)
    do = abs(scale) * ((q.abs()[..., None] * dS).sum(2) + f * (q[..., None] * S2).abs().sum(2))
    do = do + abs(scale) * f * ((q[..., None] * D).abs().sum(2) + (q.abs() * k.abs()).sum(-1, keepdim=True) * u.abs())
    return o, do + u_o * o.abs(), S2, dS


@pytest.mark.parametrize("size", STEP_SIZES)
@pytest.mark.parametrize("dtype,gates", [(BF, "same"), (BF, "fp32"), (HF, "same"), (F32, "same")])
@pytest.mark.parametrize("normalize", [False, True])
def test_step(size, dtype, gates, normalize, path):
    B, Hk, H, K, V = size
    print(f"[delta step] {size} {dtype} {gates} normalize={normalize}", flush=True)
    (q, k, v, lam, beta, _), _, _ = _inputs(B, Hk, H, 4, K, V, dtype, dtype if gates == "same" else F32, normalize, 5)
    rows = B + 3
    S = randn(gen(6), rows, H, K, V)
    ids = torch.tensor([rows - 1, -1, 0, 2, rows][:B], dtype=torch.int32)
    for t in (0, 1, 2):
        x = [y[:, :, t] for y in (q, k, v, lam, beta)]
        Sd = S.to(DEV)
        with torch.no_grad():
            o = gated_delta_rule_step(*(y.to(DEV) for y in x), Sd, slots=ids.to(DEV), normalize=normalize)
        qd, kd, vd, ld, bd = (y.double() for y in x)
        if normalize:
            qd, kd = (y / torch.sqrt((y * y).sum(-1, keepdim=True) + 1e-6) for y in (qd, kd))
        qd, kd = (y.repeat_interleave(H // Hk, 1) for y in (qd, kd))
        want = S.double()
        for b, slot in enumerate(ids.tolist()):
            if not 0 <= slot < rows:
                assert (o[b] == 0).all()
                continue
            one = slice(b, b + 1)
            eo, do, eS, dS = _step_bounds(want[slot][None], kd[one], qd[one], vd[one], ld[one], bd[one], K**-0.5, UO[dtype])
            assert ((o[b].double().cpu() - eo[0]).abs() <= do[0] + (2.0**-25 if dtype == HF else 1e-300)).all()
            assert ((Sd[slot].double().cpu() - eS[0]).abs() <= dS[0] + 1e-300).all()
            want[slot] = Sd[slot].double().cpu()
        untouched = [r for r in range(rows) if r not in ids.tolist()]
        assert torch.equal(Sd.cpu()[untouched], S[untouched])
        S = Sd.cpu()


def test_step_in_a_cache_past_32_bit_offsets():
    H, K, V = 16, 128, 128
    rows = 2**31 // (H * K * V) + 3
    S = torch.zeros(rows, H, K, V, device=DEV)
    (q, k, v, lam, beta, _), _, _ = _inputs(2, H, H, 1, K, V, BF, F32, True, 7)
    x = [t[:, :, 0].to(DEV) for t in (q, k, v, lam, beta)]
    o = gated_delta_rule_step(*x, S, slots=torch.tensor([rows - 1, 0], device=DEV), normalize=True)
    S2 = torch.zeros(2, H, K, V, device=DEV)
    o2 = gated_delta_rule_step(*x, S2, normalize=True)
    assert torch.equal(o, o2) and torch.equal(S[rows - 1], S2[0]) and torch.equal(S[0], S2[1])
    assert S[1:rows - 1].abs().max() == 0


def test_captured_decoding(path):
    """A step recorded once and replayed moves the states as eager steps do."""
    (q, k, v, lam, beta, _), S0, _ = _inputs(3, 2, 2, 6, 64, 64, BF, F32, True, 8)
    args = [t.to(DEV) for t in (q, k, v, lam, beta)]
    static = [t[:, :, 0].clone() for t in args]
    S, E = S0.to(DEV), S0.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        gated_delta_rule_step(*static, S.clone(), normalize=True)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            o = gated_delta_rule_step(*static, S, normalize=True)
        for t in range(6):
            for a, b in zip(static, args):
                a.copy_(b[:, :, t])
            graph.replay()
            want = gated_delta_rule_step(*(b[:, :, t] for b in args), E, normalize=True)
            torch.cuda.synchronize()
            assert torch.equal(o, want) and torch.equal(S, E)


# ------------------------------------------------------------------------------------------------ refusals
def _bad(q=(2, 2, 8, 16), k=None, v=(2, 4, 8, 32), g=(2, 4, 8), dt=BF, gd=F32, bd=None, **kw):
    n = lambda s, d: torch.zeros(s, dtype=d, device=DEV)  # noqa: E731
    return gated_delta_rule(n(q, dt), n(k or q, dt), n(v, dt), n(g, gd), n(g, bd or gd), **kw)


def test_refusals(path):
    assert _bad().shape == (2, 4, 8, 32)
    for kw in (dict(v=(2, 3, 8, 32), g=(2, 3, 8)), dict(k=(2, 2, 8, 17)), dict(v=(2, 4, 9, 32)), dict(g=(2, 2, 8)), dict(g=(2, 4, 9)),
               dict(q=(2, 2, 8, 257)), dict(v=(2, 4, 8, 257)), dict(dt=torch.float64), dict(gd=HF), dict(bd=BF), dict(dt=HF, gd=BF),
               dict(initial_state=torch.zeros(2, 4, 16, 32, device=DEV, dtype=BF)), dict(lengths=torch.zeros(3, device=DEV).int()),
               dict(initial_state=torch.zeros(2, 4, 32, 16, device=DEV)), dict(lengths=torch.zeros(2).int())):
        with pytest.raises(AssertionError):
            _bad(**kw)
    with pytest.raises(AssertionError):
        gated_delta_rule(*(torch.zeros(1, 1, 2, 4) for _ in range(3)), torch.zeros(1, 1, 2), torch.zeros(1, 1, 2))


def test_step_refusals(path):
    n = lambda *s, d=BF: torch.zeros(s, dtype=d, device=DEV)  # noqa: E731
    ok = dict(q=n(2, 2, 16), k=n(2, 2, 16), v=n(2, 4, 32), log_decay=n(2, 4), beta=n(2, 4), state=n(2, 4, 16, 32, d=F32))
    assert gated_delta_rule_step(**ok).shape == (2, 4, 32)
    for kw in (dict(state=n(1, 4, 16, 32, d=F32)), dict(state=n(2, 4, 16, 32)), dict(state=n(2, 4, 32, 16, d=F32).transpose(2, 3)),
               dict(beta=n(2, 4, d=F32)), dict(k=n(2, 2, 17)), dict(v=n(2, 3, 32)), dict(slots=n(3, d=torch.int32)),
               dict(q=n(2, 2, 16).requires_grad_())):
        with pytest.raises(AssertionError):
            gated_delta_rule_step(**{**ok, **kw})


def test_a_step_makes_the_backward_of_what_saved_its_state_raise(path):
    (q, k, v, lam, beta, _), S0, _ = _inputs(2, 2, 2, 40, 32, 32, F32, F32, True, 9)
    q, k, v, lam, beta, S = (t.to(DEV) for t in (q, k, v, lam, beta, S0))
    q.requires_grad_()
    o = gated_delta_rule(q, k, v, lam, beta, initial_state=S)
    with torch.no_grad():
        gated_delta_rule_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lam[:, :, 0], beta[:, :, 0], S)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
