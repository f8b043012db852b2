"""residual_norm against float64 (oracle/layer.py).

Bounds, by entry, of float32 arithmetic on D channels and one rounding of each result.  A sum of D squares or products in
float32, by lanes and then in trees, is within (D / 256 + 24) 2^-24 of the sum of its terms' magnitudes; a row's factor 1/rms
within half of that and two roundings.  With f = 2^-24 (D / 128 + 32) and u_o a rounding of the result (2^-8 bf16, 2^-11 fp16,
2^-24 float32):

  h        f (|x| + |u|) + u_x |h|
  y        (f + u_o) |y|, and twice the rounding of h (once itself, once through the row's rms): 2 u_x (|y| + rms(y) |w|)
  dx       its terms |dh| + rh (|dy w| + |h| rh^2 mean|dy w h|), f and, for h's rounding, 2 u_x of the last two; then u_x |dx|
  dbranch  its terms with |dx| replaced by |dx| and its bound; then u_o
  dgate    |n scale act'| times dx's bound, f, u_o
  sums     over rows, of their terms' bounds; f' = 2^-24 (M / 64 + 32) for the sums themselves; then u_o
"""

import pytest
import torch

from helpers import gen, randn
from linattn import residual_norm
from oracle.layer import residual_norm_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0**-8, HF: 2.0**-11, F32: 2.0**-24}


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    from dynconv import _capi

    _capi.load()
    if request.param == "python":
        monkeypatch.setattr(_capi, "binding", None)
    elif _capi.binding is None:
        pytest.skip("no native binding")


def _act(a, name):
    s = 1 / (1 + torch.exp(-a))
    return {"silu": (a * s, s * (1 + a * (1 - s))), "sigmoid": (s, s * (1 - s)), None: (a, torch.ones_like(a))}[name]


def _bounds(x, br, w, bw, a, act, sc, dy, dh, eps, u_o, u_x, u_p):
    D, M = x.shape[-1], x.numel() // x.shape[-1]
    f, fm = 2.0**-24 * (D / 128 + 32), 2.0**-24 * (M / 64 + 32)
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    rb = 1 / torch.sqrt(mean(br * br) + eps)
    n = br * rb * bw
    F, dF = _act(a, act) if a is not None else (torch.ones_like(n), torch.zeros_like(n))
    u = n * F * sc
    h = x + u
    rh = 1 / torch.sqrt(mean(h * h) + eps)
    y = h * rh * w
    th = f * (x.abs() + u.abs()) + u_x * h.abs()
    ty = (2 * f + u_o) * y.abs() + 2 * u_x * (y.abs() + torch.sqrt(mean(y * y)) * w.abs())
    p, m = rh * (dy * w).abs(), h.abs() * rh**3 * mean((dy * w * h).abs())
    dx = dh + rh * (dy * w) - h * rh**3 * mean(dy * w * h)
    tdx = 2 * f * (dh.abs() + p + m) + 2 * u_x * (p + 2 * m)
    g = lambda t: rb * ((t * F * sc * bw).abs() + br.abs() * rb**2 * mean((t * F * sc * bw * br).abs()))  # noqa: E731
    db = rb * (dx * F * sc * bw - br * rb**2 * mean(dx * F * sc * bw * br))
    tdb = g(tdx) + 2 * f * g(dx) + u_o * db.abs()
    dg, tdg = dx * n * sc * dF, (tdx + 2 * f * dx.abs()) * (n * sc * dF).abs() + 2.0**-22 * (dx * n * sc).abs()
    over = lambda t: t.reshape(M, D).sum(0)  # noqa: E731
    dw = over(dy * h * rh)
    tdw = over((2 * f + fm + 2 * u_x) * (dy * h * rh).abs() + 2 * u_x * (dy * rh).abs() * torch.sqrt(mean(h * h))) + u_p * dw.abs()
    dbw = over(dx * F * sc * br * rb)
    tdbw = over((tdx + (2 * f + fm) * dx.abs()) * (F * sc * br * rb).abs()) + u_p * dbw.abs()
    ds = over(dx * n * F)
    tds = over((tdx + (2 * f + fm) * dx.abs()) * (n * F).abs()) + u_p * ds.abs()
    return (y, h, dx, db, dw, dbw, dg, ds), (ty, th, tdx + u_x * dx.abs(), tdb, tdw, tdbw, tdg + u_o * dg.abs(), tds)


def _check(shape, dtype, xdtype=None, pdtype=None, act=None, gate=True, params="wbs", constant=None, seed=0, offset=0, grads="yh"):
    xdtype, pdtype, D = xdtype or dtype, pdtype or dtype, shape[-1]
    print(f"[residual] {shape} {dtype} x {xdtype} params {pdtype} {act} gate={gate} {params} offset={offset} {grads}", flush=True)
    g = gen(seed + D)
    ts = dict(x=randn(g, *shape, scale=4.0).to(xdtype), branch=randn(g, *shape, scale=0.5).to(dtype))
    ts["weight"] = (1 + 0.1 * randn(g, D)).to(pdtype) if "w" in params else None
    ts["branch_weight"] = (1 + 0.1 * randn(g, D)).to(pdtype) if "b" in params else None
    ts["gate"] = randn(g, *shape).to(dtype) if gate else None
    ts["scale"] = (0.3 * randn(g, D)).to(pdtype) if "s" in params else None
    dy, dh = randn(g, *shape).to(dtype), randn(g, *shape).to(xdtype)

    def put(t):
        if t is None:
            return None
        if not offset or t.dim() == 1:
            return t.to(DEV)
        flat = torch.full((t.numel() + offset,), float("nan"), dtype=t.dtype, device=DEV)
        flat[offset:] = t.flatten().to(DEV)
        return flat[offset:].view(t.shape)

    d = {k: put(t) for k, t in ts.items()}
    leaves = {k: t.detach().requires_grad_() for k, t in d.items() if t is not None}
    args = {**d, **leaves}
    if constant is not None:
        args["scale"] = constant
    y, h = residual_norm(**args, activation=act)
    assert y.dtype == dtype and h.dtype == xdtype
    outs, douts = zip(*[(o, put(t)) for o, t, n in ((y, dy, "y"), (h, dh, "h")) if n in grads])
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), douts, allow_unused=True)))

    one = torch.ones(D, dtype=torch.float64)
    f64 = {k: (None if t is None else t.double()) for k, t in ts.items()}
    sc = f64["scale"] if f64["scale"] is not None else one * (1.0 if constant is None else constant)
    want, tol = _bounds(f64["x"], f64["branch"], one if f64["weight"] is None else f64["weight"],
                        one if f64["branch_weight"] is None else f64["branch_weight"], f64["gate"], act, sc,
                        dy.double() * ("y" in grads), dh.double() * ("h" in grads), 1e-6, U[dtype], U[xdtype], U[pdtype])
    ry, rh = residual_norm_ref(f64["x"], f64["branch"], f64["weight"], f64["branch_weight"], f64["gate"], act, sc)
    assert torch.allclose(ry, want[0]) and torch.allclose(rh, want[1])
    named = dict(zip(("y", "h", "x", "branch", "weight", "branch_weight", "gate", "scale"), zip(want, tol)))
    for k, a in {"y": y, "h": h, **got}.items():
        b, t = named[k]
        if a is None:  # nothing of the loss reached it
            assert k == "weight" and "y" not in grads
            continue
        sub = 2.0**-25 if a.dtype == HF else 1e-300
        r = ((a.detach().double().cpu() - b).abs() / (t + sub)).nan_to_num(nan=float("inf"))
        assert r.max() <= 1, f"{k}: {r.max().item():.3g} times the bound at {int(r.argmax())}"


DIMS = [1, 2, 7, 8, 63, 64, 100, 512, 513, 1000, 1024, 1025, 1032, 2048, 4096, 4100, 8191, 8192]


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_sizes(D, dtype):
    _check((5, D), dtype, act="silu")


@pytest.mark.parametrize("dtype,xdtype,pdtype", [(BF, F32, BF), (BF, BF, F32), (HF, F32, F32), (BF, F32, F32), (HF, HF, HF)])
@pytest.mark.parametrize("D", [100, 1000, 2048, 5000])
def test_types(dtype, xdtype, pdtype, D):
    _check((2, 9, D), dtype, xdtype, pdtype, act="sigmoid")


@pytest.mark.parametrize("act,gate", [(None, False), (None, True), ("silu", True), ("sigmoid", True)])
@pytest.mark.parametrize("params", ["", "w", "b", "s", "wbs"])
def test_optional_inputs(act, gate, params, path):
    _check((3, 7, 192), BF, act=act, gate=gate, params=params)
    _check((2, 1536), F32, act=act, gate=gate, params=params)


def test_a_number_as_scale(path):
    _check((33, 256), BF, gate=False, params="wb", constant=0.25)
    _check((33, 256), F32, act="silu", params="", constant=-2.0)


@pytest.mark.parametrize("grads", ["y", "h"])
def test_one_output_alone(grads, path):
    _check((6, 320), BF, act="silu", grads=grads)


@pytest.mark.parametrize("rows", [1, 3, 1023, 5000])
@pytest.mark.parametrize("D", [64, 1056])
def test_rows(rows, D):
    _check((rows, D), BF, F32, act="silu")


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_alignment(offset):
    _check((9, 256), BF, act="silu", offset=offset)
    _check((9, 2048), BF, F32, act="silu", offset=offset)


@pytest.mark.parametrize("wanted", ["x", "branch", "weight", "branch_weight", "gate", "scale"])
def test_one_gradient_alone(wanted, path):
    """Inputs without a gradient change nothing of the others'."""
    g = gen(3)
    ts = dict(x=randn(g, 9, 192), branch=randn(g, 9, 192), weight=randn(g, 192), branch_weight=randn(g, 192), gate=randn(g, 9, 192),
              scale=randn(g, 192))
    ts = {k: t.to(BF).to(DEV) for k, t in ts.items()}
    dy, dh = (randn(g, 9, 192).to(BF).to(DEV) for _ in range(2))
    both = {k: t.clone().requires_grad_() for k, t in ts.items()}
    (want,) = torch.autograd.grad(residual_norm(**both, activation="silu"), both[wanted], (dy, dh))
    one = {k: t.clone().requires_grad_(k == wanted) for k, t in ts.items()}
    (got,) = torch.autograd.grad(residual_norm(**one, activation="silu"), one[wanted], (dy, dh))
    assert torch.equal(got, want)


def test_no_rows(path):
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, h = residual_norm(x, x, weight=w, branch_weight=w)
    assert y.shape == h.shape == (0, 64)
    dx, dw = torch.autograd.grad((y, h), (x, w), (y, h))
    assert dx.shape == (0, 64) and (dw == 0).all()


def test_runs_repeat_bit_by_bit():
    g = gen(1)
    x, b, a, dy, dh = (randn(g, 3000, 640).to(BF).to(DEV) for _ in range(5))
    w = (1 + 0.1 * randn(g, 640)).to(BF).to(DEV)
    leaves = [t.requires_grad_() for t in (x, b, w, a)]

    def once():
        out = residual_norm(x, b, weight=w, branch_weight=w, gate=a, activation="silu", scale=w)
        return [*out, *torch.autograd.grad(out, leaves, (dy, dh))]

    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


def test_captured_step(path):
    g = gen(2)
    sets = [[randn(g, 40, 1100).to(BF).to(DEV) for _ in range(5)] for _ in range(3)]
    static = [t.clone() for t in sets[0]]
    w = (1 + 0.1 * randn(g, 1100)).to(BF).to(DEV).requires_grad_()

    def step(x, b, a, dy, dh):
        x, b, a = (t.detach().requires_grad_() for t in (x, b, a))
        out = residual_norm(x, b, weight=w, branch_weight=w, gate=a, activation="silu")
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (x, b, w, a), (dy, dh))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rec = step(*static)
    for ts in sets * 2:
        for a, b in zip(static, ts):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in rec]
        want = step(*static)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(path):
    n = lambda *s, d=BF: torch.zeros(s, dtype=d, device=DEV)  # noqa: E731
    ok = dict(x=n(4, 64), branch=n(4, 64), weight=n(64))
    assert residual_norm(**ok)[0].shape == (4, 64)
    for kw in (dict(x=n(4, 64, d=HF)), dict(x=n(64, 4).t()), dict(branch=n(4, 65)), dict(branch=n(8, 64)[::2]), dict(weight=n(63)),
               dict(weight=n(64, d=HF)), dict(scale=n(64, d=F32)), dict(gate=n(4, 63)), dict(gate=n(4, 64, d=F32)),
               dict(activation="silu"), dict(activation="relu", gate=n(4, 64)), dict(branch=n(4, 64, d=F32)),
               dict(x=n(1, 8193), branch=n(1, 8193), weight=None), dict(x=torch.zeros(4, 64, dtype=BF))):
        with pytest.raises(AssertionError):
            residual_norm(**{**ok, **kw})
