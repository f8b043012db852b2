"""linear_attention and linear_attention_step against float64 recurrences (oracle/layer.py).

Bounds, per entry, against the value b in float64 from the same inputs:

    |a - b| <= 4 u E + f (N + |b|) + r |b| + floor

  E, u  An output is a sum of products whose one factor is rounded to the inputs' type before the matrix product: a
        decayed score p_ij (times v_j), or an entry of the state (times q).  Rounding moves a factor x by at most
        u |x| (u = 2^-8 bf16, 2^-11 fp16, 0 in fp32), with a standard deviation below u |x| / sqrt(3), independently
        from factor to factor, so E = sqrt(sum of the squared products) and 4 u E is over 6 standard deviations.  The
        state's products are bounded by q's squares times the largest square the state's entry has had.  The state
        itself is a sum of products whose one factor is kept in two parts of the type (u = 2^-16, 2^-22).
  f, N  float32 sums and decays: N is the norm of the same products, and f = 2^-24 (16 + T / 2) allows a rounding of
        the carried decay at every token.
  r     the rounding of an output: u in 16 bits, a last place in float32.
  floor fp16's smallest step, 2^-24, for each rounded factor: 4 * 2^-25 * the norm of the other factors.
"""

import pytest
import torch

from helpers import gen, randn
from linattn import linear_attention, linear_attention_step
from oracle.layer import linear_attention_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0**-8, HF: 2.0**-11, F32: 0.0}
U2 = {BF: 2.0**-16, HF: 2.0**-22, F32: 0.0}


def _decays(H, seed):
    """Weak and strong decays, none, and one that forgets at once."""
    g = gen(seed)
    lam = torch.log1p(-torch.exp2(-(0.5 + 9 * torch.rand(H, generator=g))))
    if H > 2:
        lam[1] = 0.0
        lam[2] = -float("inf")
    return lam


def _rows_live(t, n):
    t = t.detach().double().clone()
    for b, m in enumerate(n):
        t[b, :, m:] = 0
    return t


def _norms(q, k, v, lam, s_in, so, skv, lens, rev, dtype):
    """(tolerance of o, tolerance of the final state) of one pass of the recurrence, E and N above, float64."""
    B, H, T, K = q.shape
    q, k, v = (_rows_live(t, lens) for t in (q, k, v))
    if rev:
        # against time: each sequence turned over within its length
        def turn(t):
            return torch.stack([torch.cat([t[b, :, :m].flip(1), t[b, :, m:]], 1) for b, m in enumerate(lens)])
        q, k, v = turn(q), turn(k), turn(v)
    g = torch.exp(lam.double())[None, :, None, None]
    V = v.shape[-1]
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if s_in is None else s_in.double().clone()
    top, sq, fl = S.abs(), (S * S), torch.zeros(B, H, 1, V, dtype=torch.float64)
    P = torch.zeros(B, H, 1, V, dtype=torch.float64)
    out = []
    pairs = torch.tril(torch.ones(T, T, dtype=torch.float64))
    gap = (torch.arange(T)[:, None] - torch.arange(T)[None]).clamp(min=0).double()
    w = torch.where(gap[None] == 0, torch.ones(()).double(), torch.exp(lam.double()[:, None, None] * gap.clamp(min=1e-9)))
    p = (q @ k.transpose(2, 3)) * w[None] * pairs * so * skv
    E2 = (p * p) @ (v * v)
    for t in range(T):
        S = (S if (rev and t == 0) else g * S) + skv * k[:, :, t, :, None] * v[:, :, t, None, :]
        sq = g * g * sq + skv * skv * (k[:, :, t, :, None] * v[:, :, t, None, :]) ** 2
        top = torch.maximum(top, S.abs())
        qt = q[:, :, t, :, None] * so
        out.append(((qt * qt) * top * top).sum(2))
    ES = torch.stack(out, 2) if T else torch.zeros_like(v)
    E = torch.sqrt(E2 + ES)
    f = 2.0**-24 * (16 + T / 2)
    tol = 4 * U[dtype] * E + f * E
    stol = 4 * U2[dtype] * torch.sqrt(sq) + f * (torch.sqrt(sq) + top)
    if dtype == HF:
        tol = tol + 4 * 2.0**-25 * (torch.sqrt((v * v).cumsum(2)) + so * q.norm(dim=-1, keepdim=True))
        stol = stol + 4 * 2.0**-25 * torch.sqrt((v * v).sum(2, keepdim=True))
    if rev:
        tol = torch.stack([torch.cat([tol[b, :, :m].flip(1), tol[b, :, m:]], 1) for b, m in enumerate(lens)])
    return tol, stol, f


def _close(a, b, tol, dtype, f, name):
    a = a.detach().double().cpu()
    r = {BF: 2.0**-8, HF: 2.0**-11, F32: 2.0**-23}[dtype]
    bound = tol + (f + r) * b.abs() + (2.0**-25 if dtype == HF else 0) + 1e-300
    assert a.shape == b.shape, f"{name}: {tuple(a.shape)}"
    ratio = ((a - b).abs() / bound).nan_to_num(nan=float("inf"))
    assert ratio.numel() == 0 or ratio.max() <= 1, f"{name}: {ratio.max().item():.3g} times the bound at {int(ratio.argmax())}"


def _check(B, H, T, K, V, dtype, layout="head", lens=None, state=True, seed=0, poison=True):
    print(f"[linattn] B{B} H{H} T{T} K{K} V{V} {dtype} {layout} {lens} state={state}", flush=True)
    g = gen(seed + 31 * T + K)
    n = [T] * B if lens is None else lens
    scale = K**-0.5
    lam = _decays(H, seed)

    def heads(c):
        t = randn(g, B, H, T, c).to(dtype)
        if lens is not None and poison:
            for b, m in enumerate(n):
                t[b, :, m:] = float("nan")
                t[b, :, m:, ::2] = float("inf")
        d = t.to(DEV)
        if layout == "token":
            d = d.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "slice":  # columns of a wider, oddly aligned tensor
            wide = torch.full((B, T, H * c + 7), float("nan"), dtype=dtype, device=DEV)
            wide[..., 3:3 + H * c] = d.transpose(1, 2).reshape(B, T, H * c)
            d = wide[..., 3:3 + H * c].view(B, T, H, c).transpose(1, 2)
        return t, d

    (q, qd), (k, kd), (v, vd), (do, dod) = heads(K), heads(K), heads(V), heads(V)
    S0 = randn(g, B, H, K, V) if state else None
    dS = randn(g, B, H, K, V) if state else None
    leaves = [t.detach().requires_grad_() for t in (qd, kd, vd)] + ([S0.to(DEV).requires_grad_()] if state else [])
    ld = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = linear_attention(*leaves[:3], lam.to(DEV), initial_state=leaves[3] if state else None, lengths=ld,
                           return_state=state)
    o = out[0] if state else out
    grads = torch.autograd.grad(out, leaves, (dod, dS.to(DEV)) if state else dod)
    assert o.transpose(1, 2).is_contiguous()

    ref = [t.double().requires_grad_() for t in (q, k, v)] + ([S0.double().requires_grad_()] if state else [])
    ro, rS = linear_attention_ref(*ref[:3], lam, scale, ref[3] if state else None, n)
    dref = _rows_live(do, n)
    rg = torch.autograd.grad((ro, rS), ref, (dref, dS.double() if state else torch.zeros_like(rS)), allow_unused=True)
    rg = [torch.zeros_like(r) if x is None else x for x, r in zip(rg, ref)]

    ds = None if dS is None else dS.double()
    tol, stol, f = _norms(q, k, v, lam, S0, scale, 1.0, n, False, dtype)
    _close(o, ro.detach(), tol, dtype, f, "o")
    if state:
        _close(out[1], rS.detach(), stol, F32, f, "state")
    tol, _, f = _norms(do, v, k, lam, None if S0 is None else S0.transpose(2, 3), scale, 1.0, n, False, dtype)
    _close(grads[0], rg[0], tol, dtype, f, "dq")
    tol, _, f = _norms(v, do, q, lam, None if ds is None else ds.transpose(2, 3), 1.0, scale, n, True, dtype)
    _close(grads[1], rg[1], tol, dtype, f, "dk")
    tol, stol, f = _norms(k, q, do, lam, ds, 1.0, scale, n, True, dtype)
    _close(grads[2], rg[2], tol, dtype, f, "dv")
    if state:
        _close(grads[3], rg[3], stol, F32, f, "dstate")
    for b, m in enumerate(n):
        for t in (o, *grads[:3]):
            assert (t[b, :, m:] == 0).all(), "rows past the length are zero"


# lengths around the chunk of 64 and its halves, one token, several chunks
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 130, 300])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_lengths(T, dtype):
    _check(2, 3, T, 64, 64, dtype)


# head dims off the tile sizes, K != V, the largest
@pytest.mark.parametrize("K,V", [(128, 128), (100, 100), (96, 64), (7, 5), (1, 1), (33, 129), (256, 256), (256, 40),
                                 (40, 256), (192, 128)])
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
def test_head_dims(K, V, dtype):
    _check(1, 3, 150, K, V, dtype, layout="token", seed=K)


@pytest.mark.parametrize("layout", ["head", "token", "slice"])
@pytest.mark.parametrize("state", [False, True], ids=["", "state"])
def test_layouts(layout, state):
    _check(2, 4, 140, 64, 96, BF, layout=layout, state=state, seed=5)


# ragged: an empty sequence, one token, whole chunks, the whole length; NaN and infinities past every length
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
def test_ragged(dtype):
    _check(5, 3, 200, 64, 64, dtype, layout="token", lens=[0, 1, 64, 129, 200], seed=6)


# long enough that few heads' rows are cut into segments, ragged ends among them
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
def test_segments(dtype):
    _check(2, 3, 1500, 64, 64, dtype, lens=[1333, 0], seed=7)


def test_no_rows():
    lam = _decays(2, 0).to(DEV)
    q = torch.empty(3, 2, 0, 8, dtype=BF, device=DEV)
    S0 = torch.randn(3, 2, 8, 8, device=DEV)
    o, S = linear_attention(q, q, q, lam, initial_state=S0, return_state=True)
    assert o.shape == (3, 2, 0, 8) and torch.equal(S, S0)
    o, S = linear_attention(q, q, q, lam, return_state=True)
    assert (S == 0).all()


def test_lengths_outside_the_rows_are_clamped():
    q = torch.randn(2, 1, 40, 16, device=DEV)
    lam = _decays(1, 0).to(DEV)
    whole = linear_attention(q, q, q, lam, return_state=True)
    odd = linear_attention(q, q, q, lam, lengths=torch.tensor([1000, -3], dtype=torch.int32, device=DEV), return_state=True)
    for a, b in zip(whole, odd):
        assert torch.equal(a[0], b[0]) and (b[1] == 0).all()


def test_indexes_past_32_bits():
    """int64 lengths and slots whose low 32 bits would name other rows."""
    q = torch.randn(2, 1, 40, 16, device=DEV)
    lam = _decays(1, 0).to(DEV)
    whole = linear_attention(q, q, q, lam)
    far = linear_attention(q, q, q, lam, lengths=torch.tensor([1 << 32, 40 - (1 << 32)], device=DEV))
    assert torch.equal(far[0], whole[0]) and (far[1] == 0).all()
    state = torch.randn(2, 1, 16, 16, device=DEV)
    before = state.clone()
    o = linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], lam, state, slots=torch.tensor([1 << 32, 1], device=DEV))
    assert (o[0] == 0).all() and torch.equal(state[0], before[0]) and not torch.equal(state[1], before[1])


def test_shared_heads_and_partial_gradients():
    """Keys and values shared by the heads as expanded views; a loss of the state alone."""
    g = gen(11)
    B, H, T, K = 2, 4, 90, 32
    lam = _decays(H, 1)
    q, k, v = randn(g, B, H, T, K), randn(g, B, 1, T, K), randn(g, B, 1, T, K)
    dev = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    o, S = linear_attention(dev[0], dev[1].expand(-1, H, -1, -1), dev[2].expand(-1, H, -1, -1), lam.to(DEV),
                            return_state=True)
    cpu = [t.double().requires_grad_() for t in (q, k, v)]
    ro, rS = linear_attention_ref(cpu[0], cpu[1].expand(-1, H, -1, -1), cpu[2].expand(-1, H, -1, -1), lam, K**-0.5)
    do, dS = randn(g, B, H, T, K), randn(g, B, H, K, K)
    for a, b in ((o, ro), (S, rS)):
        torch.testing.assert_close(a.detach().double().cpu(), b.detach(), rtol=1e-5, atol=1e-4)
    a = torch.autograd.grad((o, S), dev, (do.to(DEV), dS.to(DEV)), retain_graph=True)
    b = torch.autograd.grad((ro, rS), cpu, (do.double(), dS.double()), retain_graph=True)
    for x, y in zip(a, b):
        torch.testing.assert_close(x.double().cpu(), y, rtol=1e-5, atol=1e-3)
    a = torch.autograd.grad(S, dev, dS.to(DEV), allow_unused=True)
    b = torch.autograd.grad(rS, cpu, dS.double(), allow_unused=True)
    assert a[0] is None or (a[0] == 0).all()
    for x, y in zip(a[1:], b[1:]):
        torch.testing.assert_close(x.double().cpu(), y, rtol=1e-5, atol=1e-3)


def test_gradient_against_differences():
    """o is linear in q, in k (with v fixed) and in v: a central difference of step 1 is exact up to float32's sums."""
    g = gen(12)
    B, H, T, K, V = 1, 3, 150, 48, 40
    lam = _decays(H, 2).to(DEV)
    x = [randn(g, B, H, T, K).to(DEV), randn(g, B, H, T, K).to(DEV), randn(g, B, H, T, V).to(DEV),
         randn(g, B, H, K, V).to(DEV)]
    do, dS = randn(g, B, H, T, V).to(DEV), randn(g, B, H, K, V).to(DEV)

    def loss(q, k, v, S0):
        o, S = linear_attention(q, k, v, lam, initial_state=S0, return_state=True)
        return (o.double() * do).sum() + (S.double() * dS).sum()

    leaves = [t.clone().requires_grad_() for t in x]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i in range(4):
        d = torch.randn_like(x[i])
        up, down = (loss(*[t + s * d if j == i else t for j, t in enumerate(x)]) for s in (1.0, -1.0))
        diff, want = (up - down) / 2, (grads[i].double() * d).sum()
        size = (grads[i].double() * d).norm()  # the sum's terms, their signs at random
        assert (diff - want).abs() <= 1e-3 * size, f"input {i}: {diff.item()} against {want.item()}"


def test_same_results_again_and_on_another_stream():
    g = gen(13)
    lam = _decays(4, 3).to(DEV)
    q, k, v, do = (randn(g, 2, 4, 700, 64).to(BF).to(DEV) for _ in range(4))

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o, S = linear_attention(*leaves, lam, return_state=True)
        return [o, S, *torch.autograd.grad(o, leaves, do)]

    a = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = step()
    side.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_graph():
    """Forward, backward and a decoding step captured and replayed on new inputs, bitwise the eager results."""
    lam = _decays(3, 4).to(DEV)
    q, k, v, do = (torch.empty(2, 3, 400, 64, dtype=BF, device=DEV) for _ in range(4))
    state = torch.empty(2, 3, 64, 64, device=DEV)

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o, S = linear_attention(*leaves, lam, return_state=True)
        grads = torch.autograd.grad(o, leaves, do)
        with torch.no_grad():
            one = linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lam, state)
        return [o, S, *grads, one]

    def fill(seed):
        g = gen(seed)
        for t in (q, k, v, do):
            t.copy_(randn(g, *t.shape))
        state.copy_(randn(g, *state.shape))

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
        want = [t.clone() for t in step()] + [state.clone()]
        fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip([*outs, state], want):
            assert torch.equal(x, y), f"replay {seed}"


@pytest.mark.parametrize("K,V", [(64, 64), (100, 37), (128, 128), (256, 40)])
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,t", [(200, 77), (64, 0), (63, 62), (40, 20)])
def test_not_finite_values_stay_behind_their_token(K, V, dtype, T, t):
    """An infinity or a NaN in a row of k or v (or of o's gradient) reaches the tokens from its own on (up to its own), and
    what it does not reach is what it is without it, to the bit."""
    g = gen(16 + T + K)
    B, H, h = 1, 3, 1
    lam = torch.tensor([-0.02, -0.05, 0.0]).to(DEV)
    clean = [randn(g, B, H, T, c).to(dtype).to(DEV) for c in (K, K, V, V)]  # q, k, v, do

    def run(q, k, v, do):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        o = linear_attention(*leaves, lam)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    want = run(*clean)
    rows = torch.arange(T, device=DEV)
    for i, c, value in ((1, K - 1, float("nan")), (2, V // 2, float("nan")), (2, V - 1, float("inf")), (3, 3, float("nan")),
                        (3, 0, -float("inf")), (0, 2, float("nan"))):
        bad = [x.clone() for x in clean]
        bad[i][:, h, t, c] = value
        got = run(*bad)
        # what it reaches: rows of o, dq, dk, dv
        late, early, own = rows >= t, rows <= t, rows == t
        none = rows < 0
        reach = {0: (own, none, early, early), 1: (late, late, none, own), 2: (late, late, own, none),
                 3: (none, own, early, early)}[i]
        for x, w, r, name in zip(got, want, reach, ("o", "dq", "dk", "dv")):
            what = f"{value} in input {i}: {name}"
            assert torch.equal(x[:, [0, 2]], w[:, [0, 2]]), f"{what}, other heads"
            assert torch.equal(x[:, h, ~r], w[:, h, ~r]), f"{what}, rows that it does not reach"
            assert r.sum() == 0 or not x[:, h, r].isfinite().all(-1).any(), f"{what}, rows that it reaches"
        if i == 2 and value != value:
            others = torch.arange(V, device=DEV) != c
            assert torch.equal(got[0][:, h][..., others], want[0][:, h][..., others]), "o's other columns"


def test_fp16_scores_and_states_past_the_type():
    """Scores and states above 65504 whose outputs are within fp16: operands are held smaller, and none is lost."""
    g = gen(15)
    B, H, T, K, V = 1, 2, 200, 64, 64
    lam = torch.tensor([0.0, -0.01])
    k, v = (300 * randn(g, B, H, T, K)).to(HF), (300 * randn(g, B, H, T, V)).to(HF)
    q = (1e-3 * randn(g, B, H, T, K)).to(HF)
    o, S = linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), lam.to(DEV), scale=0.01, return_state=True)
    ro, rS = linear_attention_ref(q, k, v, lam, 0.01)
    assert rS.abs().max() > 2 * 65504
    tol, stol, f = _norms(q, k, v, lam, None, 0.01, 1.0, [T], False, HF)
    _close(o, ro, tol, HF, f, "o")
    _close(S, rS, stol, F32, f, "state")
    # scores: q . k far above the type, values small
    q2, v2 = (300 * randn(g, B, H, T, K)).to(HF), (1e-3 * randn(g, B, H, T, V)).to(HF)
    o = linear_attention(q2.to(DEV), k.to(DEV), v2.to(DEV), lam.to(DEV), scale=1.0)
    ro, _ = linear_attention_ref(q2, k, v2, lam, 1.0)
    assert ((q2.double() @ k.double().transpose(2, 3)).abs().max() > 2 * 65504) and ro.abs().max() < 65504
    tol, _, f = _norms(q2, k, v2, lam, None, 1.0, 1.0, [T], False, HF)
    _close(o, ro, tol, HF, f, "o of large scores")


def test_rows_past_32_bits():
    """Tensors of more than 2^31 elements: their last rows, under a decay that forgets all before them."""
    K, tail = 128, 300
    T = (1 << 31) // K + 1000
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 20 GiB of GPU memory")
    x = torch.randn(T, K, device=DEV, dtype=BF).view(1, 1, T, K)
    lam = torch.tensor([-1.0], device=DEV)
    with torch.no_grad():
        o, S = linear_attention(x, x, x, lam, return_state=True)
        end = x[:, :, -tail:].contiguous()
        o2, S2 = linear_attention(end, end, end, lam, return_state=True)
    # e^-200 of what came before; the chunks lie elsewhere, so scores are rounded in other places
    assert (o[:, :, -100:].float() - o2[:, :, -100:].float()).abs().max() <= 2.0**-6 * o2.abs().max().float()
    assert (S - S2).abs().max() <= 1e-4 * S2.abs().max()


# ------------------------------------------------------------------- single tokens
@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,K,V", [(3, 4, 128, 128), (1, 1, 1, 1), (2, 3, 100, 100), (5, 2, 33, 7), (2, 1, 256, 256),
                                     (1, 3, 40, 130)])
def test_step(B, H, K, V, dtype):
    print(f"[linattn step] B{B} H{H} K{K} V{V} {dtype}", flush=True)
    g = gen(B + 7 * K + V)
    lam = _decays(H, K)
    rows = B + 4
    state = randn(g, rows, H, K, V)
    ids = torch.randperm(rows, generator=g)[:B + 1]
    ids[B // 2] = -1  # takes no part
    q, k, v = (randn(g, B + 1, H, n).to(dtype) for n in (K, K, V))
    free = [r for r in range(rows) if r not in ids.tolist()]
    state[free] = float("nan")  # rows of no sequence are not touched
    dstate = state.to(DEV)
    with torch.no_grad():
        o = linear_attention_step(q.to(DEV), k.to(DEV), v.to(DEV), lam.to(DEV), dstate,
                                  slots=ids.to(torch.int32).to(DEV))
    o, dstate = o.double().cpu(), dstate.cpu()
    assert torch.isnan(dstate[free]).all() and (o[B // 2] == 0).all()
    for b, r in enumerate(ids.tolist()):
        if r < 0:
            continue
        ro, rS = linear_attention_ref(*(t[b][None, :, None] for t in (q, k, v)), lam, K**-0.5, state[r][None])
        # float32 throughout: g S + k v in two roundings, K products to a sum
        S0 = torch.exp(lam.double())[:, None, None] * state[r].double()
        kv = k[b].double()[..., None] * v[b].double()[..., None, :]
        assert ((dstate[r] - rS[0]).abs() <= 2.0**-22 * (S0.abs() + kv.abs())).all()
        terms = (q[b].double()[..., None] * (S0.abs() + kv.abs())).abs().sum(1) * K**-0.5
        rnd = {BF: 2.0**-8, HF: 2.0**-11, F32: 2.0**-24}[dtype]
        bound = 2.0**-20 * terms + 1.01 * rnd * ro[0, :, 0].abs() + (2.0**-25 if dtype == HF else 0)
        assert ((o[b] - ro[0, :, 0]).abs() <= bound).all()


def test_steps_follow_the_whole_sequence():
    """A prompt in two pieces, then single tokens, against the whole sequence at once (float32)."""
    g = gen(21)
    B, H, T, K, V = 2, 3, 150, 32, 48
    lam = _decays(H, 5).to(DEV)
    q, k, v = randn(g, B, H, T, K).to(DEV), randn(g, B, H, T, K).to(DEV), randn(g, B, H, T, V).to(DEV)
    with torch.no_grad():
        whole, end = linear_attention(q, k, v, lam, return_state=True)
        o1, S = linear_attention(q[:, :, :70], k[:, :, :70], v[:, :, :70], lam, return_state=True)
        o2, S = linear_attention(q[:, :, 70:147], k[:, :, 70:147], v[:, :, 70:147], lam, initial_state=S, return_state=True)
        rest = [linear_attention_step(q[:, :, t], k[:, :, t], v[:, :, t], lam, S) for t in range(147, T)]
    o = torch.cat([o1, o2, torch.stack(rest, 2)], 2)
    torch.testing.assert_close(o, whole, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(S, end, rtol=1e-4, atol=1e-4)


def test_step_in_a_cache_past_32_bits():
    """Rows of the state whose offsets pass 2^32 elements."""
    rows, H, K, V = 70000, 1, 256, 256
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 18 GiB of GPU memory")
    state = torch.empty(rows, H, K, V, device=DEV)
    ids = torch.tensor([rows - 1, 3, 65536], dtype=torch.int32, device=DEV)
    g = gen(22)
    first = randn(g, 3, H, K, V).to(DEV)
    state[ids.long()] = first
    q, k, v = (randn(g, 3, H, K).to(DEV) for _ in range(3))
    lam = torch.tensor([-0.1], device=DEV)
    small = first.clone()
    with torch.no_grad():
        a = linear_attention_step(q, k, v, lam, state, slots=ids)
        b = linear_attention_step(q, k, v, lam, small)
    assert torch.equal(a, b) and torch.equal(state[ids.long()], small)


def test_native_binding_and_python_functions_agree(monkeypatch):
    """The native nodes (where built) and the Python Functions launch the same kernels: bitwise equal results."""
    from dynconv import _capi

    _capi.load()
    if _capi.binding is None:
        pytest.skip("no native binding")
    g = gen(14)
    lam = _decays(2, 5).to(DEV)
    x = [randn(g, 2, 2, 90, 32).to(BF).to(DEV) for _ in range(4)]
    S0, dS = randn(g, 2, 2, 32, 32).to(DEV), randn(g, 2, 2, 32, 32).to(DEV)
    n = torch.tensor([90, 17], dtype=torch.int32, device=DEV)

    def run():
        leaves = [t.detach().requires_grad_() for t in (*x[:3], S0)]
        o, S = linear_attention(*leaves[:3], lam, 0.5, leaves[3], n, return_state=True)
        grads = torch.autograd.grad((o, S), leaves, (x[3], dS))
        alone = torch.autograd.grad(linear_attention(*leaves[:3], lam), leaves[:3], x[3])
        with torch.no_grad():
            S1 = S0.clone()
            one = linear_attention_step(x[0][:, :, 0], x[1][:, :, 0], x[2][:, :, 0], lam, S1, slots=n % 2)
            quiet = linear_attention(*x[:3], lam)
        return [o, S, *grads, *alone, one, S1, quiet], o.grad_fn.name()

    a, name = run()
    monkeypatch.setattr(_capi, "binding", None)
    b, other = run()
    assert name != other, "the native node takes the plain call"
    for p, q in zip(a, b):
        assert torch.equal(p, q) and p.stride() == q.stride()


def test_refusals():
    lam = torch.zeros(2, device=DEV)
    q = torch.randn(1, 2, 4, 8, device=DEV)
    S = torch.zeros(1, 2, 8, 8, device=DEV)
    big = torch.randn(1, 2, 4, 257, device=DEV)
    ok = dict(log_decay=lam)
    bad = [
        lambda: linear_attention(q.cpu(), q, q, lam),
        lambda: linear_attention(q, q[..., :4], q, **ok),
        lambda: linear_attention(q, q, q[:, :1], **ok),
        lambda: linear_attention(q, q.half(), q, **ok),
        lambda: linear_attention(q.double(), q.double(), q.double(), **ok),
        lambda: linear_attention(big, big, q, **ok),
        lambda: linear_attention(q, q, q, lam.double()),
        lambda: linear_attention(q, q, q, lam[:1]),
        lambda: linear_attention(q, q, q, lam.cpu()),
        lambda: linear_attention(q, q, q, lam.clone().requires_grad_()),
        lambda: linear_attention(q, q, q, lam, initial_state=S.half()),
        lambda: linear_attention(q, q, q, lam, initial_state=S[..., :4]),
        lambda: linear_attention(q, q, q, lam, lengths=torch.tensor([4, 4], dtype=torch.int32, device=DEV)),
        lambda: linear_attention(q, q, q, lam, lengths=torch.tensor([4.0], device=DEV)),
        lambda: linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], lam, S[..., :4].contiguous()),
        lambda: linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], lam, S.transpose(2, 3)),
        lambda: linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], lam, S.half()),
        lambda: linear_attention_step(q[:, :, 0].repeat(3, 1, 1), q[:, :, 0].repeat(3, 1, 1), q[:, :, 0].repeat(3, 1, 1), lam, S),
        lambda: linear_attention_step(q[:, :, 0].requires_grad_(), q[:, :, 0], q[:, :, 0], lam, S),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError):
            f()
            pytest.fail(f"call {i} was taken")
