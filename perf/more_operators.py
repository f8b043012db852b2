"""Performance cases of the gated delta rule (whole sequences, and single tokens from a state) and of the norms around a
block fused with its gate, its residual scale and the residual sum.

A case is a dict:
    op         "delta"     gated_delta_rule: q, k [B, Hk, T, K], v [B, H, T, V], gates [B, H, T]
               "step"      gated_delta_rule_step: one token of each of B sequences, states in a cache of `slots` slots
               "residual"  residual_norm: x, branch [B, T, D]
    pass       "train": forward and backward, every gradient returned; "infer": the forward alone
    dtype      of the activations (states are float32)
    gates      (delta, step) type of log_decay and beta: "same" as the activations, or "fp32"
    layout     (delta) "head": q, k, v are [B, H, T, .] in memory, as the grouped convolution writes them with head_dim;
               "token": [B, T, H, .], as it writes them without
    normalize  (delta, step) the rows of q and k are divided by their norms within the call (else they come so)
    ragged     (delta) sequences of different lengths up to T (one of them empty where B allows); else all are T long
    state      (delta) starts from a state and returns the new one, as a prompt taken in pieces does
    stream     (residual) type of the residual stream x: "same" as the branch, or "fp32"
    gate       (residual) activation of the branch's gate: "silu", "sigmoid", or "none" for no gate
    scale      (residual) a residual scale for each channel

Sizes are those of this repository's benchmark and tests (D 256-4096, T up to 8192, B 1-8, head dims 64 and 128), a
longer prompt, serving batches, and ragged ones between them.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    dr = dict(op="delta", dtype="bf16", gates="same", layout="head", normalize=True, ragged=False, state=False)
    st = dict(op="step", dtype="bf16", gates="fp32", normalize=True, **{"pass": "infer"})
    rn = dict(op="residual", dtype="bf16", stream="same", gate="silu", scale=True)
    return [
        # a short question to a small model: latency
        {"name": "dr_short", **dr, "pass": "infer", "gates": "fp32", "B": 1, "Hk": 8, "H": 8, "T": 37, "K": 64, "V": 64,
         "state": True},
        # training: the repository's benchmark shape, and its q|k|v layer with two value heads to a key head
        {"name": "dr_train", **dr, "pass": "train", "B": 4, "Hk": 16, "H": 16, "T": 4096, "K": 128, "V": 128},
        {"name": "dr_train_qkv", **dr, "pass": "train", "B": 2, "Hk": 16, "H": 32, "T": 8192, "K": 128, "V": 128,
         "layout": "token"},
        # the fp32 tier on sizes off the powers of two
        {"name": "dr_train_fp32", **dr, "pass": "train", "dtype": "fp32", "B": 3, "Hk": 10, "H": 10, "T": 1537, "K": 100,
         "V": 100, "layout": "token", "ragged": True, "state": True, "normalize": False},
        # a piece of a long sequence in training: states and gates in float32, and their gradients
        {"name": "dr_train_piece", **dr, "pass": "train", "B": 2, "Hk": 8, "H": 16, "T": 2048, "K": 64, "V": 128,
         "gates": "fp32", "state": True},
        # a piece of a long prompt for one user: few heads' rows, long axis
        {"name": "dr_prompt", **dr, "pass": "infer", "gates": "fp32", "B": 1, "Hk": 16, "H": 16, "T": 32768, "K": 128,
         "V": 128, "layout": "token", "state": True},
        # one decoding step: a few sequences, and a serving batch in a cache that holds more of them
        {"name": "step_small", **st, "B": 8, "Hk": 16, "H": 16, "K": 128, "V": 128, "slots": 8},
        {"name": "step_serving", **st, "B": 256, "Hk": 16, "H": 32, "K": 128, "V": 128, "slots": 320},
        # the norms of one decoding step, of the q|k|v layer's training, and of a ragged shape on a float32 stream
        {"name": "rn_decode", **rn, "pass": "infer", "B": 8, "T": 1, "D": 2048},
        {"name": "rn_train", **rn, "pass": "train", "B": 2, "T": 8192, "D": 4096},
        {"name": "rn_ragged", **rn, "pass": "train", "dtype": "fp16", "stream": "fp32", "gate": "none", "B": 3, "T": 1537,
         "D": 1000},
    ]


def draw(rng):
    """One case of the same ranges: sizes over their logarithms, ragged ones among them."""

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    cases = {c["name"]: c for c in listed()}
    while True:
        op = rng.choice(["delta"] * 5 + ["step"] * 2 + ["residual"] * 2)
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        train = rng.random() < 0.6
        gates = rng.choice(["same", "fp32"])
        if op == "delta":
            dim = rng.choice([32, 64, 64, 96, 100, 128, 128, 128, 192, 256])
            Hk = log(1, 32)
            c = {"B": log(1, 8), "Hk": Hk, "H": Hk * rng.choice([1, 1, 1, 2, 4]), "T": log(1, 32768), "K": dim,
                 "V": rng.choice([dim, dim, dim, 64, 128, 256]), "layout": rng.choice(["head", "token"]), "gates": gates,
                 "normalize": rng.random() < 0.7, "ragged": rng.random() < 0.3, "state": rng.random() < 0.4}
            if c["T"] > 1 and rng.random() < 0.3:
                c["T"] = 1 << round(math.log2(c["T"]))
            most = "dr_train_qkv"
        elif op == "step":
            dim = rng.choice([32, 64, 96, 100, 128, 128, 256])
            train, B, Hk = False, log(1, 256), log(1, 32)
            c = {"B": B, "Hk": Hk, "H": Hk * rng.choice([1, 1, 2]), "K": dim, "V": rng.choice([dim, dim, 64, 128]),
                 "gates": gates, "normalize": rng.random() < 0.7, "slots": B + rng.randrange(64)}
            most = "step_serving"
        else:
            c = {"B": log(1, 8), "T": log(256 if train else 1, 8192), "D": log(64, 8192),
                 "stream": rng.choice(["same", "same", "fp32"]), "gate": rng.choice(["none", "silu", "sigmoid"]),
                 "scale": rng.random() < 0.6}
            if rng.random() < 0.6:
                c["D"] = max(64, round(c["D"] / 64) * 64)
            most = "rn_train"
        c.update({"op": op, "pass": "train" if train else "infer", "dtype": dtype})
        # within the largest listed case of its kind (fp32 products run on slower units: an eighth of its operations)
        w, m = work(c), work(cases[most])
        if w["bytes"] <= m["bytes"] and w["flops"] <= m["flops"] / (8 if dtype == "fp32" else 1):
            return c


def prepare(case, seed):
    """The tensors that a program holds before the call."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train = case["pass"] == "train"

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    s = {"case": case}
    op, B = case["op"], case["B"]
    if op in ("delta", "step"):
        H, Hk, K, V = case["H"], case["Hk"], case["K"], case["V"]
        s["scale"] = K ** -0.5
        gd = dt if case["gates"] == "same" else torch.float32
        T = case.get("T", 1)

        def keys():
            # rows of a head lean one way, as activated projections do
            t = torch.randn(B, Hk, T, K, generator=g, device=dev) + 0.5 * torch.randn(Hk, 1, K, generator=g, device=dev)
            return t if case["normalize"] else t / torch.sqrt((t * t).sum(-1, keepdim=True))

        def gate(f):
            t = f(torch.randn(B, T, H, generator=g, device=dev), torch.rand(H, generator=g, device=dev))
            return t.to(gd).transpose(1, 2)  # a projection gives them token by token

        q, k, v = keys(), keys(), torch.randn(B, H, T, V, generator=g, device=dev)
        # decays a token from 1/2 to 1 - 2^-10, the softplus of a projection times a rate of each head
        lam = gate(lambda x, u: -torch.log1p(torch.exp(x)) * torch.exp2(-9 * u))
        beta = gate(lambda x, u: 1 / (1 + torch.exp(-x)))
    if op == "delta":
        def heads(t):
            t = t.to(dt)
            return (t if case["layout"] == "head" else t.transpose(1, 2).contiguous().transpose(1, 2)).requires_grad_(train)

        s["q"], s["k"], s["v"] = heads(q), heads(k), heads(v)
        s["log_decay"], s["beta"] = lam.requires_grad_(train), beta.requires_grad_(train)
        s["initial"] = normal(B, H, K, V, dtype=torch.float32).requires_grad_(train) if case["state"] else None
        s["lengths"] = None
        if case["ragged"]:
            n = torch.randint(1, T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
            n[0] = T
            if B > 2:
                n[1] = 0
            s["lengths"] = n
        if train:
            # the gradient of the output comes back through the norm, which reads it token by token
            s["do"] = normal(B, T, H, V).transpose(1, 2)
            s["dstate"] = normal(B, H, K, V, dtype=torch.float32) if case["state"] else None
    elif op == "step":
        s["q"], s["k"], s["v"] = (t[:, :, 0].to(dt) for t in (q, k, v))
        s["log_decay"], s["beta"] = lam[:, :, 0], beta[:, :, 0]
        s["state"] = normal(case["slots"], H, K, V, dtype=torch.float32)
        # the slots that a serving loop has given its running sequences: distinct, in no order
        s["slots"] = torch.randperm(case["slots"], generator=g, device=dev)[:B].to(torch.int32)
    else:
        T, D = case["T"], case["D"]
        xd = dt if case["stream"] == "same" else torch.float32
        s["x"] = normal(B, T, D, scale=4.0, dtype=xd).requires_grad_(train)
        s["branch"] = normal(B, T, D, scale=0.5).requires_grad_(train)
        s["weight"] = (1 + normal(D, scale=0.1, dtype=torch.float32)).to(dt).requires_grad_(train)
        s["branch_weight"] = (1 + normal(D, scale=0.1, dtype=torch.float32)).to(dt).requires_grad_(train)
        s["gate"] = None if case["gate"] == "none" else normal(B, T, D).requires_grad_(train)
        s["scale"] = normal(D, scale=0.3).requires_grad_(train) if case["scale"] else None
        if train:
            s["dy"], s["dh"] = normal(B, T, D), normal(B, T, D, dtype=xd)
    return s


def _leaves(s):
    names = (("q", "k", "v", "log_decay", "beta", "initial") if s["case"]["op"] == "delta"
             else ("x", "branch", "weight", "branch_weight", "gate", "scale"))
    return [s[n] for n in names if s[n] is not None]


# ---------------------------------------------------------------- the framework's operators
def _own_delta(s):
    from linattn import gated_delta_rule

    c = s["case"]
    train = c["pass"] == "train"
    with torch.set_grad_enabled(train):
        out = gated_delta_rule(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], scale=s["scale"],
                               initial_state=s["initial"], lengths=s["lengths"], return_state=c["state"],
                               normalize=c["normalize"])
    out = out if c["state"] else (out,)
    if not train:
        return {"out": out}
    douts = (s["do"], s["dstate"]) if c["state"] else (s["do"],)
    return {"out": out, "grads": torch.autograd.grad(out, _leaves(s), douts)}


def _own_step(s):
    from linattn import gated_delta_rule_step

    o = gated_delta_rule_step(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], scale=s["scale"],
                              slots=s["slots"], normalize=s["case"]["normalize"])
    return {"o": o, "state": s["state"]}


def _own_residual(s):
    from linattn import residual_norm

    c = s["case"]
    train = c["pass"] == "train"
    with torch.set_grad_enabled(train):
        y, h = residual_norm(s["x"], s["branch"], weight=s["weight"], branch_weight=s["branch_weight"], gate=s["gate"],
                             activation=None if s["gate"] is None else c["gate"], scale=s["scale"], eps=EPS)
    if not train:
        return {"out": (y, h)}
    return {"out": (y, h), "grads": torch.autograd.grad((y, h), _leaves(s), (s["dy"], s["dh"]))}


# ---------------------------------------------------------------- plain forms
CHUNK = 64


def _norm_rows(t, on):
    """t's rows divided by their norms, and what they were multiplied with."""
    r = 1 / torch.sqrt((t * t).sum(-1, keepdim=True) + EPS) if on else torch.ones_like(t[..., :1])
    return t * r, r


def _norm_rows_backward(dt, t, r, on):
    """The gradient of the rows before, from that of the normed rows t."""
    return r * (dt - t * (t * dt).sum(-1, keepdim=True)) if on else dt


def _chunks(t, lengths, dtype=torch.float32):
    """t [B, H, T, ...] as [B, H, N, CHUNK, ...], widened, rows past each sequence's length zero whatever they hold."""
    t = t.detach().to(dtype)
    T = t.shape[2]
    if lengths is not None:
        live = (torch.arange(T, device=t.device)[None] < lengths[:, None]).view(t.shape[0], 1, T, *[1] * (t.dim() - 3))
        t = torch.where(live, t, torch.zeros_like(t))
    n = -(-T // CHUNK)
    full = torch.zeros(*t.shape[:2], n * CHUNK, *t.shape[3:], device=t.device, dtype=dtype)
    full[:, :, :T] = t
    return full.view(*t.shape[:2], n, CHUNK, *t.shape[3:])


def _whole(t, T):
    return t.flatten(2, 3)[:, :, :T]


def _plain_delta(s):
    """Chunks of tokens: within each the triangular system of its corrections, the state carried between them; the backward
    from the last chunk on."""
    c, lengths = s["case"], s["lengths"]
    T, G = c["T"], c["H"] // c["Hk"]
    dt = s["q"].dtype
    q0, rq = _norm_rows(_chunks(s["q"], lengths), c["normalize"])
    k0, rk = _norm_rows(_chunks(s["k"], lengths), c["normalize"])
    q, k = q0.repeat_interleave(G, 1) * s["scale"], k0.repeat_interleave(G, 1)
    v, b = _chunks(s["v"], lengths), _chunks(s["beta"], lengths)[..., None]
    # decays up to and with each token of its chunk: sums of logarithms in 64 bits, as their differences count
    L = _chunks(s["log_decay"], lengths, torch.float64).cumsum(-1)
    past = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    E = torch.exp(torch.where(past, L[..., :, None] - L[..., None, :], -math.inf)).float()
    g, d, gl = torch.exp(L).float()[..., None], torch.exp(L[..., -1:] - L).float()[..., None], torch.exp(L[..., -1]).float()
    gl = gl[..., None, None]
    P = (q @ k.transpose(3, 4)) * E
    M = ((k @ k.transpose(3, 4)) * E).tril(-1)
    A = b * M
    # the inverse of 1 + A, row by row
    X = torch.eye(CHUNK, device=q.device).expand_as(A).clone()
    for i in range(1, CHUNK):
        X[..., i, :i] = -(A[..., i, None, :i] @ X[..., :i, :i])[..., 0, :]
    W, Ub = X @ (b * g * k), X @ (b * v)
    N = L.shape[2]
    S = torch.zeros(c["B"], c["H"], c["K"], c["V"], device=q.device)
    if s["initial"] is not None:
        S = S + s["initial"].detach()
    states, U = [], []
    dk = (d * k).transpose(3, 4)
    for n in range(N):
        states.append(S)
        U.append(Ub[:, :, n] - W[:, :, n] @ S)
        S = gl[:, :, n] * S + dk[:, :, n] @ U[-1]
    first, U = torch.stack(states, 2), torch.stack(U, 2)
    o = _whole(g * (q @ first) + P @ U, T)
    outs = (o.to(dt),) + ((S,) if c["state"] else ())
    if c["pass"] == "infer":
        return {"out": outs}
    do = _chunks(s["do"], lengths)
    dS = s["dstate"].clone() if c["state"] else torch.zeros_like(S)
    dUo, into, read = P.transpose(3, 4) @ do, (g * q).transpose(3, 4) @ do, (b * g * k).transpose(3, 4)
    dstates, dR = [None] * N, [None] * N
    for n in reversed(range(N)):
        dstates[n] = dS
        dR[n] = X[:, :, n].transpose(2, 3) @ (dUo[:, :, n] + (d * k)[:, :, n] @ dS)
        dS = gl[:, :, n] * dS + into[:, :, n] - read[:, :, n] @ dR[n]
    last, dR = torch.stack(dstates, 2), torch.stack(dR, 2)
    dP = (do @ U.transpose(3, 4)).tril()
    dA = -(dR @ U.transpose(3, 4)).tril(-1)
    doS, dRS, UdS = do @ first.transpose(3, 4), dR @ first.transpose(3, 4), U @ last.transpose(3, 4)
    dPE, dME = dP * E, b * dA * E
    dq = g * doS + dPE @ k
    dk = dPE.transpose(3, 4) @ q + d * UdS - b * g * dRS + dME @ k + dME.transpose(3, 4) @ k
    dv = b * dR
    db = (dR * v).sum(-1) - (g * k * dRS).sum(-1) + (dA * M).sum(-1)
    # through every decay's logarithm, then through the sums
    pairs = (dP.double() * P + dA.double() * A)
    kept = (d * k * UdS).double().sum(-1)
    dL = pairs.sum(-1) - pairs.sum(-2) + (g * (q * doS - b * k * dRS)).double().sum(-1) - kept
    dL[..., -1] += kept.sum(-1) + (gl * first * last).double().sum((-1, -2))
    dlam = dL.flip(-1).cumsum(-1).flip(-1)

    def shared(t):
        return t.unflatten(1, (c["Hk"], G)).sum(2)

    dq = _norm_rows_backward(shared(dq) * s["scale"], q0, rq, c["normalize"])
    dk = _norm_rows_backward(shared(dk), k0, rk, c["normalize"])
    grads = [_whole(t, T) for t in (dq, dk, dv, dlam, db)]
    if lengths is not None:
        live = (torch.arange(T, device=q.device)[None] < lengths[:, None])[:, None]
        grads = [t * (live[..., None] if t.dim() == 4 else live) for t in grads]
    gd = s["beta"].dtype
    grads = [t.to(dt) for t in grads[:3]] + [t.to(gd) for t in grads[3:]] + ([dS] if c["state"] else [])
    return {"out": outs, "grads": tuple(grads)}


def _plain_step(s):
    c, slots = s["case"], s["slots"].long()
    G = c["H"] // c["Hk"]
    q, k = (_norm_rows(s[n].float(), c["normalize"])[0].repeat_interleave(G, 1) for n in ("q", "k"))
    v, b = s["v"].float(), s["beta"].float()[..., None]
    S = s["state"][slots] * torch.exp(s["log_decay"].float())[..., None, None]
    u = b * (v - (k[..., :, None] * S).sum(2))
    S = S + k[..., :, None] * u[..., None, :]
    s["state"][slots] = S
    o = (q[..., :, None] * S).sum(2) * s["scale"]
    return {"o": o.to(s["q"].dtype), "state": s["state"]}


def _plain_residual(s):
    c = s["case"]
    dt, xd = s["branch"].dtype, s["x"].dtype
    x, br, w, bw = (s[n].detach().float() for n in ("x", "branch", "weight", "branch_weight"))
    rb = torch.rsqrt((br * br).mean(-1, keepdim=True) + EPS)
    bh = br * rb
    n = bh * bw
    if s["gate"] is not None:
        a = s["gate"].detach().float()
        sg = 1 / (1 + torch.exp(-a))
        act, dact = (a * sg, sg * (1 + a * (1 - sg))) if c["gate"] == "silu" else (sg, sg * (1 - sg))
    else:
        act = torch.ones_like(n)
    sc = s["scale"].detach().float() if c["scale"] else torch.ones_like(w)
    h = (x + n * act * sc).to(xd)
    hf = h.float()
    rh = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    hh = hf * rh
    y = (hh * w).to(dt)
    if c["pass"] == "infer":
        return {"out": (y, h)}
    dy = s["dy"].float()
    dhh = dy * w
    dx = s["dh"].float() + rh * (dhh - hh * (dhh * hh).mean(-1, keepdim=True))
    dn = dx * act * sc
    dbh = dn * bw
    dbr = rb * (dbh - bh * (dbh * bh).mean(-1, keepdim=True))
    grads = [dx.to(xd), dbr.to(dt), (dy * hh).sum((0, 1)).to(dt), (dn * bh).sum((0, 1)).to(dt)]
    if s["gate"] is not None:
        grads.append((dx * n * sc * dact).to(dt))
    if c["scale"]:
        grads.append((dx * n * act).sum((0, 1)).to(dt))
    return {"out": (y, h), "grads": tuple(grads)}


def run(state):
    """One pass: the outputs, the updated state, and for "train" the gradients of every input."""
    op = state["case"]["op"]
    if own:
        return {"delta": _own_delta, "step": _own_step, "residual": _own_residual}[op](state)
    with torch.no_grad():
        return {"delta": _plain_delta, "step": _plain_step, "residual": _plain_residual}[op](state)


def work(case):
    """Bytes and operations of one pass.  A training pass is two calls (the gradient of the output exists only
    after the forward): each reads its inputs and writes its outputs once.  Operations are those of the recurrent
    form (2 a multiply-add), or of the plain triangle for short sequences."""
    e = 4 if case["dtype"] == "fp32" else 2
    B, train = case["B"], case["pass"] == "train"
    if case["op"] in ("delta", "step"):
        H, Hk, K, V = case["H"], case["Hk"], case["K"], case["V"]
        eg = 4 if case["gates"] == "fp32" else e
        st = 4 * B * H * K * V
        if case["op"] == "step":
            return {"bytes": e * B * (2 * Hk * K + 2 * H * V) + 2 * eg * B * H + 2 * st, "flops": 7 * B * H * K * V}
        rows = B * case["T"]
        n = rows * (0.5 if case["ragged"] else 1)
        byt = n * (e * (2 * Hk * K + H * V) + 2 * eg * H) + rows * e * H * V  # rows that no length reaches are written too
        pair = min(2 * K * V, case["T"] * max(K, V))  # one product of a token with a state
        flops = 3 * pair * n * H
        if train:
            byt += n * (e * (2 * Hk * K + 2 * H * V) + 2 * eg * H) + rows * (e * (2 * Hk * K + H * V) + 2 * eg * H)
            flops += 6 * pair * n * H
        states = (2 if not train else 4) * st if case["state"] else 0
        return {"bytes": int(byt + states), "flops": int(flops)}
    n = B * case["T"] * case["D"]
    ex = 4 if case["stream"] == "fp32" else e
    gate = case["gate"] != "none"
    byt = n * (2 * ex + e * (3 if gate else 2))  # x, h; branch, gate, y
    if train:
        byt += n * (3 * ex + e * (5 if gate else 3))  # h, dh, dx; branch, gate, dy, dbranch, dgate
    return {"bytes": byt, "flops": n * (14 + (30 if train else 0))}


# ---------------------------------------------------------------- 64 bits, from the definitions
def _exact_delta(s):
    """The recurrence token by token over all heads at once, and its adjoint from the last token on."""
    c = s["case"]
    B, H, Hk, T, K, V = (c[n] for n in ("B", "H", "Hk", "T", "K", "V"))
    train, span = c["pass"] == "train", 64
    dev = s["q"].device
    f64 = dict(dtype=torch.float64, device=dev)
    lens = torch.full((B,), T, device=dev) if s["lengths"] is None else s["lengths"].long()
    live = (torch.arange(T, device=dev)[:, None] < lens).to(torch.float64)[:, :, None]  # [T, B, 1]

    def tokens(t):
        """[T, B, heads, ...]; nothing of the rows past the lengths."""
        t = t.detach().double().movedim(2, 0)
        keep = live.reshape(T, B, *[1] * (t.dim() - 2)) > 0
        return torch.where(keep, t, torch.zeros((), **f64)).contiguous()

    def unit(t):
        n = torch.sqrt((t * t).sum(-1, keepdim=True) + EPS) if c["normalize"] else torch.ones_like(t[..., :1])
        return (t / n).repeat_interleave(H // Hk, 2), n

    q, nq = unit(tokens(s["q"]))
    k, nk = unit(tokens(s["k"]))
    v, beta, a = tokens(s["v"]), tokens(s["beta"]), torch.exp(tokens(s["log_decay"]))
    sc = s["scale"]
    S = torch.zeros(B, H, K, V, **f64) if s["initial"] is None else s["initial"].detach().double().clone()

    def delta(t, S):
        """The state decayed, and what it gets wrong of token t."""
        D = a[t, :, :, None, None] * S
        return D, v[t] - (k[t][:, :, None] @ D)[:, :, 0]

    o, marks = torch.zeros(T, B, H, V, **f64), {}
    for t in range(T):
        if train and t % span == 0:
            marks[t] = S.clone()
        D, y = delta(t, S)
        S = D + k[t][..., None] * (beta[t][..., None] * y)[:, :, None]
        o[t] = (q[t][:, :, None] @ S)[:, :, 0] * sc
    out = {"out": (o.movedim(0, 2),) + ((S,) if c["state"] else ())}
    if not train:
        return out
    do = tokens(s["do"]) * sc
    dS = s["dstate"].double().clone() if c["state"] else torch.zeros_like(S)
    dq, dk, dv, dl, db = (torch.zeros_like(t) for t in (q, k, v, a, beta))
    for t0 in sorted(marks, reverse=True):
        before, S = [], marks.pop(t0)
        for t in range(t0, min(t0 + span, T)):
            before.append(S)
            D, y = delta(t, S)
            S = D + k[t][..., None] * (beta[t][..., None] * y)[:, :, None]
        for t in range(min(t0 + span, T) - 1, t0 - 1, -1):
            S = before.pop()
            D, y = delta(t, S)
            u = beta[t][..., None] * y
            kt, qt = k[t][..., None], q[t][..., None]
            dq[t] = ((D + kt * u[:, :, None]) @ do[t][..., None])[..., 0]
            dS += qt * do[t][:, :, None]
            du = (kt.transpose(2, 3) @ dS)[:, :, 0]
            dy = beta[t][..., None] * du
            dk[t] = (dS @ u[..., None])[..., 0] - (D @ dy[..., None])[..., 0]
            dv[t], db[t] = dy, (du * y).sum(-1)
            dS -= kt * dy[:, :, None]
            dl[t] = (dS * D).sum((2, 3)) * live[t]
            dS *= a[t, :, :, None, None]

    def rows(dt, t, n):
        """Back through the shared heads and the rows' norms."""
        dt = dt.view(T, B, Hk, H // Hk, K).sum(3)
        t = t.view(T, B, Hk, H // Hk, K)[:, :, :, 0]
        return ((dt - t * (dt * t).sum(-1, keepdim=True)) / n if c["normalize"] else dt)

    grads = (rows(dq, q, nq), rows(dk, k, nk), dv, dl, db)
    out["grads"] = tuple(t.movedim(0, 2) for t in grads) + ((dS,) if c["state"] else ())
    return out


def exact(case, seed):
    """run()'s outputs from the same inputs in 64 bits, by the formulas of the operators."""
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "delta":
            return _exact_delta(s)
        if case["op"] == "step":
            G = case["H"] // case["Hk"]
            state = s["state"].double()
            o = torch.empty(case["B"], case["H"], case["V"], dtype=torch.float64, device=state.device)
            for b, slot in enumerate(s["slots"].tolist()):
                q, k = s["q"][b].double(), s["k"][b].double()
                if case["normalize"]:
                    q, k = (t / torch.sqrt((t ** 2).sum(-1, keepdim=True) + EPS) for t in (q, k))
                q, k = q.repeat_interleave(G, 0), k.repeat_interleave(G, 0)
                D = torch.exp(s["log_decay"][b].double())[:, None, None] * state[slot]
                y = s["v"][b].double() - torch.einsum("hk,hkv->hv", k, D)
                state[slot] = D + torch.einsum("h,hk,hv->hkv", s["beta"][b].double(), k, y)
                o[b] = torch.einsum("hk,hkv->hv", q, state[slot]) * s["scale"]
            return {"o": o, "state": state}
        leaves = [t.detach().double().requires_grad_() for t in _leaves(s)]
        x, branch, w, bw = leaves[:4]
        more = leaves[4:]
        with torch.enable_grad():
            u = bw * branch / torch.sqrt(branch.pow(2).mean(-1, keepdim=True) + EPS)
            if s["gate"] is not None:
                a = more.pop(0)
                u = u * (a / (1 + torch.exp(-a)) if case["gate"] == "silu" else 1 / (1 + torch.exp(-a)))
            h = x + (u * more.pop(0) if case["scale"] else u)
            y = w * h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + EPS)
        out = {"out": (y.detach(), h.detach())}
        if case["pass"] == "train":
            out["grads"] = torch.autograd.grad((y, h), leaves, (s["dy"].double(), s["dh"].double()))
        return out
