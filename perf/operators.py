"""Performance cases of the operators behind the convolutions: linear attention with a decay for each head (whole
sequences, and single tokens from a state), the group norm with its gate, and the convolutions' single-token form.

A case is a dict:
    op      "attention"  linear_attention: q, k [B, H, T, K], v [B, H, T, V]
            "step"       linear_attention_step: one token of each of B sequences, states in a cache of `slots` slots
            "norm"       group_norm: x [B, T, D] in `groups` groups of channels
            "conv"       lowrank_dynamic_convolution_step_grouped: one token of each of B sequences, G convolutions
    pass    "train": forward and backward, every gradient returned; "infer": the forward alone
    dtype   of the activations (states and decays are float32)
    layout  (attention) "head": q, k, v are [B, H, T, .] in memory, as the grouped convolution writes them with
            head_dim; "token": [B, T, H, .], as it writes them without
    ragged  (attention) sequences of different lengths up to T (one of them empty where B allows); else all are T long
    state   (attention) starts from a state and returns the new one, as a prompt taken in pieces does

Sizes are those of this repository's benchmark and tests (D 256-4096, T up to 8192, B 1-8, head dims 64 and
128, W 2-16, kernel ranks 8-64), a longer prompt, serving batches, and ragged ones between them.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    at = dict(op="attention", layout="head", ragged=False, state=False)
    gn = dict(op="norm", dtype="bf16", gate=True)
    cv = dict(op="conv", dtype="bf16", G=3, W=4, static=True)
    return [
        # a short question to a small model: latency
        {"name": "at_short", **at, "pass": "infer", "dtype": "bf16", "B": 1, "H": 8, "T": 37, "K": 64, "V": 64,
         "state": True},
        # training: the repository's benchmark shape, and its q|k|v layer
        {"name": "at_train", **at, "pass": "train", "dtype": "bf16", "B": 4, "H": 16, "T": 4096, "K": 128, "V": 128},
        {"name": "at_train_qkv", **at, "pass": "train", "dtype": "bf16", "B": 2, "H": 32, "T": 8192, "K": 128,
         "V": 128, "layout": "token"},
        # the fp32 tier on sizes off the powers of two
        {"name": "at_train_fp32", **at, "pass": "train", "dtype": "fp32", "B": 3, "H": 10, "T": 1537, "K": 100,
         "V": 100, "layout": "token", "ragged": True, "state": True},
        # a piece of a long prompt for one user: few heads' rows, long axis
        {"name": "at_prompt", **at, "pass": "infer", "dtype": "fp16", "B": 1, "H": 16, "T": 32768, "K": 128, "V": 128,
         "state": True},
        # one decoding step: a few sequences, and a serving batch in a cache that holds more of them
        {"name": "step_small", "op": "step", "pass": "infer", "dtype": "bf16", "B": 8, "H": 16, "K": 128, "V": 128,
         "slots": 8},
        {"name": "step_serving", "op": "step", "pass": "infer", "dtype": "bf16", "B": 256, "H": 32, "K": 128, "V": 128,
         "slots": 320},
        # the norm of one decoding step, of the q|k|v layer's training, and of a ragged shape without a gate
        {"name": "norm_decode", **gn, "pass": "infer", "B": 8, "T": 1, "D": 2048, "groups": 16},
        {"name": "norm_train", **gn, "pass": "train", "B": 2, "T": 8192, "D": 4096, "groups": 32},
        {"name": "norm_ragged", **gn, "pass": "train", "dtype": "fp16", "B": 3, "T": 1537, "D": 1000, "groups": 10,
         "gate": False},
        # the q, k and v convolutions of one decoding step
        {"name": "conv_small", **cv, "pass": "infer", "B": 8, "D": 2048, "R": 15, "slots": 8},
        {"name": "conv_serving", **cv, "pass": "infer", "B": 256, "D": 4096, "R": 31, "slots": 320},
    ]


def draw(rng):
    """One case of the same ranges: sizes over their logarithms, ragged ones among them."""

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    cases = {c["name"]: c for c in listed()}
    while True:
        op = rng.choice(["attention"] * 5 + ["step"] * 2 + ["norm"] * 2 + ["conv"] * 2)
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        train = rng.random() < 0.6
        if op == "attention":
            dim = rng.choice([32, 64, 64, 96, 100, 128, 128, 128, 192, 256])
            c = {"B": log(1, 8), "H": log(1, 32), "T": log(1, 32768), "K": dim,
                 "V": rng.choice([dim, dim, dim, 64, 128, 256]), "layout": rng.choice(["head", "token"]),
                 "ragged": rng.random() < 0.3, "state": rng.random() < 0.4}
            if c["T"] > 1 and rng.random() < 0.3:
                c["T"] = 1 << round(math.log2(c["T"]))
            most = "at_train_qkv"
        elif op == "step":
            dim = rng.choice([32, 64, 96, 100, 128, 128, 256])
            train, B = False, log(1, 256)
            c = {"B": B, "H": log(1, 32), "K": dim, "V": rng.choice([dim, dim, 64, 128]), "slots": B + rng.randrange(64)}
            most = "step_serving"
        elif op == "norm":
            size = rng.choice([8, 16, 64, 100, 128, 128, 256, 512])
            groups = log(1, 64)
            c = {"B": log(1, 8), "T": log(256 if train else 1, 8192), "D": size * groups, "groups": groups,
                 "gate": rng.random() < 0.7}
            if c["D"] < 64 or c["D"] > 8192:
                continue
            most = "norm_train"
        else:
            train, B, static = False, log(1, 256), rng.random() < 0.6
            c = {"B": B, "G": rng.choice([1, 3]), "W": rng.choice([2, 3, 4, 4, 4, 8, 16]), "static": static,
                 "D": 128 * max(2, round(log(256, 4096) / 128)), "R": rng.choice([8, 16, 32, 64]) - int(static),
                 "slots": B + rng.randrange(64)}
            most = "conv_serving"
        c.update({"op": op, "pass": "train" if train else "infer", "dtype": dtype})
        widths = [c["H"] * c[n] for n in "KV"] if "H" in c else [c.get("G", 1) * c["D"]]
        if 3072 in list(c.values()) + widths:
            continue
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

    def slots(n, of):
        # the slots that a serving loop has given its running sequences: distinct, in no order
        return torch.randperm(of, generator=g, device=dev)[:n].to(torch.int32)

    s = {"case": case}
    op, B = case["op"], case["B"]
    if op in ("attention", "step"):
        H, K, V = case["H"], case["K"], case["V"]
        s["scale"] = K ** -0.5
        # decays spread over the heads from 1 - 2^-5 to 1 - 2^-12, as retention layers have them
        u = 5 + 7 * torch.rand(H, generator=g, device=dev)
        s["log_decay"] = torch.log1p(-torch.exp2(-u))
    if op == "attention":
        T = case["T"]

        def heads(n):
            t = normal(B, H, T, n) if case["layout"] == "head" else normal(B, T, H, n).transpose(1, 2)
            return t.requires_grad_(train)

        s["q"], s["k"], s["v"] = heads(K), heads(K), heads(V)
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
        s["q"], s["k"], s["v"] = normal(B, H, K), normal(B, H, K), normal(B, H, V)
        s["state"] = normal(case["slots"], H, K, V, dtype=torch.float32)
        s["slots"] = slots(B, case["slots"])
    elif op == "norm":
        T, D = case["T"], case["D"]
        s["x"] = normal(B, T, D, scale=4.0).requires_grad_(train)
        s["gate"] = normal(B, T, D).requires_grad_(train) if case["gate"] else None
        s["weight"] = (1 + normal(D, scale=0.1, dtype=torch.float32)).to(dt).requires_grad_(train)
        s["bias"] = normal(D, scale=0.1).requires_grad_(train)
        s["eps"] = 1e-5
        if train:
            s["dy"] = normal(B, T, D)
    else:
        G, D, R, W = case["G"], case["D"], case["R"], case["W"]
        rank = R + int(case["static"])
        s["x"] = normal(B, G * D)
        s["z"] = [normal(B, R) for _ in range(G)]
        s["U"] = [normal(R, W * D, scale=(rank * W) ** -0.5) for _ in range(G)]
        s["static_w"] = [((torch.rand(W, D, generator=g, device=dev) * 2 - 1) * W ** -0.5).to(dt)
                         for _ in range(G)] if case["static"] else None
        s["state"] = normal(case["slots"], W - 1, G * D)
        s["slots"] = slots(B, case["slots"])
    return s


def _leaves(s):
    names = ("q", "k", "v", "initial") if s["case"]["op"] == "attention" else ("x", "weight", "bias", "gate")
    return [s[n] for n in names if s[n] is not None]


# ---------------------------------------------------------------- the framework's operators
def _own_attention(s):
    from linattn import linear_attention

    c = s["case"]
    train = c["pass"] == "train"
    with torch.set_grad_enabled(train):
        out = linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], initial_state=s["initial"],
                               lengths=s["lengths"], return_state=c["state"])
    out = out if c["state"] else (out,)
    if not train:
        return {"out": out}
    douts = (s["do"], s["dstate"]) if c["state"] else (s["do"],)
    return {"out": out, "grads": torch.autograd.grad(out, _leaves(s), douts)}


def _own_step(s):
    from linattn import linear_attention_step

    o = linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"], slots=s["slots"])
    return {"o": o, "state": s["state"]}


def _own_norm(s):
    from linattn import group_norm

    train = s["case"]["pass"] == "train"
    with torch.set_grad_enabled(train):
        y = group_norm(s["x"], s["case"]["groups"], weight=s["weight"], bias=s["bias"], gate=s["gate"],
                       activation="silu", eps=s["eps"])
    if not train:
        return {"y": y}
    return {"y": y, "grads": torch.autograd.grad(y, _leaves(s), s["dy"])}


def _own_conv(s):
    from lowrank import lowrank_dynamic_convolution_step_grouped

    ys = lowrank_dynamic_convolution_step_grouped(s["x"], s["z"], s["U"], s["state"], static_w=s["static_w"],
                                                  residual=True, slots=s["slots"])
    return {"y": tuple(ys), "state": s["state"]}


# ---------------------------------------------------------------- plain forms
CHUNK = 128


def _rows(t, lengths, dtype=torch.float32):
    """t [B, H, T, n] widened, rows past each sequence's length zero whatever they hold."""
    t = t.detach().to(dtype)
    if lengths is None:
        return t
    live = torch.arange(t.shape[2], device=t.device)[None] < lengths[:, None]
    return torch.where(live[:, None, :, None], t, torch.zeros_like(t))


def _decayed(log_decay, lengths, B, T):
    """Tokens up to and with t that decay the state, times the log of the decay: [B, H, T]."""
    n = torch.arange(1, T + 1, device=log_decay.device)[None].expand(B, T)
    if lengths is not None:
        n = torch.minimum(n, lengths[:, None].to(n.dtype))
    return n[:, None, :] * log_decay[None, :, None].to(torch.float32)


def _plain_attention(s):
    """Chunks of tokens one after another, the state carried between them; the backward from the last chunk on."""
    c = s["case"]
    B, T = c["B"], c["T"]
    q, k, v = (_rows(s[n], s["lengths"]) for n in ("q", "k", "v"))
    live = None if s["lengths"] is None else (torch.arange(T, device=q.device)[None] < s["lengths"][:, None])
    L = _decayed(s["log_decay"], s["lengths"], B, T)
    S = torch.zeros(B, c["H"], c["K"], c["V"], device=q.device)
    if s["initial"] is not None:
        S = S + s["initial"].detach()
    out, states, parts = [], [], []
    before = torch.zeros_like(L[:, :, :1])
    for t in range(0, T, CHUNK):
        a = slice(t, min(t + CHUNK, T))
        n = a.stop - t
        Lc = L[:, :, a] - before
        diff = Lc[..., :, None] - Lc[..., None, :]
        past = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        w = torch.exp(torch.where(past, diff, torch.full_like(diff, -math.inf)))
        wi, wl = torch.exp(Lc)[..., None], torch.exp(Lc[..., -1:] - Lc)[..., None]
        o = wi * (q[:, :, a] @ S) + ((q[:, :, a] @ k[:, :, a].transpose(2, 3)) * w) @ v[:, :, a]
        if live is not None:
            o = o * live[:, None, a, None]
        out.append(o * s["scale"])
        states.append(S)
        parts.append((a, w, wi, wl))
        S = wi[:, :, -1:] * S + (k[:, :, a] * wl).transpose(2, 3) @ v[:, :, a]
        before = L[:, :, a.stop - 1:a.stop]
    outs = (torch.cat(out, 2).to(s["q"].dtype),) + ((S,) if c["state"] else ())
    if c["pass"] == "infer":
        return {"out": outs}
    do = _rows(s["do"], s["lengths"]) * s["scale"]
    dS = s["dstate"].clone() if c["state"] else torch.zeros_like(S)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for (a, w, wi, wl), S in zip(reversed(parts), reversed(states)):
        dp = (do[:, :, a] @ v[:, :, a].transpose(2, 3)) * w
        p = (q[:, :, a] @ k[:, :, a].transpose(2, 3)) * w
        dq[:, :, a] = dp @ k[:, :, a] + wi * (do[:, :, a] @ S.transpose(2, 3))
        dk[:, :, a] = dp.transpose(2, 3) @ q[:, :, a] + wl * (v[:, :, a] @ dS.transpose(2, 3))
        dv[:, :, a] = p.transpose(2, 3) @ do[:, :, a] + wl * (k[:, :, a] @ dS)
        dS = wi[:, :, -1:] * dS + (q[:, :, a] * wi).transpose(2, 3) @ do[:, :, a]
    grads = [dq, dk, dv]
    if live is not None:
        grads = [t * live[:, None, :, None] for t in grads]
    grads = [t.to(s["q"].dtype) for t in grads] + ([dS] if c["state"] else [])
    return {"out": outs, "grads": tuple(grads)}


def _plain_step(s):
    slots = s["slots"].long()
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    S = s["state"][slots] * torch.exp(s["log_decay"])[None, :, None, None] + k[..., :, None] * v[..., None, :]
    s["state"][slots] = S
    o = (q[..., :, None] * S).sum(2) * s["scale"]
    return {"o": o.to(s["q"].dtype), "state": s["state"]}


def _plain_norm(s):
    c = s["case"]
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    shape = x.shape[:-1] + (c["groups"], c["D"] // c["groups"])
    xg = x.reshape(shape)
    mean = xg.mean(-1, keepdim=True)
    rstd = torch.rsqrt(((xg - mean) ** 2).mean(-1, keepdim=True) + s["eps"])
    xhat = ((xg - mean) * rstd)
    u = xhat.reshape(x.shape) * w + b
    a = s["gate"].detach().float() if c["gate"] else u
    sig = 1 / (1 + torch.exp(-a))
    y = u * (a * sig if c["gate"] else sig)
    y = y.to(s["x"].dtype)
    if c["pass"] == "infer":
        return {"y": y}
    dy = s["dy"].float()
    dsilu = sig * (1 + a * (1 - sig))
    du = dy * (a * sig if c["gate"] else dsilu)
    dxh = (du * w).reshape(shape)
    dx = rstd * (dxh - dxh.mean(-1, keepdim=True) - xhat * (dxh * xhat).mean(-1, keepdim=True))
    grads = [dx.reshape(x.shape), (du * xhat.reshape(x.shape)).sum((0, 1)), du.sum((0, 1))]
    if c["gate"]:
        grads.append(dy * u * dsilu)
    return {"y": y, "grads": tuple(t.to(s["x"].dtype) for t in grads)}


def _plain_conv(s):
    c = s["case"]
    D, W, slots = c["D"], c["W"], s["slots"].long()
    # rows t - W + 1 .. t of each sequence
    rows = torch.cat([s["state"][slots], s["x"][:, None]], 1)
    ys = []
    for g in range(c["G"]):
        taps = (s["z"][g].float() @ s["U"][g].float()).view(-1, W, D)
        if c["static"]:
            taps = taps + s["static_w"][g].float()
        x = rows[..., g * D:(g + 1) * D].float()
        ys.append(((taps * x.flip(1)).sum(1) + x[:, -1]).to(s["x"].dtype))
    s["state"][slots] = rows[:, 1:]
    return {"y": tuple(ys), "state": s["state"]}


def run(state):
    """One pass: the outputs, the updated state, and for "train" the gradients of every input."""
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "step": _own_step, "norm": _own_norm, "conv": _own_conv}[op](state)
    with torch.no_grad():
        return {"attention": _plain_attention, "step": _plain_step, "norm": _plain_norm, "conv": _plain_conv}[op](state)


def work(case):
    """Bytes and operations of one pass.  A training pass is two calls (the gradient of the output exists only
    after the forward): each reads its inputs and writes its outputs once.  Operations are those of the recurrent
    form, the cheapest for long sequences (2 a multiply-add), or of the plain triangle for short ones."""
    e = 4 if case["dtype"] == "fp32" else 2
    B, train = case["B"], case["pass"] == "train"
    if case["op"] in ("attention", "step"):
        H, K, V = case["H"], case["K"], case["V"]
        st = 4 * B * H * K * V
        if case["op"] == "step":
            return {"bytes": e * B * H * (2 * K + 2 * V) + 2 * st, "flops": 5 * B * H * K * V}
        n = B * H * case["T"] * (0.5 if case["ragged"] else 1)
        out = B * H * case["T"]  # rows that no length reaches are written too
        byt = n * (2 * K + V) + out * V
        pair = min(2 * K * V, case["T"] * max(K, V))  # one product of a token with a state
        flops = 2 * pair * n
        if train:
            byt += n * (2 * K + 2 * V) + out * (2 * K + V)
            flops += 5 * pair * n
        states = (2 if not train else 4) * st if case["state"] else 0
        return {"bytes": int(e * byt + states), "flops": int(flops)}
    if case["op"] == "norm":
        n = B * case["T"] * case["D"]
        per = 3 if case["gate"] else 2
        return {"bytes": e * n * (per + (per + 2 if train and case["gate"] else per + 1 if train else 0)),
                "flops": n * (14 + (30 if train else 0))}
    G, D, R, W = case["G"], case["D"], case["R"], case["W"]
    rank = R + int(case["static"])
    return {"bytes": e * G * (rank * W * D + B * R + B * D * (2 + 2 * (W - 1))),
            "flops": 2 * B * G * D * W * (rank + 1)}


# ---------------------------------------------------------------- 64 bits, from the definitions
def _exact_attention(s):
    """All pairs of tokens, a block of rows and a head at a time, and the initial state's part apart."""
    c = s["case"]
    B, H, T, lam = c["B"], c["H"], c["T"], s["log_decay"].double()
    sc, train = s["scale"], c["pass"] == "train"
    f64 = dict(dtype=torch.float64, device=lam.device)
    o = torch.zeros(B, H, T, c["V"], **f64)
    S = torch.zeros(B, H, c["K"], c["V"], **f64)
    dq, dk, dv, dS0 = (torch.zeros(B, H, T, c["K"], **f64), torch.zeros(B, H, T, c["K"], **f64),
                       torch.zeros(B, H, T, c["V"], **f64), torch.zeros_like(S))
    lens = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    for b in range(B):
        n = lens[b]
        t = torch.arange(n, **f64)
        for h in range(H):
            q, k, v = (s[x].detach()[b, h, :n].double() for x in ("q", "k", "v"))
            S0 = s["initial"].detach()[b, h].double() if c["state"] else None
            first = torch.exp(lam[h] * (t + 1))[:, None]  # what is left of the initial state
            last = torch.exp(lam[h] * (n - 1 - t))[:, None]  # what the final state holds of a token
            if train:
                do = s["do"][b, h, :n].double() * sc
                dS = s["dstate"][b, h].double() if c["state"] else None
            for r in range(0, n, 2048):
                a = slice(r, min(r + 2048, n))
                gap = t[a, None] - t[None, :a.stop]
                w = torch.where(gap >= 0, torch.exp(lam[h] * gap.clamp(min=0)), torch.zeros_like(gap))
                p = (q[a] @ k[:a.stop].t()) * w
                o[b, h, a] = p @ v[:a.stop] * sc
                if train:
                    dp = (do[a] @ v[:a.stop].t()) * w
                    dq[b, h, a] = dp @ k[:a.stop]
                    dk[b, h, :a.stop] += dp.t() @ q[a]
                    dv[b, h, :a.stop] += p.t() @ do[a]
            S[b, h] = (k * last).t() @ v
            if c["state"]:
                o[b, h, :n] += sc * first * (q @ S0)
                S[b, h] += torch.exp(lam[h] * n) * S0
            if train and c["state"]:
                dq[b, h, :n] += first * (do @ S0.t())
                dk[b, h, :n] += last * (v @ dS.t())
                dv[b, h, :n] += last * (k @ dS)
                dS0[b, h] = (q * first).t() @ do + torch.exp(lam[h] * n) * dS
    out = {"out": (o, S) if c["state"] else (o,)}
    if train:
        out["grads"] = (dq, dk, dv) + ((dS0,) if c["state"] else ())
    return out


def exact(case, seed):
    """run()'s outputs from the same inputs in 64 bits, by the formulas of the operators."""
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attention":
            return _exact_attention(s)
        if case["op"] == "step":
            state = s["state"].double()
            o = torch.empty(case["B"], case["H"], case["V"], dtype=torch.float64, device=state.device)
            for b, slot in enumerate(s["slots"].tolist()):
                state[slot] = (torch.exp(s["log_decay"].double())[:, None, None] * state[slot]
                               + torch.einsum("hk,hv->hkv", s["k"][b].double(), s["v"][b].double()))
                o[b] = torch.einsum("hk,hkv->hv", s["q"][b].double(), state[slot]) * s["scale"]
            return {"o": o, "state": state}
        if case["op"] == "norm":
            leaves = [t.detach().double().requires_grad_() for t in _leaves(s)]
            x, w, b = leaves[:3]
            with torch.enable_grad():
                rows = x.reshape(-1, case["groups"], case["D"] // case["groups"])
                var, mean = torch.var_mean(rows, dim=2, correction=0, keepdim=True)
                u = ((rows - mean) / torch.sqrt(var + s["eps"])).reshape(x.shape) * w + b
                y = u * leaves[3] / (1 + torch.exp(-leaves[3])) if case["gate"] else u / (1 + torch.exp(-u))
            if case["pass"] == "infer":
                return {"y": y.detach()}
            return {"y": y.detach(), "grads": torch.autograd.grad(y, leaves, s["dy"].double())}
        D, W = case["D"], case["W"]
        state, ys = s["state"].double(), []
        x, slots = s["x"].double(), s["slots"].long()
        for g in range(case["G"]):
            c = slice(g * D, (g + 1) * D)
            U = s["U"][g].double().view(-1, W, D)
            y = x[:, c].clone()
            for k in range(W):
                past = x[:, c] if k == 0 else state[slots, W - 1 - k][:, c]
                y += (s["z"][g].double() @ U[:, k].contiguous() + (s["static_w"][g][k].double() if case["static"] else 0)) * past
            ys.append(y)
        for k in range(W - 2):
            state[slots, k] = state[slots, k + 1]
        if W > 1:
            state[slots, W - 2] = x
        return {"y": tuple(ys), "state": state}
