"""float64 restatements of the operators behind the convolutions (test infrastructure only), by their recurrences,
differentiable through autograd.  The reference has no counterpart; tests/test_oracle_layer.py pins them on
hand-computed values, by a second formulation and by torch.autograd.gradcheck.
"""

import torch


def linear_attention_ref(q, k, v, log_decay, scale, initial=None, lengths=None):
    """(o, final state) of S_t = g S_{t-1} + k_t^T v_t, o_t = scale q_t S_t, token by token in float64.

    q, k [B, H, T, K], v [B, H, T, V], log_decay [H], initial [B, H, K, V] or None, lengths: list of B ints or None."""
    B, H, T, K = q.shape
    V = v.shape[-1]
    g = torch.exp(log_decay.double())[None, :, None, None]
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if initial is None else initial.double()
    n = [T] * B if lengths is None else lengths
    rows = []
    for t in range(T):
        live = torch.tensor([t < m for m in n])[:, None, None, None]
        # rows past the length are not used, whatever they hold
        kt, vt, qt = (torch.where(live[..., 0], x[:, :, t].double(), torch.zeros((), dtype=torch.float64))
                      for x in (k, v, q))
        S = torch.where(live, g * S + kt[..., :, None] * vt[..., None, :], S)
        rows.append(scale * (qt[..., :, None] * S).sum(2))
    o = torch.stack(rows, 2) if T else torch.zeros(B, H, 0, V, dtype=torch.float64)
    return o, S


def group_norm_ref(x, groups, weight=None, bias=None, gate=None, activation="silu", eps=1e-5):
    """Group norm of each row's channel groups, then act(u) or u act(gate), in float64."""
    D = x.shape[-1]
    r = x.double().reshape(-1, groups, D // groups)
    mean = r.mean(-1, keepdim=True)
    var = ((r - mean) ** 2).mean(-1, keepdim=True)
    u = ((r - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    u = u if weight is None else u * weight.double()
    u = u if bias is None else u + bias.double()
    a = u if gate is None else gate.double()
    act = a / (1 + torch.exp(-a)) if activation == "silu" else a
    return act if gate is None else u * act


def lowrank_step_ref(x, z, U, state, static_w=None, residual=False):
    """(y [N, D], new state) of one token x [N, D] after the rows state [N, W-1, D], in float64."""
    N, D = x.shape
    W = U.shape[-1] // D
    rows = torch.cat([state.double(), x.double()[:, None]], 1)
    taps = (z.double() @ U.double()).view(N, W, D)
    if static_w is not None:
        taps = taps + static_w.double()
    y = sum(taps[:, w] * rows[:, W - 1 - w] for w in range(W))
    return (y + x.double() if residual else y), rows[:, 1:]


def gated_delta_rule_ref(q, k, v, log_decay, beta, scale, initial=None, lengths=None, normalize=False, eps=1e-6):
    """(o, final state) of S' = a S, u = b (v - k S'), S = S' + k^T u, o = scale q S, token by token in float64.

    q, k [B, Hk, T, K], v [B, H, T, V], log_decay, beta [B, H, T], initial [B, H, K, V] or None, lengths: list of ints."""
    (B, Hk, T, K), H, V = q.shape, v.shape[1], v.shape[-1]
    zero = torch.zeros((), dtype=torch.float64)
    live = torch.ones(B, T, dtype=torch.bool) if lengths is None else torch.arange(T)[None] < torch.tensor(lengths)[:, None]

    def rows(t):  # rows past the length are not used, whatever they hold
        return torch.where(live[:, None, :, None], t.double(), zero)

    def unit(t):
        n = torch.sqrt((t * t).sum(-1, keepdim=True) + eps)
        return t / torch.where(live[:, None, :, None], n, zero + 1) if normalize else t

    q, k = (unit(rows(t)).repeat_interleave(H // Hk, 1) for t in (q, k))
    v = rows(v)
    b = torch.where(live[:, None], beta.double(), zero)
    a = torch.exp(torch.where(live[:, None], log_decay.double(), zero))
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if initial is None else initial.double()
    out = []
    for t in range(T):
        S = a[:, :, t, None, None] * S
        u = b[:, :, t, None] * (v[:, :, t] - (k[:, :, t, :, None] * S).sum(2))
        S = S + k[:, :, t, :, None] * u[:, :, None, :]
        out.append(scale * (q[:, :, t, :, None] * S).sum(2))
    o = torch.stack(out, 2) if T else torch.zeros(B, H, 0, V, dtype=torch.float64)
    return torch.where(live[:, None, :, None], o, zero), S


def gated_delta_rule_chunked(q, k, v, log_decay, beta, scale, do, initial=None, dstate=None, lengths=None, normalize=False,
                             eps=1e-6, chunk=64, dtype=torch.float64, r=lambda t: t, before=None):
    """(o, final state), (dq, dk, dv, dlog_decay, dbeta, dinitial) by the chunked formulas of csrc/delta.hip, in `dtype`, with
    r() applied to the operands of products that the kernels round.  It says how far those roundings alone take a result.
    `before`, a list, is given the gradients of q's and k's normed rows over the rows' norms, what dq and dk are the
    difference of when those lie along the rows."""
    (B, Hk, T, K), H, V = q.shape, v.shape[1], v.shape[-1]
    N = -(-T // chunk)
    live = torch.ones(B, T, dtype=torch.bool) if lengths is None else torch.arange(T)[None] < torch.tensor(lengths)[:, None]

    def cut(t, dtype=dtype):  # [B, H, N, chunk, ...]
        t = torch.where(live.view(B, 1, T, *[1] * (t.dim() - 3)), t.to(dtype), torch.zeros((), dtype=dtype))
        full = torch.zeros(*t.shape[:2], N * chunk, *t.shape[3:], dtype=dtype)
        full[:, :, :T] = t
        return full.view(*t.shape[:2], N, chunk, *t.shape[3:])

    def whole(t):
        return t.flatten(2, 3)[:, :, :T]

    tokens = cut(torch.ones(B, 1, T)) > 0  # rows behind the last are none: whatever eps is, nothing comes of them

    def heads(t):
        t = cut(t)
        n = torch.where(tokens[..., None], torch.sqrt((t * t).sum(-1, keepdim=True) + eps), torch.inf)
        n = 1 / n if normalize else torch.ones_like(t[..., :1])
        return (t * n).repeat_interleave(H // Hk, 1), n

    (qh, nq), (kh, nk) = heads(q), heads(k)
    qh, v, b, do = qh * scale, cut(v), cut(beta)[..., None], cut(do)
    b = torch.where(b.abs() < 2.0**-60, torch.full_like(b, 2.0**-60), b)
    c = cut(log_decay, torch.float64).clamp(min=-128).cumsum(-1)
    low = torch.ones(chunk, chunk, dtype=torch.bool).tril()
    E = torch.exp(torch.where(low, c[..., :, None] - c[..., None, :], -torch.inf)).to(dtype)
    G, D, Gl = (torch.exp(t).to(dtype) for t in (c[..., None], (c[..., -1:] - c)[..., None], c[..., -1][..., None, None]))
    bj = b.transpose(3, 4)
    P = r((qh @ kh.transpose(3, 4)) * E * bj)
    A = ((kh @ kh.transpose(3, 4)) * E * bj).tril(-1)
    M = r(torch.linalg.solve_triangular(A + torch.eye(chunk, dtype=dtype), torch.eye(chunk, dtype=dtype).expand_as(A),
                                        upper=False, unitriangular=True))
    S = torch.zeros(B, H, K, V, dtype=dtype) if initial is None else initial.to(dtype)
    states, Zs, o = [], [], []
    for n in range(N):
        states.append(r(S))
        Z = M[:, :, n] @ r(v[:, :, n] - G[:, :, n] * (kh[:, :, n] @ states[-1]))
        Zs.append(Z)
        o.append(G[:, :, n] * (qh[:, :, n] @ states[-1]) + P[:, :, n] @ r(Z))
        S = Gl[:, :, n] * S + kh[:, :, n].transpose(2, 3) @ r((D * b)[:, :, n] * Z)
    if N == 0:
        return (torch.zeros(B, H, 0, V, dtype=dtype), S), None
    Ss, Z, o = torch.stack(states, 2), torch.stack(Zs, 2), torch.stack(o, 2)
    dS = torch.zeros_like(S) if dstate is None else dstate.to(dtype)
    last, dX = [None] * N, [None] * N
    for n in reversed(range(N)):
        last[n] = r(dS)
        Y = P[:, :, n].transpose(2, 3) @ do[:, :, n] + (D * b)[:, :, n] * (kh[:, :, n] @ last[n])
        dX[n] = M[:, :, n].transpose(2, 3) @ r(Y)
        dS = (Gl[:, :, n] * dS + qh[:, :, n].transpose(2, 3) @ r(G[:, :, n] * do[:, :, n])
              - kh[:, :, n].transpose(2, 3) @ r(G[:, :, n] * dX[n]))
    last, dX = torch.stack(last, 2), torch.stack(dX, 2)
    after = torch.cat([Ss[:, :, 1:], S[:, :, None]], 2)
    Zr, Xr = r(Z), r(dX)
    PE = r((do @ Zr.transpose(3, 4)).tril() * E * bj)
    NZ = -(Xr @ Zr.transpose(3, 4))
    NE = r(NZ.tril(-1) * E * bj)
    dq = G * (do @ Ss.transpose(3, 4)) + PE @ kh
    W = PE.transpose(3, 4) @ qh + D * b * (Zr @ last.transpose(3, 4)) + NE.transpose(3, 4) @ kh
    R = NE @ kh - G * (Xr @ Ss.transpose(3, 4))
    dc = (qh * dq).sum(-1) + (kh * (R - W)).sum(-1)
    dg = dc.flip(-1).cumsum(-1).flip(-1) + (after * last).sum((-1, -2))[..., None]
    db = -torch.diagonal(NZ, dim1=-2, dim2=-1) / b[..., 0]

    def back(dt, t, n, s=1.0):
        dt, t = (x.unflatten(1, (Hk, H // Hk)) for x in (dt * s, t / s))
        dt, t = dt.sum(2), t[:, :, 0]
        if before is not None:
            before.append(whole(n * dt))
        return n * (dt - t * (t * dt).sum(-1, keepdim=True)) if normalize else dt

    grads = [whole(t) for t in (back(dq, qh, nq, scale), back(R + W, kh, nk), dX, dg, db)]
    grads = [torch.where(live.view(B, 1, T, *[1] * (t.dim() - 3)), t, torch.zeros((), dtype=dtype)) for t in grads]
    return (torch.where(live[:, None, :, None], whole(o), torch.zeros((), dtype=dtype)), S), (*grads, dS)


def residual_norm_ref(x, branch, weight=None, branch_weight=None, gate=None, activation=None, scale=None, eps=1e-6):
    """(y, h) of the norms around a block, its gate, scale and the residual sum, in float64."""
    x, u = x.double(), branch.double()
    u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + eps)
    u = u if branch_weight is None else u * branch_weight.double()
    if gate is not None:
        a = gate.double()
        u = u * {"silu": a / (1 + torch.exp(-a)), "sigmoid": 1 / (1 + torch.exp(-a)), None: a}[activation]
    if scale is not None:
        u = u * (scale.double() if isinstance(scale, torch.Tensor) else scale)
    h = x + u
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.double()), h
