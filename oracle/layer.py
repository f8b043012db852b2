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
