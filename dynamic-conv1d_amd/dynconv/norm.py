"""Norms of rows on MI355X: the group norm with an activation or a gate, and the norms around a block.

The norm of linear attention's heads (whose outputs have no scale of their
own) before the output projection.  Channels last and row by row, so a token
does not see another: with T = 1 it is its own form for single tokens.

residual_norm is what stands between two blocks of a model: the norm of the
block's output, its gate and scale, the residual sum, and the norm before the
next block, in one pass over the rows.

The reference has no counterpart.  Kernels: csrc/group_norm.hip, csrc/residual_norm.hip.
"""

import torch

from . import _capi

ACTIVATIONS = {None: 0, "silu": 1}  # dc_activation
MAX_GROUP = 4096  # channels of a group
GATE_ACTIVATIONS = {**ACTIVATIONS, "sigmoid": 2}
MAX_ROW = 8192  # DC_RN_MAX_DIM


class _GroupNormFn(torch.autograd.Function):
    """Plain calls take its native form (_capi.binding)."""

    @staticmethod
    @_capi.on_tensor_device
    def forward(ctx, x, weight, bias, gate, groups, act, eps):
        D = x.shape[-1]
        M = x.numel() // D
        y = torch.empty_like(x)
        param = weight if weight is not None else bias
        pdtype = _capi.dtype_code(x.dtype if param is None else param.dtype)
        dtype = _capi.dtype_code(x.dtype)
        if M > 0:
            status = _capi.load().dc_group_norm_fwd(
                _capi.ptr(x), _capi.ptr(weight), _capi.ptr(bias), _capi.ptr(gate), _capi.ptr(y), M, D, groups, eps, act,
                dtype, pdtype, _capi.stream_of(x))
            _capi.check(status, "group norm forward")
        ctx.save_for_backward(x, weight, bias, gate)
        ctx.args = M, D, groups, eps, act, dtype, pdtype
        return y

    @staticmethod
    @_capi.on_tensor_device
    def backward(ctx, dy):
        x, weight, bias, gate = ctx.saved_tensors
        M, D, groups, eps, act, dtype, pdtype = ctx.args
        dy = dy.to(x.dtype).contiguous()
        dx = torch.empty_like(x)
        dgate = None if gate is None else torch.empty_like(gate)
        want_w = weight is not None and ctx.needs_input_grad[1]
        want_b = bias is not None and ctx.needs_input_grad[2]
        if M == 0:
            return (dx, torch.zeros_like(weight) if want_w else None, torch.zeros_like(bias) if want_b else None, dgate,
                    None, None, None)
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        lib = _capi.load()
        nws = lib.dc_group_norm_bwd_ws_bytes(M, D, groups, dtype) if want_w or want_b else 0
        _capi.check(int(nws) if nws < 0 else 0, "group norm backward workspace query")
        ws = torch.empty(nws, dtype=torch.uint8, device=x.device) if nws > 0 else None
        status = lib.dc_group_norm_bwd(
            _capi.ptr(x), _capi.ptr(weight), _capi.ptr(bias), _capi.ptr(gate), _capi.ptr(dy), _capi.ptr(dx),
            _capi.ptr(dgate), _capi.ptr(dw), _capi.ptr(db), _capi.ptr(ws), nws, M, D, groups, eps, act, dtype, pdtype,
            _capi.stream_of(x))
        _capi.check(status, "group norm backward")
        return dx, dw, db, dgate, None, None, None


def group_norm(
    x: torch.Tensor,
    groups: int,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    activation: str | None = "silu",
    eps: float = 1e-5,
) -> torch.Tensor:
    """Normalise each row's groups of neighbouring channels, then activate, or gate.

        u = (x - mean) / sqrt(var + eps) * weight + bias       mean and (biased) variance of each row and group
        y = u * act(gate)  with a gate,   y = act(u)  without

    Args:
        x:          [..., D], contiguous (bfloat16, float16 or float32), e.g. linear attention's heads side by side.
        groups:     of D // groups channels each (at most 4096).
        weight, bias: [D], of x's dtype or float32 (both alike), or None.
        gate:       like x, or None.
        activation: "silu" or None (the identity).
        eps:        added to the variance.

    Returns:
        y like x.  Statistics and sums are float32; results are the same run to run.
    """
    if _capi.binding is not None and activation in ACTIVATIONS:
        y = _capi.binding.group_norm(x, groups, weight, bias, gate, ACTIVATIONS[activation], eps)
        if y is not None:
            return y
    assert x.is_cuda and x.dim() >= 1 and x.is_contiguous(), "x must be contiguous, on the GPU"
    _capi.dtype_code(x.dtype)
    D = x.shape[-1]
    groups = int(groups)
    assert groups > 0 and D > 0 and D % groups == 0, "groups must divide the channels"
    assert D // groups <= MAX_GROUP, "a group holds at most 4096 channels"
    assert activation in ACTIVATIONS, f"activation must be one of {list(ACTIVATIONS)}"
    params = [p for p in (weight, bias) if p is not None]
    for p in params:
        assert p.device == x.device and p.is_contiguous() and tuple(p.shape) == (D,), "weight and bias must be [D]"
        assert p.dtype in (x.dtype, torch.float32) and p.dtype == params[0].dtype, \
            "weight and bias must be of x's dtype or float32, both alike"
    if gate is not None:
        assert gate.shape == x.shape and gate.dtype == x.dtype and gate.device == x.device, "gate must be like x"
        gate = gate.contiguous()
    return _GroupNormFn.apply(x, weight, bias, gate, groups, ACTIVATIONS[activation], float(eps))


class _ResidualNormFn(torch.autograd.Function):
    """(y, h).  Plain calls take its native form (_capi.binding)."""

    @staticmethod
    @_capi.on_tensor_device
    def forward(ctx, x, branch, weight, branch_weight, gate, scale, constant, act, eps):
        D = x.shape[-1]
        M = x.numel() // D
        y, h = torch.empty_like(branch), torch.empty_like(x)
        param = next((p for p in (weight, branch_weight, scale) if p is not None), branch)
        codes = tuple(_capi.dtype_code(t.dtype) for t in (branch, x, param))
        if M > 0:
            status = _capi.load().dc_residual_norm_fwd(
                _capi.ptr(x), _capi.ptr(branch), _capi.ptr(weight), _capi.ptr(branch_weight), _capi.ptr(gate),
                _capi.ptr(scale), _capi.ptr(y), _capi.ptr(h), M, D, constant, eps, act, *codes, _capi.stream_of(x))
            _capi.check(status, "residual norm forward")
        ctx.save_for_backward(h, branch, weight, branch_weight, gate, scale)
        ctx.args = M, D, constant, eps, act, codes
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @_capi.on_tensor_device
    def backward(ctx, dy, dh):
        h, branch, weight, branch_weight, gate, scale = ctx.saved_tensors
        M, D, constant, eps, act, codes = ctx.args
        # an output that did not reach the loss has no gradient
        dy = None if dy is None else dy.to(branch.dtype).contiguous()
        dh = None if dh is None else dh.to(h.dtype).contiguous()
        dx, dbranch = torch.empty_like(h), torch.empty_like(branch)
        dgate = None if gate is None else torch.empty_like(gate)
        new = torch.zeros_like if M == 0 else torch.empty_like
        dw, dbw, ds = (new(p) if p is not None and ctx.needs_input_grad[i] else None
                       for i, p in ((2, weight), (3, branch_weight), (5, scale)))
        if M > 0:
            lib = _capi.load()
            sums = any(t is not None for t in (dw, dbw, ds))
            nws = lib.dc_residual_norm_bwd_ws_bytes(M, D, codes[0]) if sums else 0
            _capi.check(int(nws) if nws < 0 else 0, "residual norm backward workspace query")
            ws = torch.empty(nws, dtype=torch.uint8, device=h.device) if nws > 0 else None
            status = lib.dc_residual_norm_bwd(
                *(_capi.ptr(t) for t in (h, branch, weight, branch_weight, gate, scale, dy, dh, dx, dbranch, dgate, dw, dbw,
                                         ds, ws)), nws, M, D, constant, eps, act, *codes, _capi.stream_of(h))
            _capi.check(status, "residual norm backward")
        return dx, dbranch, dw, dbw, dgate, ds, None, None, None


def residual_norm(
    x: torch.Tensor,
    branch: torch.Tensor,
    weight: torch.Tensor | None = None,
    branch_weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    activation: str | None = None,
    scale: torch.Tensor | float | None = None,
    eps: float = 1e-6,
):
    """The norm after a block, its gate and residual scale, the residual sum, and the norm before the next block.

        u = branch / sqrt(mean(branch^2) + eps) * branch_weight      over each row's channels
        h = x + scale * act(gate) * u
        y = h / sqrt(mean(h^2) + eps) * weight

    Args:
        x:          [..., D], the residual stream, of branch's dtype or float32, contiguous, D <= 8192.
        branch:     like x in shape (bfloat16, float16 or float32), contiguous: the block's output.
        weight, branch_weight: [D], of branch's dtype or float32 (scale's too, where it is a tensor), or None.
        gate:       like branch, or None: no factor.
        activation: of the gate: "silu", "sigmoid" or None (the gate itself).
        scale:      [D], a number, or None.

    Returns:
        (y, h): the next block's input in branch's dtype, and the residual stream in x's; h is rounded to x's dtype before
        its norm.  Statistics and sums are float32; results are the same run to run.
    """
    constant = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        constant, scale = float(scale), None
    if _capi.binding is not None and activation in GATE_ACTIVATIONS:
        out = _capi.binding.residual_norm(x, branch, weight, branch_weight, gate, GATE_ACTIVATIONS[activation], scale, constant, eps)
        if out is not None:
            return out
    assert x.is_cuda and x.dim() >= 1 and x.is_contiguous(), "x must be contiguous, on the GPU"
    assert branch.shape == x.shape and branch.device == x.device and branch.is_contiguous(), \
        "branch must be like x, contiguous"
    _capi.dtype_code(branch.dtype)
    assert x.dtype in (branch.dtype, torch.float32), "x must be of branch's dtype or float32"
    D = x.shape[-1]
    assert 0 < D <= MAX_ROW, "rows have between 1 and 8192 channels"
    assert activation in GATE_ACTIVATIONS, f"activation must be one of {list(GATE_ACTIVATIONS)}"
    assert gate is not None or activation is None, "an activation is the gate's"
    params = [p for p in (weight, branch_weight, scale) if p is not None]
    for p in params:
        assert p.device == x.device and p.is_contiguous() and tuple(p.shape) == (D,), \
            "weight, branch_weight and scale must be [D]"
        assert p.dtype in (branch.dtype, torch.float32) and p.dtype == params[0].dtype, \
            "weight, branch_weight and scale must be of branch's dtype or float32, all alike"
    if gate is not None:
        assert gate.shape == x.shape and gate.dtype == branch.dtype and gate.device == x.device, "gate must be like branch"
        gate = gate.contiguous()
    return _ResidualNormFn.apply(x, branch, weight, branch_weight, gate, scale, constant, GATE_ACTIVATIONS[activation],
                                 float(eps))
