"""Group norm over the channels of each row, with an activation or a gate, on MI355X.

The norm of linear attention's heads (whose outputs have no scale of their
own) before the output projection.  Channels last and row by row, so a token
does not see another: with T = 1 it is its own form for single tokens.  The
reference has no counterpart.  Kernels: csrc/group_norm.hip.
"""

import torch

from . import _capi

ACTIVATIONS = {None: 0, "silu": 1}  # dc_activation
MAX_GROUP = 4096  # channels of a group


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
