"""The gated delta rule on MI355X: whole sequences (training, prompts) and single tokens.

The operator of layers whose recurrent state is corrected rather than only added to, with a decay and a strength of each
token's own.  With a = exp(log_decay_t) and b = beta_t, for each sequence and head,

    S' = a S_{t-1}                       the state, [K, V], float32
    u  = b (v_t - k_t S')                what the state gets wrong of this token
    S_t = S' + k_t^T u,   o_t = scale * q_t S_t

The reference has no counterpart (its README.md:106-110 stops at q, k, v in heads).  Kernels: csrc/delta*.hip, through
include/dynconv_layer.h.
"""

import torch

from . import _capi
from .linattn import MAX_DIM, _index, _like, _rows, _strides

_NORMALIZE, _PRECISE, _KEEP = 1, 2, 4  # dc_delta_flags


class _GatedDeltaRuleFn(torch.autograd.Function):
    """o, and the final state where it is asked for.  Plain calls take its native form (_capi.binding)."""

    @staticmethod
    @_capi.on_tensor_device
    def forward(ctx, q, k, v, log_decay, beta, initial, lengths, scale, eps, flags, return_state):
        B, Hk, T, K = q.shape
        H, V = v.shape[1], v.shape[-1]
        # token-major memory: the norm and the output projection read [B, T, H * V]
        o = torch.empty(B, T, H, V, dtype=q.dtype, device=q.device).transpose(1, 2)
        state = torch.empty(B, H, K, V, dtype=torch.float32, device=q.device) if return_state else None
        lib = _capi.load()
        dtype, gdtype = _capi.dtype_code(q.dtype), _capi.dtype_code(beta.dtype)
        nws = lib.dc_delta_rule_ws_bytes(B, Hk, H, T, K, V, dtype, flags, 0)
        _capi.check(int(nws) if nws < 0 else 0, "gated delta rule workspace query")
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws > 0 else None
        status = lib.dc_delta_rule_fwd(
            _capi.ptr(q), _strides(q, 3), _capi.ptr(k), _strides(k, 3), _capi.ptr(v), _strides(v, 3),
            _capi.ptr(log_decay), _strides(log_decay, 3), _capi.ptr(beta), _strides(beta, 3), _capi.ptr(initial),
            _capi.ptr(lengths), _capi.ptr(o), _strides(o, 3), _capi.ptr(state), _capi.ptr(ws), nws, B, Hk, H, T, K, V,
            scale, eps, dtype, gdtype, flags, _capi.stream_of(q))
        _capi.check(status, "gated delta rule forward")
        # ws: each chunk's triangular systems and states, a function of the inputs, which the backward takes up again
        ctx.save_for_backward(q, k, v, log_decay, beta, initial, lengths, ws)
        ctx.args = scale, eps, flags
        ctx.set_materialize_grads(False)
        return (o, state) if return_state else o

    @staticmethod
    @_capi.on_tensor_device
    def backward(ctx, do, dstate=None):
        q, k, v, log_decay, beta, initial, lengths, fwd_ws = ctx.saved_tensors
        scale, eps, flags = ctx.args
        B, Hk, T, K = q.shape
        H, V = v.shape[1], v.shape[-1]
        # an output that did not reach the loss has no gradient
        do = torch.zeros(B, H, T, V, dtype=q.dtype, device=q.device) if do is None else _rows(do.to(q.dtype))
        dstate = None if dstate is None else dstate.to(torch.float32).contiguous()
        dq, dk, dv, dg, db = (_like(t) for t in (q, k, v, log_decay, beta))
        dinitial = torch.empty_like(initial) if initial is not None and ctx.needs_input_grad[5] else None
        lib = _capi.load()
        dtype, gdtype = _capi.dtype_code(q.dtype), _capi.dtype_code(beta.dtype)
        nws = lib.dc_delta_rule_ws_bytes(B, Hk, H, T, K, V, dtype, flags, 1 if fwd_ws is None else 2)
        _capi.check(int(nws) if nws < 0 else 0, "gated delta rule backward workspace query")
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws > 0 else None
        status = lib.dc_delta_rule_bwd(
            _capi.ptr(q), _strides(q, 3), _capi.ptr(k), _strides(k, 3), _capi.ptr(v), _strides(v, 3),
            _capi.ptr(log_decay), _strides(log_decay, 3), _capi.ptr(beta), _strides(beta, 3), _capi.ptr(initial),
            _capi.ptr(lengths), _capi.ptr(do), _strides(do, 3), _capi.ptr(dstate), _capi.ptr(dq), _strides(dq, 3),
            _capi.ptr(dk), _strides(dk, 3), _capi.ptr(dv), _strides(dv, 3), _capi.ptr(dg), _strides(dg, 3),
            _capi.ptr(db), _strides(db, 3), _capi.ptr(dinitial), _capi.ptr(fwd_ws), _capi.ptr(ws), nws, B, Hk, H, T, K, V,
            scale, eps, dtype, gdtype, flags, _capi.stream_of(q))
        _capi.check(status, "gated delta rule backward")
        return dq, dk, dv, dg, db, dinitial, None, None, None, None, None


def _check_heads(q, k, v):
    """What whole sequences and single tokens share: q, k [B, Hk, ..., K], v [B, H, ..., V]."""
    assert k.shape == q.shape, "k must have q's shape"
    assert v.shape[0] == q.shape[0] and v.shape[2:-1] == q.shape[2:-1], "v must have q's batch and rows"
    assert q.dtype == k.dtype == v.dtype, "q, k and v must share one dtype"
    assert k.device == q.device and v.device == q.device, "q, k and v must be on one device"
    _capi.dtype_code(q.dtype)
    (B, Hk), K, H, V = q.shape[:2], q.shape[-1], v.shape[1], v.shape[-1]
    assert B > 0 and Hk > 0 and H > 0 and H % Hk == 0, "q's heads must divide v's"
    assert 0 < K <= MAX_DIM and 0 < V <= MAX_DIM, "head dims must be between 1 and 256"


def _check_gates(log_decay, beta, v):
    for t in (log_decay, beta):
        assert t.device == v.device and tuple(t.shape) == tuple(v.shape[:-1]), "log_decay and beta must be v's shape without its channels"
        assert t.dtype in (v.dtype, torch.float32) and t.dtype == beta.dtype, \
            "log_decay and beta must be of q's dtype or float32, both alike"


def gated_delta_rule(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    scale: float | None = None,
    initial_state: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    return_state: bool = False,
    normalize: bool = False,
    eps: float = 1e-6,
):
    """The gated delta rule over whole sequences.

    Args:
        q, k:          [B, Hk, T, K], v: [B, H, T, V] of one dtype (bfloat16, float16, float32), K, V <= 256, in any
                       layout with contiguous channels (as linear_attention).  Hk divides H: head h of v goes with head
                       h // (H // Hk) of q and k.
        log_decay:     [B, H, T], the logarithm of each token's decay (<= 0; -inf forgets at once), beta: [B, H, T], how
                       much of the error is corrected (0 .. 1, or up to 2), both of q's dtype or float32, in any layout.
        scale:         of q; K ** -0.5 if None.
        initial_state: [B, H, K, V] float32, the state before the first token (None: zero).
        lengths:       [B] int32 on the device: sequence b has its first lengths[b] rows (0 .. T).  Rows past them
                       are not used, whatever they hold; their outputs and gradients are zero.
        return_state:  return the state after each sequence's last token too.
        normalize:     divide each row of q and k by sqrt(|row|^2 + eps) (eps >= 0; with 0 no row of a sequence may be
                       zero).  The rule wants keys of at most about that length: a state grows without bound where
                       beta |k|^2 passes 2.

    Returns:
        o [B, H, T, V] in q's dtype, over token-major memory (o.transpose(1, 2).reshape(B, T, H * V) is a view), or
        (o, state [B, H, K, V] float32).  Every input but lengths has a gradient.

    Values are finite: an infinity or NaN reaches its head's outputs from the start of its block of up to 64 tokens on.  In 16
    bits products run on matrix cores with float32 sums; what they take of the states and corrections has 16 bits (for a backward
    in bf16 11, and v's gradients their own 8), so that results are good to little more than their own rounding, unless a
    result is float32: a returned state, or a gradient of float32 gates or of the initial state.  Then everything is as good as
    float32, at two to three times the time.  A |beta| below 2^-60 counts as 2^-60.  Where a backward may follow, the states of
    each block stay in memory for it if they take at most twice that of q, k, v and o.
    """
    if _capi.binding is not None:
        out = _capi.binding.gated_delta_rule(q, k, v, log_decay, beta, scale, initial_state, lengths, return_state, normalize, eps)
        if out is not None:
            return out
    assert q.is_cuda and q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k, v must be [B, heads, T, .] on the GPU"
    _check_heads(q, k, v)
    _check_gates(log_decay, beta, v)
    B, H, _, V = v.shape
    K = q.shape[-1]
    if initial_state is not None:
        assert initial_state.device == q.device and initial_state.dtype == torch.float32, "states are float32"
        assert tuple(initial_state.shape) == (B, H, K, V), "initial_state must be [B, H, K, V]"
        initial_state = initial_state.contiguous()
    lengths = _index(lengths, B, q.device, "lengths")
    scale = K ** -0.5 if scale is None else float(scale)
    flags = (_NORMALIZE if normalize else 0) | (_PRECISE if _wide_results(q, log_decay, beta, initial_state, return_state) else 0)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, beta, initial_state)):
        flags |= _KEEP
    return _GatedDeltaRuleFn.apply(_rows(q), _rows(k), _rows(v), log_decay, beta, initial_state, lengths, scale, float(eps),
                                   flags, bool(return_state))


def _wide_results(q, log_decay, beta, initial, return_state) -> bool:
    """Whether a result of a call in 16 bits is float32: a state, or a gradient of the gates or of the initial state."""
    if q.dtype == torch.float32:
        return False
    grads = [t for t in (log_decay, beta, initial) if t is not None and t.dtype == torch.float32 and t.requires_grad]
    return return_state or (torch.is_grad_enabled() and bool(grads))


def gated_delta_rule_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    state: torch.Tensor,
    scale: float | None = None,
    slots: torch.Tensor | None = None,
    normalize: bool = False,
    eps: float = 1e-6,
) -> torch.Tensor:
    """gated_delta_rule for one more token of each sequence; `state` is updated in place.

    Args:
        q, k:      [B, Hk, K], v: [B, H, V] of one dtype, contiguous channels.
        log_decay, beta: [B, H] of q's dtype or float32.
        state:     [slots, H, K, V] float32, contiguous: a cache of states.
        slots:     [B] int32 on the device, the row of `state` of each sequence; distinct, except that ids outside
                   the cache (-1) mark sequences that take no part: their outputs are zero.  None: row b.

    Returns:
        o [B, H, V] in q's dtype.  Serving only: no gradients; a backward that has saved `state` from before raises, as
        after torch's own in-place operations.
    """
    if _capi.binding is not None:
        o = _capi.binding.gated_delta_rule_step(q, k, v, log_decay, beta, state, scale, slots, normalize, eps)
        if o is not None:
            return o
    assert q.is_cuda and q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "q, k, v must be [B, heads, .] on the GPU"
    _check_heads(q, k, v)
    _check_gates(log_decay, beta, v)
    assert not _capi.differentiated((q, k, v, log_decay, beta, state)), \
        "gated_delta_rule_step has no gradient and no tangent: call it under torch.no_grad(), without dual tensors"
    (B, H, V), K = v.shape, q.shape[-1]
    assert state.device == q.device and state.dtype == torch.float32 and state.is_contiguous(), \
        "state must be contiguous float32 on q's device"
    assert state.dim() == 4 and tuple(state.shape[1:]) == (H, K, V), "state must be [slots, H, K, V]"
    assert slots is not None or B <= state.shape[0], "more sequences than rows of state"
    slots = _index(slots, B, q.device, "slots")
    scale = K ** -0.5 if scale is None else float(scale)
    return _step(_rows(q), _rows(k), _rows(v), log_decay, beta, state, slots, scale, float(eps), _NORMALIZE if normalize else 0)


@_capi.on_first_device
def _step(q, k, v, log_decay, beta, state, slots, scale, eps, flags):
    B, Hk, K = q.shape
    H, V = v.shape[1:]
    o = torch.empty(B, H, V, dtype=q.dtype, device=q.device)
    status = _capi.load().dc_delta_rule_step(
        _capi.ptr(q), _strides(q, 2), _capi.ptr(k), _strides(k, 2), _capi.ptr(v), _strides(v, 2), _capi.ptr(log_decay),
        _strides(log_decay, 2), _capi.ptr(beta), _strides(beta, 2), _capi.ptr(state), _capi.ptr(slots), _capi.ptr(o), B, Hk,
        H, K, V, state.shape[0], scale, eps, _capi.dtype_code(q.dtype), _capi.dtype_code(beta.dtype), flags,
        _capi.stream_of(q))
    _capi.check(status, "gated delta rule step")
    _capi.written(state)
    return o
