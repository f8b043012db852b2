"""Linear attention with a decay for each head on MI355X: whole sequences (training, prompts) and single tokens.

The operator that takes the q, k and v of the convolutions in layers with a
recurrent state instead of softmax attention.  With g = exp(log_decay[h]), for
each sequence and head,

    S_t = g S_{t-1} + k_t^T v_t          the state, [K, V], float32
    o_t = scale * q_t S_t

The reference has no counterpart (its README.md:106-110 stops at q, k, v in
heads).  Kernels: csrc/linattn*.hip, through include/dynconv_layer.h.
"""

import torch

from . import _capi
from .norm import group_norm  # noqa: F401

MAX_DIM = 256  # DC_LA_MAX_DIM


def _strides(t, n):
    return _capi.int64_array(t.stride()[:n])


def _rows(t):
    """t with contiguous channels (copied if they are not)."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _like(t):
    """An empty tensor of t's shape and layout (contiguous where t's elements overlap or leave gaps)."""
    return torch.empty_like(t)


class _LinearAttentionFn(torch.autograd.Function):
    """o, and the final state where it is asked for.  Plain calls take its native form (_capi.binding)."""

    @staticmethod
    @_capi.on_tensor_device
    def forward(ctx, q, k, v, initial, log_decay, lengths, scale, return_state):
        B, H, T, K = q.shape
        V = v.shape[-1]
        # token-major memory: the norm and the output projection read [B, T, H * V]
        o = torch.empty(B, T, H, V, dtype=q.dtype, device=q.device).transpose(1, 2)
        state = torch.empty(B, H, K, V, dtype=torch.float32, device=q.device) if return_state else None
        lib = _capi.load()
        dtype = _capi.dtype_code(q.dtype)
        nws = lib.dc_linear_attention_ws_bytes(B, H, T, K, V, dtype, 0)
        _capi.check(int(nws) if nws < 0 else 0, "linear attention workspace query")
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws > 0 else None
        status = lib.dc_linear_attention_fwd(
            _capi.ptr(q), _strides(q, 3), _capi.ptr(k), _strides(k, 3), _capi.ptr(v), _strides(v, 3),
            _capi.ptr(log_decay), _capi.ptr(initial), _capi.ptr(lengths), _capi.ptr(o), _strides(o, 3),
            _capi.ptr(state), _capi.ptr(ws), nws, B, H, T, K, V, scale, dtype, _capi.stream_of(q))
        _capi.check(status, "linear attention forward")
        # ws: the states before each segment, a function of the inputs, which the backward starts from
        ctx.save_for_backward(q, k, v, initial, log_decay, lengths, ws)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (o, state) if return_state else o

    @staticmethod
    @_capi.on_tensor_device
    def backward(ctx, do, dstate=None):
        q, k, v, initial, log_decay, lengths, states = ctx.saved_tensors
        B, H, T, K = q.shape
        V = v.shape[-1]
        # an output that did not reach the loss has no gradient
        do = torch.zeros(B, H, T, V, dtype=q.dtype, device=q.device) if do is None else _rows(do.to(q.dtype))
        dstate = None if dstate is None else dstate.to(torch.float32).contiguous()
        dq, dk, dv = _like(q), _like(k), _like(v)
        dinitial = torch.empty_like(initial) if initial is not None and ctx.needs_input_grad[3] else None
        lib = _capi.load()
        dtype = _capi.dtype_code(q.dtype)
        nws = lib.dc_linear_attention_ws_bytes(B, H, T, K, V, dtype, 1 if states is None else 2)
        _capi.check(int(nws) if nws < 0 else 0, "linear attention backward workspace query")
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws > 0 else None
        status = lib.dc_linear_attention_bwd(
            _capi.ptr(q), _strides(q, 3), _capi.ptr(k), _strides(k, 3), _capi.ptr(v), _strides(v, 3),
            _capi.ptr(log_decay), _capi.ptr(initial), _capi.ptr(lengths), _capi.ptr(do), _strides(do, 3),
            _capi.ptr(dstate), _capi.ptr(dq), _strides(dq, 3), _capi.ptr(dk), _strides(dk, 3), _capi.ptr(dv),
            _strides(dv, 3), _capi.ptr(dinitial), _capi.ptr(states), _capi.ptr(ws), nws, B, H, T, K, V, ctx.scale, dtype,
            _capi.stream_of(q))
        _capi.check(status, "linear attention backward")
        return dq, dk, dv, dinitial, None, None, None, None


def _check_decay(log_decay, H, device):
    assert log_decay.device == device and log_decay.is_contiguous(), "log_decay must be contiguous, on q's device"
    assert log_decay.dtype == torch.float32 and tuple(log_decay.shape) == (H,), "log_decay must be float32 [H]"
    assert not (log_decay.requires_grad and torch.is_grad_enabled()), \
        "log_decay is a constant of the operator: it has no gradient here"


def _index(t, n, device, name):
    """A vector of n int32 indexes on the device (int64 is converted)."""
    if t is None:
        return None
    assert t.device == device and t.dtype in (torch.int32, torch.int64), f"{name} must be int32, on q's device"
    assert tuple(t.shape) == (n,), f"{name} must have one entry a sequence"
    return _capi.int32(t)


def linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    scale: float | None = None,
    initial_state: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    return_state: bool = False,
):
    """Causal linear attention over whole sequences, with a decay for each head.

    Args:
        q, k:          [B, H, T, K], v: [B, H, T, V] of one dtype (bfloat16, float16, float32), K, V <= 256, in any
                       layout with contiguous channels: the [B, H, T, hd] outputs of the grouped convolution with
                       head_dim, or its [B, T, D] outputs as .view(B, T, H, hd).transpose(1, 2).  Heads that share
                       keys or values may be expanded views.
        log_decay:     [H] float32, the logarithm of each head's decay per token (<= 0; -inf forgets at once).  A
                       constant: no gradient.
        scale:         of the scores; K ** -0.5 if None.
        initial_state: [B, H, K, V] float32, the state before the first token (None: zero).
        lengths:       [B] int32 on the device: sequence b has its first lengths[b] rows (0 .. T).  Rows past them
                       are not used, whatever they hold; their outputs and gradients are zero.
        return_state:  return the state after each sequence's last token too.

    Returns:
        o [B, H, T, V] in q's dtype, over token-major memory (o.transpose(1, 2).reshape(B, T, H * V) is a view), or
        (o, state [B, H, K, V] float32).

    Products of 16-bit inputs run on matrix cores with float32 sums; the state is float32 throughout.  As operands of such
    products the decayed scores, and the state where a token's q meets it, are rounded to the inputs' type; a caller who
    wants neither rounded passes q, k and v in float32.
    """
    if _capi.binding is not None:
        out = _capi.binding.linear_attention(q, k, v, log_decay, scale, initial_state, lengths, return_state)
        if out is not None:
            return out
    assert q.is_cuda and q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k, v must be [B, H, T, .] on the GPU"
    B, H, T, K = q.shape
    assert k.shape == q.shape, "k must have q's shape"
    assert v.shape[:3] == q.shape[:3], "v must be [B, H, T, V]"
    assert q.dtype == k.dtype == v.dtype, "q, k and v must share one dtype"
    assert k.device == q.device and v.device == q.device, "q, k and v must be on one device"
    _capi.dtype_code(q.dtype)
    V = v.shape[-1]
    assert B > 0 and H > 0 and 0 < K <= MAX_DIM and 0 < V <= MAX_DIM, "head dims must be between 1 and 256"
    _check_decay(log_decay, H, q.device)
    if initial_state is not None:
        assert initial_state.device == q.device and initial_state.dtype == torch.float32, "states are float32"
        assert tuple(initial_state.shape) == (B, H, K, V), "initial_state must be [B, H, K, V]"
        initial_state = initial_state.contiguous()
    lengths = _index(lengths, B, q.device, "lengths")
    scale = K ** -0.5 if scale is None else float(scale)
    return _LinearAttentionFn.apply(_rows(q), _rows(k), _rows(v), initial_state, log_decay, lengths, scale,
                                    bool(return_state))


def linear_attention_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    state: torch.Tensor,
    scale: float | None = None,
    slots: torch.Tensor | None = None,
) -> torch.Tensor:
    """linear_attention for one more token of each sequence; `state` is updated in place.

    Args:
        q, k:      [B, H, K], v: [B, H, V] of one dtype, contiguous channels.
        log_decay: [H] float32.
        state:     [slots, H, K, V] float32, contiguous: a cache of states.
        slots:     [B] int32 on the device, the row of `state` of each sequence; distinct, except that ids outside
                   the cache (-1) mark sequences that take no part: their outputs are zero.  None: row b.

    Returns:
        o [B, H, V] in q's dtype.  Serving only: no gradients; a backward that has saved `state` from before raises, as
        after torch's own in-place operations.
    """
    if _capi.binding is not None:
        o = _capi.binding.linear_attention_step(q, k, v, log_decay, state, scale, slots)
        if o is not None:
            return o
    assert q.is_cuda and q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "q, k, v must be [B, H, .] on the GPU"
    B, H, K = q.shape
    assert k.shape == q.shape and v.shape[:2] == q.shape[:2], "k must have q's shape, v must be [B, H, V]"
    assert q.dtype == k.dtype == v.dtype, "q, k and v must share one dtype"
    assert k.device == q.device and v.device == q.device, "q, k and v must be on one device"
    dtype = _capi.dtype_code(q.dtype)
    V = v.shape[-1]
    assert B > 0 and H > 0 and 0 < K <= MAX_DIM and 0 < V <= MAX_DIM, "head dims must be between 1 and 256"
    assert not _capi.differentiated((q, k, v, log_decay, state)), \
        "linear_attention_step has no gradient and no tangent: call it under torch.no_grad(), without dual tensors"
    _check_decay(log_decay, H, q.device)
    assert state.device == q.device and state.dtype == torch.float32 and state.is_contiguous(), \
        "state must be contiguous float32 on q's device"
    assert state.dim() == 4 and tuple(state.shape[1:]) == (H, K, V), "state must be [slots, H, K, V]"
    assert slots is not None or B <= state.shape[0], "more sequences than rows of state"
    slots = _index(slots, B, q.device, "slots")
    q, k, v = _rows(q), _rows(k), _rows(v)
    scale = K ** -0.5 if scale is None else float(scale)
    return _step(q, k, v, log_decay, state, slots, scale, dtype)


@_capi.on_first_device
def _step(q, k, v, log_decay, state, slots, scale, dtype):
    B, H, K = q.shape
    V = v.shape[-1]
    o = torch.empty(B, H, V, dtype=q.dtype, device=q.device)
    status = _capi.load().dc_linear_attention_step(
        _capi.ptr(q), _strides(q, 2), _capi.ptr(k), _strides(k, 2), _capi.ptr(v), _strides(v, 2),
        _capi.ptr(log_decay), _capi.ptr(state), _capi.ptr(slots), _capi.ptr(o), B, H, K, V, state.shape[0], scale,
        dtype, _capi.stream_of(q))
    _capi.check(status, "linear attention step")
    _capi.written(state)
    return o
