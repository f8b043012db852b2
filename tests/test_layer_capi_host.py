"""C ABI of include/dynconv_layer.h without a GPU: exports, signatures, size queries, refusals (no pointer is used)."""

import ctypes
import os
import re

import pytest
import torch

from helpers import ROOT
from dynconv import _capi

HEADER = os.path.join(ROOT, "include", "dynconv_layer.h")
E_NULL, E_SHAPE, E_DTYPE, E_UNSUP, E_WS, E_ALIGN, E_DEV = -1, -2, -3, -4, -5, -6, -7
P = 0x10000  # a fake device pointer
NO_DEV = not torch.cuda.is_available()


@pytest.fixture(scope="module")
def lib():
    return _capi.load()


def st(*values):
    return _capi.int64_array(values)


def test_exports_every_declared_symbol(lib):
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(dc_\w+)\s*\(", txt))
    assert names == set(_capi.LAYER_SIGNATURES), "ctypes signatures out of sync with the header"
    raw = ctypes.CDLL(_capi.LIB_PATH)
    assert all(hasattr(raw, n) for n in names)


def la_fwd(lib, B=1, H=2, T=8, K=16, V=16, q=P, o=P, lam=P, s=st(1, 1, 1), dt=0, ws=P, nws=1 << 40):
    return lib.dc_linear_attention_fwd(q, s, P, s, P, s, lam, None, None, o, s, None, ws, nws, B, H, T, K, V, 1.0, dt, None)


def la_bwd(lib, B=1, H=2, T=8, K=16, V=16, dq=P, s=st(1, 1, 1), dt=0, ws=P, nws=1 << 40, states=None):
    return lib.dc_linear_attention_bwd(P, s, P, s, P, s, P, None, None, P, s, None, dq, s, P, s, P, s, None, states, ws, nws,
                                       B, H, T, K, V, 1.0, dt, None)


@pytest.mark.parametrize("call", [la_fwd, la_bwd])
def test_linear_attention_refusals(lib, call):
    assert call(lib, dt=3) == E_DTYPE
    for bad in (dict(B=0), dict(H=0), dict(T=-1), dict(K=0), dict(V=-5), dict(B=1 << 31), dict(B=1 << 20, H=1 << 20)):
        assert call(lib, **bad) == E_SHAPE, bad
    assert call(lib, K=257) == E_UNSUP and call(lib, V=257) == E_UNSUP
    assert call(lib, s=None) == E_NULL
    need = lib.dc_linear_attention_ws_bytes(1, 2, 1 << 16, 16, 16, 0, int(call is la_bwd))
    assert need >= 0
    if need > 0:
        assert call(lib, T=1 << 16, nws=need - 1) == E_WS and call(lib, T=1 << 16, ws=None) == E_WS
    if NO_DEV:
        assert call(lib) == E_DEV


def test_linear_attention_forward_pointers(lib):
    assert la_fwd(lib, q=None) == E_NULL and la_fwd(lib, o=None) == E_NULL and la_fwd(lib, lam=None) == E_NULL
    assert la_fwd(lib, q=P + 1) == E_ALIGN and la_fwd(lib, q=P + 2, dt=2) == E_ALIGN
    assert la_fwd(lib, lam=P + 2) == E_ALIGN
    assert la_bwd(lib, states=P + 8) == E_WS
    assert la_bwd(lib, dq=None) == E_NULL and la_bwd(lib, dq=P + 1) == E_ALIGN
    if NO_DEV:  # no rows: the activations' pointers do not matter
        assert la_fwd(lib, T=0, q=None, o=None) == E_DEV


def test_linear_attention_step_refusals(lib):
    def step(B=2, H=2, K=16, V=16, slots=2, ids=None, q=P, state=P, dt=0, s=st(1, 1)):
        return lib.dc_linear_attention_step(q, s, P, s, P, s, P, state, ids, P, B, H, K, V, slots, 1.0, dt, None)

    assert step(dt=9) == E_DTYPE
    assert step(B=0) == E_SHAPE and step(slots=0) == E_SHAPE and step(B=3) == E_SHAPE
    assert step(K=300) == E_UNSUP
    assert step(q=None) == E_NULL and step(state=None) == E_NULL and step(s=None) == E_NULL
    assert step(state=P + 2) == E_ALIGN and step(ids=P + 2, B=3) == E_ALIGN
    if NO_DEV:
        assert step() == E_DEV and step(B=3, ids=P) == E_DEV


def test_group_norm_refusals(lib):
    def fwd(M=4, D=64, groups=4, act=1, dt=0, pdt=0, x=P, w=None, y=P):
        return lib.dc_group_norm_fwd(x, w, None, None, y, M, D, groups, 1e-5, act, dt, pdt, None)

    def bwd(M=4, D=64, groups=4, gate=None, dgate=None, dw=None, ws=None, nws=0, dx=P):
        return lib.dc_group_norm_bwd(P, P, P, gate, P, dx, dgate, dw, None, ws, nws, M, D, groups, 1e-5, 1, 0, 0, None)

    assert fwd(dt=4) == E_DTYPE and fwd(pdt=-1) == E_DTYPE
    assert fwd(M=0) == E_SHAPE and fwd(D=0) == E_SHAPE and fwd(groups=3) == E_SHAPE and fwd(groups=0) == E_SHAPE
    assert fwd(act=2) == E_UNSUP and fwd(D=4097, groups=1) == E_UNSUP
    assert fwd(x=None) == E_NULL and fwd(y=None) == E_NULL
    assert fwd(x=P + 1) == E_ALIGN and fwd(w=P + 2, pdt=2) == E_ALIGN
    assert bwd(gate=P) == E_NULL and bwd(dx=None) == E_NULL
    need = lib.dc_group_norm_bwd_ws_bytes(4, 64, 4, 0)
    assert need > 0
    assert bwd(dw=P) == E_WS and bwd(dw=P, ws=P, nws=need - 1) == E_WS and bwd(dw=P, ws=P + 4, nws=need) == E_WS
    assert lib.dc_group_norm_bwd_ws_bytes(4, 64, 3, 0) == E_SHAPE
    if NO_DEV:
        assert fwd() == E_DEV and bwd() == E_DEV and bwd(dw=P, ws=P, nws=need) == E_DEV


def test_lowrank_step_refusals(lib):
    def step(G=2, N=3, D=64, R=15, W=4, slots=3, ids=None, x=P, x_ld=128, sw=True, state=P, dt=0, z=P, y=P):
        arr = lambda p: (ctypes.c_void_p * 4)(*[p] * 4)  # noqa: E731
        return lib.dc_lowrank_step_grouped(G, x, x_ld, arr(z), arr(P), arr(P) if sw else None, state, ids, arr(y), N, D, R,
                                           W, slots, dt, 1, None)

    assert step(dt=5) == E_DTYPE
    for bad in (dict(G=0), dict(G=5), dict(N=0), dict(D=0), dict(R=0), dict(W=0), dict(slots=0), dict(N=4),
                dict(x_ld=127), dict(D=1 << 30)):
        assert step(**bad) == E_SHAPE, bad
    assert step(W=1025) == E_UNSUP and step(R=256) == E_UNSUP
    assert step(x=None) == E_NULL and step(z=None) == E_NULL and step(y=None) == E_NULL and step(state=None) == E_NULL
    assert step(x=P + 1) == E_ALIGN and step(z=P + 2, dt=2) == E_ALIGN and step(ids=P + 1, N=4) == E_ALIGN
    if NO_DEV:
        assert step() == E_DEV and step(W=1, state=None) == E_DEV and step(N=4, ids=P) == E_DEV


def test_linear_attention_backward_workspace_with_the_forwards(lib):
    """Given the forward's workspace, the backward needs room for one set of states instead of two."""
    size = (1, 2, 1 << 16, 16, 16, 0)
    fwd, alone, given = (lib.dc_linear_attention_ws_bytes(*size, which) for which in (0, 1, 2))
    assert fwd > 0 and given == fwd and alone == 2 * fwd
    assert la_bwd(lib, T=1 << 16, states=P, nws=given - 1) == E_WS
    assert la_bwd(lib, T=1 << 16, nws=given) == E_WS and la_bwd(lib, T=1 << 16, nws=alone - 1) == E_WS
    assert lib.dc_linear_attention_ws_bytes(1, 2, 8, 16, 16, 0, 2) == 0
    if NO_DEV:
        assert la_bwd(lib, T=1 << 16, states=P, nws=given) == E_DEV and la_bwd(lib, T=1 << 16, nws=alone) == E_DEV
