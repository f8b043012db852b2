"""C ABI of the gated delta rule and the residual norm without a GPU: size queries and refusals (no pointer is used)."""

import pytest
import torch

import helpers  # noqa: F401  (the package's path)
from dynconv import _capi

E_NULL, E_SHAPE, E_DTYPE, E_UNSUP, E_WS, E_ALIGN, E_DEV = -1, -2, -3, -4, -5, -6, -7
P = 0x10000  # a fake device pointer
NO_DEV = not torch.cuda.is_available()


@pytest.fixture(scope="module")
def lib():
    return _capi.load()


def st(*values):
    return _capi.int64_array(values)


def fwd(lib, B=1, Hk=1, H=2, T=8, K=16, V=16, q=P, g=P, o=P, s=st(1, 1, 1), gs=st(1, 1, 1), dt=0, gdt=2, flags=1, ws=P, nws=1 << 40):
    return lib.dc_delta_rule_fwd(q, s, P, s, P, s, g, gs, P, gs, None, None, o, s, None, ws, nws, B, Hk, H, T, K, V, 1.0, 1e-6, dt, gdt,
                                 flags, None)


def bwd(lib, B=1, Hk=1, H=2, T=8, K=16, V=16, dq=P, dg=P, s=st(1, 1, 1), gs=st(1, 1, 1), dt=0, gdt=2, flags=1, ws=P, nws=1 << 40,
        fws=None):
    return lib.dc_delta_rule_bwd(P, s, P, s, P, s, P, gs, P, gs, None, None, P, s, None, dq, s, P, s, P, s, dg, gs, P, gs, None, fws, ws,
                                 nws, B, Hk, H, T, K, V, 1.0, 1e-6, dt, gdt, flags, None)


@pytest.mark.parametrize("call", [fwd, bwd])
def test_delta_rule_refusals(lib, call):
    assert call(lib, dt=3) == E_DTYPE and call(lib, dt=0, gdt=1) == E_DTYPE and call(lib, dt=2, gdt=0) == E_DTYPE
    for bad in (dict(B=0), dict(H=0), dict(Hk=0), dict(Hk=3), dict(T=-1), dict(K=0), dict(V=-5), dict(B=1 << 31),
                dict(B=1 << 20, H=1 << 20), dict(Hk=4, H=2)):
        assert call(lib, **bad) == E_SHAPE, bad
    assert call(lib, K=257) == E_UNSUP and call(lib, V=257) == E_UNSUP and call(lib, flags=8) == E_UNSUP
    assert call(lib, s=None) == E_NULL and call(lib, gs=None) == E_NULL
    which = 1 if call is bwd else 0
    need = lib.dc_delta_rule_ws_bytes(1, 1, 2, 8, 16, 16, 0, 1, which)
    assert need > 0
    assert call(lib, nws=need - 1) == E_WS and call(lib, ws=None) == E_WS and call(lib, ws=P + 8) == E_WS
    if NO_DEV:
        assert call(lib) == E_DEV and call(lib, nws=need) == E_DEV


def test_delta_rule_sizes_past_any_memory(lib):
    """Workspaces are counted in 64 bits: sizes that would pass them are refused, the largest others give a count."""
    q = lambda B, H, T, dt, flags, which: lib.dc_delta_rule_ws_bytes(B, 1, H, T, 256, 256, dt, flags, which)  # noqa: E731
    for dt in (0, 1, 2):
        for which in (0, 1, 2):
            assert q(1 << 20, 1, (1 << 20) + 1, dt, 3, which) == E_SHAPE
            assert q(1 << 20, 1, 1 << 20, dt, 3, which) > 1 << 40
            assert q(1 << 10, 1 << 10, 1 << 20, dt, 0, which) > 1 << 40


def test_delta_rule_states_kept_for_a_backward(lib):
    """What the forward keeps the backward need not hold; it is kept where it is at most twice q, k, v and o."""
    q = lambda flags, which, T=640, H=4, K=128, V=128, dt=0: lib.dc_delta_rule_ws_bytes(2, 2, H, T, K, V, dt, flags, which)  # noqa: E731
    n = 10 * 8  # chunks of 64 tokens, of all heads
    kept = n * (64 * 128 + 128 * 128) * 2
    assert q(5, 0) == q(1, 0) + kept and q(5, 2) == q(1, 2) - kept and q(5, 1) == q(1, 1)
    for flags, sizes in ((3, {}), (1, dict(K=256, V=64, H=2)), (1, dict(K=256, V=256, dt=1)), (1, dict(K=256, V=256, dt=2))):
        if sizes.get("dt", 0) or flags == 3:  # 32 tokens to a chunk and two or three parts of everything
            assert q(flags | 4, 0, **sizes) == q(flags, 0, **sizes) and q(flags | 4, 2, **sizes) == q(flags, 2, **sizes)
        else:
            assert q(flags | 4, 0, **sizes) > q(flags, 0, **sizes)


def test_delta_rule_states_are_apart(lib):
    s, gs = st(1, 1, 1), st(1, 1, 1)
    call = lambda a, b: lib.dc_delta_rule_fwd(P, s, P, s, P, s, P, gs, P, gs, a, None, P, s, b, P, 1 << 40, 1, 1, 2, 8, 16, 16, 1.0,  # noqa: E731
                                              1e-6, 0, 2, 1, None)
    assert call(P, P) == E_UNSUP
    back = lambda a, b: lib.dc_delta_rule_bwd(P, s, P, s, P, s, P, gs, P, gs, None, None, P, s, a, P, s, P, s, P, s, P, gs, P, gs, b,  # noqa: E731
                                              None, P, 1 << 40, 1, 1, 2, 8, 16, 16, 1.0, 1e-6, 0, 2, 1, None)
    assert back(P, P) == E_UNSUP
    if NO_DEV:
        assert call(P, P + 16) == E_DEV and call(None, P) == E_DEV and back(P, P + 16) == E_DEV


def test_delta_rule_pointers(lib):
    assert fwd(lib, q=None) == E_NULL and fwd(lib, o=None) == E_NULL and fwd(lib, g=None) == E_NULL
    assert fwd(lib, q=P + 1) == E_ALIGN and fwd(lib, g=P + 2) == E_ALIGN and fwd(lib, g=P + 1, gdt=0) == E_ALIGN
    assert bwd(lib, dq=None) == E_NULL and bwd(lib, dq=P + 1) == E_ALIGN and bwd(lib, dg=P + 2) == E_ALIGN
    assert bwd(lib, fws=P + 8) == E_WS
    if NO_DEV:
        assert fwd(lib, T=0, q=None, o=None, g=None) == E_DEV


def test_delta_rule_workspaces(lib):
    """None without tokens; given the forward's, the backward needs less; sizes grow with the length; refusals."""
    size = lambda T, flags, which: lib.dc_delta_rule_ws_bytes(2, 2, 4, T, 64, 64, 0, flags, which)  # noqa: E731
    for flags in (0, 1, 2, 3):
        assert size(0, flags, 0) == size(0, flags, 1) == 0
        f, alone, given = (size(1000, flags, w) for w in (0, 1, 2))
        assert 0 < f < alone and 0 < given < alone
        assert bwd(lib, B=2, Hk=2, H=4, T=1000, K=64, V=64, flags=flags, fws=P, nws=given - 1) == E_WS
        assert bwd(lib, B=2, Hk=2, H=4, T=1000, K=64, V=64, flags=flags, nws=alone - 1) == E_WS
    assert lib.dc_delta_rule_ws_bytes(2, 3, 4, 10, 64, 64, 0, 0, 0) == E_SHAPE
    assert lib.dc_delta_rule_ws_bytes(2, 2, 4, 10, 64, 300, 0, 0, 0) == E_UNSUP


def test_delta_rule_step_refusals(lib):
    def step(B=2, Hk=1, H=2, K=16, V=16, slots=2, ids=None, q=P, g=P, state=P, dt=0, gdt=2, s=st(1, 1), gs=st(1, 1), flags=0):
        return lib.dc_delta_rule_step(q, s, P, s, P, s, g, gs, P, gs, state, ids, P, B, Hk, H, K, V, slots, 1.0, 1e-6, dt, gdt, flags, None)

    assert step(dt=9) == E_DTYPE and step(gdt=1) == E_DTYPE
    assert step(B=0) == E_SHAPE and step(slots=0) == E_SHAPE and step(B=3) == E_SHAPE and step(Hk=3) == E_SHAPE
    assert step(K=300) == E_UNSUP and step(flags=8) == E_UNSUP
    assert step(q=None) == E_NULL and step(state=None) == E_NULL and step(s=None) == E_NULL and step(g=None) == E_NULL
    assert step(gs=None) == E_NULL and step(state=P + 2) == E_ALIGN and step(ids=P + 2, B=3) == E_ALIGN
    if NO_DEV:
        assert step() == E_DEV and step(B=3, ids=P) == E_DEV


def test_residual_norm_refusals(lib):
    def f(M=4, D=64, act=0, dt=0, xdt=0, pdt=0, x=P, br=P, w=None, y=P, h=P):
        return lib.dc_residual_norm_fwd(x, br, w, None, None, None, y, h, M, D, 1.0, 1e-6, act, dt, xdt, pdt, None)

    def b(M=4, D=64, act=0, gate=None, dgate=None, dw=None, ds=None, ws=None, nws=0, dx=P, dh=P, dt=0, xdt=0):
        return lib.dc_residual_norm_bwd(P, P, None, None, gate, None, P, dh, dx, P, dgate, dw, None, ds, ws, nws, M, D, 1.0, 1e-6, act, dt,
                                        xdt, dt, None)

    assert f(dt=4) == E_DTYPE and f(xdt=1) == E_DTYPE and f(pdt=1) == E_DTYPE and f(dt=2, xdt=0) == E_DTYPE
    assert f(M=0) == E_SHAPE and f(D=0) == E_SHAPE and f(M=1 << 31) == E_SHAPE
    assert f(D=8193) == E_UNSUP and f(act=3) == E_UNSUP
    assert f(x=None) == E_NULL and f(br=None) == E_NULL and f(y=None) == E_NULL and f(h=None) == E_NULL
    assert f(x=P + 1) == E_ALIGN and f(x=P + 2, xdt=2) == E_ALIGN and f(w=P + 2, pdt=2) == E_ALIGN
    assert b(gate=P) == E_NULL and b(dx=None) == E_NULL and b(dh=P + 1) == E_ALIGN
    need = lib.dc_residual_norm_bwd_ws_bytes(4, 64, 0)
    assert need > 0
    for kw in (dict(dw=P), dict(ds=P)):
        assert b(**kw) == E_WS and b(**kw, ws=P, nws=need - 1) == E_WS and b(**kw, ws=P + 4, nws=need) == E_WS
    assert lib.dc_residual_norm_bwd_ws_bytes(4, 8193, 0) == E_UNSUP and lib.dc_residual_norm_bwd_ws_bytes(0, 64, 0) == E_SHAPE
    if NO_DEV:
        assert f() == E_DEV and b() == E_DEV and b(dw=P, ws=P, nws=need) == E_DEV and b(gate=P, dgate=P) == E_DEV
