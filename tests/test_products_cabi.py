"""What the products by expert and in 8-bit integers refuse, through the C ABI: checked before anything is launched, so no GPU is
needed."""

import ctypes

import pytest

BAD_ARG, BAD_SHAPE, UNSUPPORTED = -1, -2, -5
P = ctypes.c_void_p(4096)  # (never dereferenced)


@pytest.fixture
def L():
    from nkilib import _native as nv

    return nv.lib()


def test_row_offsets_refusals(L):
    call = lambda b=P, N=4, B=2, E=3, o=P: L.moe_expert_row_offsets(b, N, B, E, o, None)
    assert call(b=None) == BAD_ARG and call(o=None) == BAD_ARG and call(N=-1) == BAD_ARG
    assert call(B=0) == BAD_SHAPE and call(E=0) == BAD_SHAPE and call(E=1025) == BAD_SHAPE and call(N=2**31) == BAD_SHAPE
    assert call(N=2**16, B=2**15) == BAD_SHAPE and call(N=2, B=2**31) == BAD_SHAPE


def test_grouped_refusals(L):
    def fwd(x=P, w=P, dt=0, o=P, S=0, K=64, N=64, E=2, out=P):
        return L.moe_grouped_matmul(x, w, dt, o, S, K, N, E, out, None)

    def bwd(d=P, x=P, w=P, dt=0, o=P, S=0, K=64, N=64, E=2, dx=P, dw=None, wdt=0):
        return L.moe_grouped_matmul_bwd(d, x, w, dt, o, S, K, N, E, dx, dw, wdt, None)

    assert fwd() == 0 and bwd() == 0  # (no rows)
    for name in ("x", "w", "o", "out"):
        assert fwd(**{name: None}) == BAD_ARG, name
    assert bwd(d=None) == BAD_ARG and bwd(w=None) == BAD_ARG and bwd(o=None) == BAD_ARG and bwd(dx=None) == BAD_ARG
    assert bwd(dw=P, x=None) == BAD_ARG and bwd(dw=P, wdt=1) == BAD_ARG and bwd(dw=P, wdt=3) == BAD_ARG
    for call in (fwd, bwd):
        assert call(dt=2) == BAD_ARG and call(dt=3) == BAD_ARG and call(dt=-1) == BAD_ARG and call(S=-1) == BAD_ARG
        for size in (dict(K=0), dict(N=0), dict(E=0), dict(E=1025), dict(K=2**20 + 1), dict(N=2**20 + 1), dict(S=2**31), dict(S=2**31 - 1024),
                     dict(K=2**62)):
            assert call(**size) == BAD_SHAPE, size


def test_int8_refusals(L):
    def call(x=P, xs=P, w=P, ws=P, bias=None, o=P, S=0, K=64, N=64, E=2, out=P, dt=0):
        return L.moe_int8_matmul(x, xs, w, ws, bias, o, S, K, N, E, out, dt, None)

    assert call() == 0 and call(o=None, E=1, bias=P) == 0
    for name in ("x", "xs", "w", "ws", "out"):
        assert call(**{name: None}) == BAD_ARG, name
    assert call(o=None) == BAD_ARG and call(dt=3) == BAD_ARG and call(dt=-1) == BAD_ARG and call(S=-1) == BAD_ARG
    assert call(bias=P) == UNSUPPORTED
    for size in (dict(K=0), dict(N=0), dict(E=1025), dict(K=2**17), dict(N=2**20 + 1), dict(S=2**31)):
        assert call(**size) == BAD_SHAPE, size


def test_host_tensors_are_refused():
    import torch
    from nkilib._native import NativeLibraryError
    from nkilib.core.int8_matmul import grouped_int8_matmul, int8_matmul
    from nkilib.core.moe.grouped_matmul import expert_row_offsets, grouped_matmul, grouped_matmul_bwd

    x, w, o = torch.zeros(4, 8).bfloat16(), torch.zeros(2, 8, 8).bfloat16(), torch.zeros(3, dtype=torch.int32)
    q, f = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: grouped_matmul(x, w, o), lambda: grouped_matmul_bwd(x, x, w, o), lambda: expert_row_offsets(o, 1, 2),
                 lambda: int8_matmul(q, f, q, f), lambda: grouped_int8_matmul(q, f, w.to(torch.int8), f, o)):
        with pytest.raises(NativeLibraryError, match="no CPU path"):
            call()


def test_norm_refusals(L):
    def fwd(x=P, dt=0, r=None, g=P, gd=0, norm=1, eps=1e-6, rows=0, H=64, cd=7, c=P, s=P, o=None):
        return L.moe_rmsnorm_quant_rows(x, dt, r, g, gd, norm, eps, rows, H, cd, c, s, o, None)

    assert fwd() == 0 and fwd(cd=3, r=P, o=P, g=None) == 0
    for name in ("x", "c", "s"):
        assert fwd(**{name: None}) == BAD_ARG, name
    assert fwd(dt=3) == BAD_ARG and fwd(gd=7) == BAD_ARG and fwd(cd=4) == BAD_ARG and fwd(rows=-1) == BAD_ARG
    assert fwd(r=P) == BAD_ARG and fwd(o=P) == BAD_ARG and fwd(eps=-1.0) == BAD_ARG and fwd(eps=float("nan")) == BAD_ARG
    assert fwd(H=0) == BAD_SHAPE and fwd(H=16385) == BAD_SHAPE and fwd(rows=2**31) == BAD_SHAPE

    need = L.moe_rmsnorm_quant_rows_bwd_workspace_bytes
    assert need(1, 64) == 256 and need(5000, 100) == 512 * 400 and need(0, 64) == 0 and need(4, 16385) == 0 and need(4, 0) == 0

    def bwd(d=P, x=P, dt=0, g=P, gd=0, r=None, eps=1e-6, rows=4, H=64, dx=P, dg=P, ws=P, n=4 * 256):
        return L.moe_rmsnorm_quant_rows_bwd(d, x, dt, g, gd, r, eps, rows, H, dx, dg, ws, n, None)

    for name in ("d", "x", "dx", "g"):
        assert bwd(**{name: None}) == BAD_ARG, name
    assert bwd(dt=7) == BAD_ARG and bwd(gd=3) == BAD_ARG and bwd(eps=-1.0) == BAD_ARG and bwd(rows=-1) == BAD_ARG
    assert bwd(rows=0) == BAD_SHAPE and bwd(H=0) == BAD_SHAPE and bwd(H=16385) == BAD_SHAPE
    assert bwd(ws=None) == -3 and bwd(n=1023) == -3 and bwd(ws=ctypes.c_void_p(4098)) == BAD_ARG

    def deq(c=P, cd=7, s=P, rows=0, H=64, o=P, dt=0):
        return L.moe_dequantize_rows(c, cd, s, rows, H, o, dt, None)

    assert deq() == 0 and deq(cd=3) == 0
    for name in ("c", "s", "o"):
        assert deq(**{name: None}) == BAD_ARG, name
    assert deq(cd=4) == BAD_ARG and deq(dt=3) == BAD_ARG and deq(rows=-1) == BAD_ARG
    assert deq(H=0) == BAD_SHAPE and deq(H=2**24) == BAD_SHAPE and deq(rows=2**31) == BAD_SHAPE
