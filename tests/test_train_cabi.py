"""What the training operators refuse, through the C ABI: checked before anything is launched, so no GPU is needed."""

import ctypes

import pytest

BAD_ARG, BAD_SHAPE = -1, -2
P = ctypes.c_void_p(4096)  # (never dereferenced)


@pytest.fixture
def L():
    from nkilib import _native as nv

    return nv.lib()


def test_token_slots_refusals(L):
    assert L.moe_token_slots(None, 4, 4, 2, P, None) == BAD_ARG
    assert L.moe_token_slots(P, 4, 4, 2, None, None) == BAD_ARG
    assert L.moe_token_slots(P, -1, 4, 2, P, None) == BAD_ARG
    for k in (0, 65):
        assert L.moe_token_slots(P, 4, 4, k, P, None) == BAD_SHAPE
    assert L.moe_token_slots(P, 2**31, 4, 2, P, None) == BAD_SHAPE
    assert L.moe_token_slots(P, 4, 2**31, 2, P, None) == BAD_SHAPE
    assert L.moe_token_slots(P, 4, 0, 2, P, None) == 0  # no tokens: nothing to write


def test_permute_refusals(L):
    call = lambda x=P, t=P, S=4, T=4, n=16, out=P: L.moe_permute_tokens(x, t, S, T, n, out, None)
    assert call(x=None) == BAD_ARG and call(t=None) == BAD_ARG and call(out=None) == BAD_ARG and call(n=-1) == BAD_ARG
    assert call(S=2**31) == BAD_SHAPE and call(T=2**31) == BAD_SHAPE and call(n=2**31) == BAD_SHAPE
    assert call(S=0) == 0 and call(n=0) == 0


def _combine(L, **kw):
    a = dict(y=P, dtype=0, aff=P, aff_dtype=0, T1=5, E=3, tp=P, b2e=P, B=4, N=2, slots=P, k=2, build=0, S=8, T=0, H=16, out=P)
    a.update(kw)
    return L.moe_combine_tokens(a["y"], a["dtype"], a["aff"], a["aff_dtype"], a["T1"], a["E"], a["tp"], a["b2e"], a["B"], a["N"],
                                a["slots"], a["k"], a["build"], a["S"], a["T"], a["H"], a["out"], None)


def test_combine_refusals(L):
    assert _combine(L) == 0 and _combine(L, build=1) == 0  # (no tokens)
    assert _combine(L, T=4, dtype=7) == BAD_ARG and _combine(L, T=4, dtype=3) == BAD_ARG
    assert _combine(L, aff=None) == BAD_ARG and _combine(L, b2e=None) == BAD_ARG
    assert _combine(L, slots=None) == BAD_ARG and _combine(L, y=None) == BAD_ARG and _combine(L, out=None) == BAD_ARG
    assert _combine(L, tp=None, build=1) == BAD_ARG and _combine(L, tp=None) == 0
    assert _combine(L, aff_dtype=1) == BAD_ARG  # fp16 affinities
    assert _combine(L, T=6) == BAD_SHAPE  # fewer rows of affinities than tokens
    assert _combine(L, E=0) == BAD_SHAPE
    assert _combine(L, k=0) == BAD_SHAPE and _combine(L, k=65) == BAD_SHAPE
    assert _combine(L, B=0) == BAD_SHAPE and _combine(L, S=9) == BAD_SHAPE and _combine(L, S=2**31, B=2**30) == BAD_SHAPE
    assert _combine(L, B=2**33, N=2**33) == BAD_SHAPE and _combine(L, T=-1) == BAD_ARG


def test_combine_bwd_refusals(L):
    def call(**kw):
        a = dict(d=P, y=P, dtype=0, aff=P, aff_dtype=0, T1=5, E=3, tp=P, b2e=P, B=4, N=2, slots=P, k=2, build=1, T=4, H=16, dy=P, da=P)
        a.update(kw)
        return L.moe_combine_tokens_bwd(a["d"], a["y"], a["dtype"], a["aff"], a["aff_dtype"], a["T1"], a["E"], a["tp"], a["b2e"],
                                        a["B"], a["N"], a["slots"], a["k"], a["build"], a["T"], a["H"], a["dy"], a["da"], None)

    for name in ("d", "y", "aff", "tp", "b2e", "slots", "dy", "da"):
        assert call(**{name: None}) == BAD_ARG, name
    assert call(dtype=6) == BAD_ARG and call(aff_dtype=1) == BAD_ARG and call(H=-1) == BAD_ARG
    assert call(T=6) == BAD_SHAPE and call(k=65) == BAD_SHAPE and call(B=0) == BAD_SHAPE and call(B=2**30, N=2) == BAD_SHAPE


def test_glu_refusals(L):
    f = (ctypes.c_float * 4)()

    def fwd(x=P, dtype=0, R=4, I=64, act=0, mask=0, clamps=None, n=0, h=P, c=P, s=P):
        return L.moe_glu_checkpoint(x, dtype, R, I, act, mask, clamps, None, n, h, c, s, None)

    def bwd(c=P, s=P, d=P, dtype=0, R=4, I=64, act=0, mask=0, clamps=None, dgu=P):
        return L.moe_glu_checkpoint_bwd(c, s, d, dtype, R, I, act, mask, clamps, None, 0, dgu, None, None)

    assert fwd(R=0) == 0 and bwd(R=0) == 0
    assert fwd(x=None) == BAD_ARG and fwd(h=None) == BAD_ARG and fwd(c=None) == BAD_ARG and fwd(s=None) == BAD_ARG
    assert bwd(c=None) == BAD_ARG and bwd(d=None) == BAD_ARG and bwd(dgu=None) == BAD_ARG
    for call in (fwd, bwd):
        assert call(dtype=3) == BAD_ARG and call(act=4) == BAD_ARG and call(act=-1) == BAD_ARG
        assert call(I=0) == BAD_ARG and call(R=-1) == BAD_ARG
        assert call(mask=16, clamps=f) == BAD_ARG and call(mask=1) == BAD_ARG
        assert call(I=2**17 + 1) == BAD_SHAPE and call(R=2**31) == BAD_SHAPE
    pack = lambda x=P, N=2, I=64, B=4: L.moe_pack_gate_up_checkpoint(x, N, I, B, None, 0, P, P, None)
    assert pack(N=0) == 0
    assert pack(x=None) == BAD_ARG and pack(B=0) == BAD_ARG and pack(I=0) == BAD_ARG
    assert pack(I=2**17 + 1) == BAD_SHAPE and pack(N=2**29) == BAD_SHAPE
    assert L.moe_dequantize_checkpoint(P, P, 2, 64, P, 3, None) == BAD_ARG
    assert L.moe_dequantize_checkpoint(P, None, 2, 64, P, 0, None) == BAD_ARG
    assert L.moe_dequantize_checkpoint(P, P, 0, 64, P, 0, None) == 0


def test_glu_with_kept_bits_refusals(L):
    f = (ctypes.c_float * 4)()
    fwd = lambda R=4, mask=0, clamps=None: L.moe_glu_checkpoint_clamped(P, 0, R, 64, 0, mask, clamps, None, 0, P, P, P, P, None)
    bwd = lambda R=4, mask=0, clamps=None: L.moe_glu_checkpoint_bwd_clamped(P, P, P, P, 0, R, 64, 0, mask, clamps, None, 0, P, None, None)
    pack = lambda R=4, mask=0, clamps=None: L.moe_pack_gate_up_checkpoint_clamped(P, R, 64, 4, mask, clamps, None, 0, P, P, P, None)
    for call in (fwd, bwd, pack):
        assert call(R=0) == 0 and call(R=0, mask=15, clamps=f) == 0
        assert call(mask=16, clamps=f) == BAD_ARG and call(mask=1) == BAD_ARG and call(R=-1) == BAD_ARG
    assert L.moe_glu_checkpoint_bwd_clamped(None, P, P, P, 0, 4, 64, 0, 0, None, None, 0, P, None, None) == BAD_ARG


def test_rows_of_a_record_as_its_values(L):
    """A record of R < 2^31 rows is one of 2 R rows of codes."""
    assert L.moe_dequantize_checkpoint(P, P, 2**32, 64, P, 0, None) == BAD_SHAPE
    assert L.moe_glu_checkpoint(P, 0, 2**31, 1, 0, 0, None, None, 0, P, P, P, None) == BAD_SHAPE


def test_blocks_whose_product_is_past_64_bits_are_refused(L):
    pack = lambda N, B: L.moe_pack_gate_up_checkpoint(P, N, 1, B, None, 0, P, P, None)
    for N, B in ((2**62, 4), (4, 2**62), (2**33, 2**31), (2**31, 1), (1, 2**31)):
        assert pack(N, B) == BAD_SHAPE, (N, B)


def test_host_tensors_are_refused():
    """There is no CPU path: the operators say so."""
    import torch
    from nkilib._native import NativeLibraryError
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd, pack_gate_up_checkpoint
    from nkilib.core.moe.token_permute import build_token_slots, combine_tokens, permute_tokens

    x, t = torch.zeros(4, 8), torch.zeros(8, dtype=torch.int32)
    u8 = torch.zeros(4, 2, 8, dtype=torch.uint8)
    for call in (lambda: permute_tokens(x, t), lambda: build_token_slots(t, 4, 2), lambda: combine_tokens(x, x, t, t, 1, 4, 2),
                 lambda: glu_checkpoint(x.view(2, 2, 8)), lambda: glu_checkpoint_bwd(u8, u8, x),
                 lambda: pack_gate_up_checkpoint(x.view(1, 2, 2, 8).bfloat16())):
        with pytest.raises(NativeLibraryError, match="no CPU path"):
            call()


def test_router_bwd_refusals(L):
    ws = L.moe_router_topk_bwd_workspace_bytes
    need = ws(64, 256, 8)
    assert need > 0 and ws(0, 256, 8) == 0 and ws(64, 200, 8) == 0 and ws(64, 256, 513) == 0 and ws(2**26 + 1, 128, 8) == 0

    def call(**kw):
        a = dict(g=P, gd=2, x=P, w=P, l=P, ld=2, ids=P, T=64, H=256, E=8, k=2, act=1, pre=1, norm=0, mask=1, dx=P, dw=P, db=None, bd=2,
                 ws=P, n=need)
        a.update(kw)
        return L.moe_router_topk_bwd(a["g"], a["gd"], a["x"], a["w"], a["l"], a["ld"], a["ids"], a["T"], a["H"], a["E"], a["k"],
                                     a["act"], a["pre"], a["norm"], a["mask"], a["dx"], a["dw"], a["db"], a["bd"], a["ws"], a["n"], None)

    for name in ("g", "x", "w", "l", "ids", "dx", "dw"):
        assert call(**{name: None}) == BAD_ARG, name
    assert call(gd=1) == BAD_ARG and call(ld=3) == BAD_ARG and call(act=2) == BAD_ARG and call(db=P, bd=1) == BAD_ARG
    assert call(T=0) == BAD_ARG and call(H=192) == BAD_SHAPE and call(E=513) == BAD_SHAPE and call(k=0) == BAD_SHAPE
    assert call(k=9) == BAD_SHAPE and call(E=4, k=5) == BAD_SHAPE
    assert call(ws=None) == -3 and call(n=need - 1) == -3 and call(ws=ctypes.c_void_p(4100)) == BAD_ARG
