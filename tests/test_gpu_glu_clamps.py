"""Which values of a record pass a gradient where the activation clamps, against masks taken from the values ahead of the record.

A clamped value passes none, whatever limit it met.  Of the others those do that lie further inside than the record's rounding at
the limit (half a step of e4m3: 2^-4 of the limit, or 2^-10 of the group's scale where that is more), twice of which is left out
here: 1/8 of the limit and 2^-9 of the largest value of the group (whose scale is at least 1/448 and at most 1/224 of it).
"""

import numpy as np
import pytest

from oracle import train as ot
from train_helpers import tensor, values

pytestmark = pytest.mark.gpu

NAMES = ("gate_clamp_upper_limit", "gate_clamp_lower_limit", "up_clamp_upper_limit", "up_clamp_lower_limit")
# limits that e4m3 holds, that it rounds inwards and outwards, one beside the border between two of its values, one that its
# bf16 puts on the other side of that border
LIMITS = [(7.0, None, 7.0, -7.0), (7.2, None, 0.9, -0.7), (10.5, -6.2, 20.6, -20.6), (1.1, -1.1, 0.9, -0.9), (6.2, -0.7, 7.2, -7.2),
          (0.8, -0.7, 1.06255, -1.06245), (7.2503, None, 3.6252, -3.6249), (None, 0.3, None, -0.01)]


def _kwargs(clamps):
    return {n: c for n, c in zip(NAMES, clamps) if c is not None}


def _sides(x, hi, lo):
    """(clamped, safely inside) of values [R, I] in 64 bits."""
    hi, lo = np.inf if hi is None else float(np.float32(hi)), -np.inf if lo is None else float(np.float32(lo))
    at = np.clip(x, lo, hi)
    pad = np.pad(np.abs(at), ((0, 0), (0, -x.shape[1] % 32))).reshape(len(x), -1, 32).max(-1)
    far = np.repeat(pad, 32, axis=1)[:, : x.shape[1]] * 2.0**-9
    with np.errstate(invalid="ignore"):
        inside = (x < hi - (0 if np.isinf(hi) else abs(hi) / 8) - far) & (x > lo + (0 if np.isinf(lo) else abs(lo) / 8) + far)
    return (x >= hi) | (x <= lo), inside


@pytest.mark.parametrize("clamps", LIMITS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_clamped_values_pass_nothing(clamps, dtype):
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd

    rng = np.random.default_rng(LIMITS.index(clamps))
    R, I = 60, 200
    x = rng.standard_normal((R, 2, I)) * np.exp2(rng.integers(-2, 5, (R, 2, 1)))
    for half in (0, 1):  # values around the limits, exactly at them, far beyond
        for limit in clamps[2 * half : 2 * half + 2]:
            if limit is not None:
                x[: R // 2, half, ::5] = limit * (1 + rng.uniform(-0.1, 0.1, (R // 2, len(range(0, I, 5)))))
                x[: R // 2, half, 1::50] = limit
                x[: R // 4, half, 2::50] = limit * 100
    t = tensor(x, dtype)
    v = values(t)
    _, codes, scales = glu_checkpoint(t, **_kwargs(clamps))
    d_gu, _ = glu_checkpoint_bwd(codes, scales, torch.ones((R, I), device="cuda"), **_kwargs(clamps))
    got = values(d_gu)
    for half in (0, 1):
        out, inside = _sides(v[:, half], *clamps[2 * half : 2 * half + 2])
        assert out.any() and inside.any()
        assert not got[:, half][out].any(), f"{np.count_nonzero(got[:, half][out])} of {out.sum()} clamped values pass a gradient"
    # d gate = up act'(gate), d up = act(gate): not zero for what is inside, unless the other factor is
    c, s = codes.cpu().numpy(), scales.cpu().numpy()
    rec = ot.record_values(c, s)
    g, u = ot.clamp_glu(rec[:, 0], rec[:, 1], [None if l is None else float(np.float32(l)) for l in clamps])
    act, slope = ot.act(g, "silu")
    for half, factor in ((0, u * slope), (1, act)):
        _, inside = _sides(v[:, half], *clamps[2 * half : 2 * half + 2])
        inside &= np.abs(factor) > 2.0**-100
        assert got[:, half][inside].all(), f"{np.count_nonzero(got[:, half][inside] == 0)} of {inside.sum()} values inside pass nothing"


@pytest.mark.parametrize("clamps", LIMITS)
def test_gradient_of_records_with_any_limit(clamps):
    """Value by value as the oracle has it."""
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint_bwd

    rng = np.random.default_rng(40)
    R, I = 33, 100
    codes, scales = ot.record((rng.standard_normal((R, 2, I)) * np.exp2(rng.integers(-3, 8, (R, 2, 1)))).astype(np.float32))
    v = ot.record_values(codes, scales)
    d = rng.standard_normal((R, I)).astype(np.float32)
    d_gu, h = glu_checkpoint_bwd(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), tensor(d), **_kwargs(clamps))
    f32 = [None if l is None else float(np.float32(l)) for l in clamps]
    dg, du, want_h = ot.glu_bwd(v[:, 0], v[:, 1], d, "silu", f32, scales)
    got = values(d_gu)
    # (s(x) = act(x) / x is held in fp32, where what lies below 2^-126 may be zero: what it multiplies counts 2^-126 times, and whether
    # a value is zero is asked where s and the slope are above 2^-100.  Otherwise 32 steps of 2^-24 of the slope's two parts, which
    # add up to less than 2 (s to 1 at most, |x s'| to 0.3): an exponential with its argument's rounding made good, a reciprocal, four products.)
    g, u = ot.clamp_glu(v[:, 0], v[:, 1], f32)
    act, slope = ot.act(g, "silu")
    small = 2.0**-126 * (1 + np.abs(g))
    assert not ((got[:, 0] == 0) != (dg == 0))[np.abs(slope) > 2.0**-100].any()
    assert not ((got[:, 1] == 0) != (du == 0))[np.abs(act) > 2.0**-100].any()
    assert (np.abs(got[:, 0] - dg) <= 2.0**-18 * np.abs(d * u) + small * np.abs(d * u) + 2.0**-126).all()
    assert (np.abs(got[:, 1] - du) <= 2.0**-18 * np.abs(du) + small * np.abs(d) + 2.0**-126).all()
    assert (np.abs(values(h) - want_h) <= 2.0**-18 * np.abs(want_h) + small * np.abs(u) + 2.0**-126).all()


@pytest.mark.parametrize("clamps", [c for c in LIMITS if c[3] is not None])
def test_records_of_a_layers_checkpoint(clamps):
    """The layer clamps in fp32 and keeps bf16: what the limit is rounded to there is clamped too."""
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint_bwd, pack_gate_up_checkpoint

    rng = np.random.default_rng(50 + LIMITS.index(clamps))
    N, I, B = 2, 96, 40
    x = rng.standard_normal((N * B, 2, I)).astype(np.float32) * 8
    g, u = ot.clamp_glu(x[:, 0], x[:, 1], [None if l is None else np.float32(l) for l in clamps])
    kept = tensor(np.stack((g, u), 1).reshape(N, B, 2, I).transpose(0, 2, 3, 1), "bfloat16")
    codes, scales = pack_gate_up_checkpoint(kept)
    d_gu, _ = glu_checkpoint_bwd(codes, scales, torch.ones((N * B, I), device="cuda"), **_kwargs(clamps))
    got = values(d_gu)
    for half in (0, 1):
        out, _ = _sides(x[:, half].astype(np.float64), *clamps[2 * half : 2 * half + 2])
        assert out.any() or clamps[2 * half : 2 * half + 2] == (None, None)
        assert not got[:, half][out].any(), f"{np.count_nonzero(got[:, half][out])} of {out.sum()} clamped values pass a gradient"


def test_a_clamped_layer_and_its_gradient():
    """``moe_cte`` with the clamps of the layer's own tests, its checkpoint packed: no gradient where the product in 64 bits lies at or
    beyond a limit (further than the layer's own rounding), one where it lies well inside."""
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint_bwd, pack_gate_up_checkpoint
    from nkilib.core.moe.moe_cte import MoECTEImplementation, MoECTESpec, ShardOnIConfig, build_token_blocks, moe_cte
    from nkilib.core.router_topk import route_for_moe
    from nkilib.core.utils.common_types import RouterActFnType

    g = torch.Generator(device="cuda").manual_seed(3)
    T, H, I, E, k, B = 120, 256, 128, 4, 2, 128
    r = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).bfloat16()
    x = torch.cat((r(T, H), torch.zeros((1, H), device="cuda").bfloat16()))
    wgu, wd = r(E, H, 2, I, std=H**-0.5), r(E, I, H, std=I**-0.5)
    ids, aff = route_for_moe(x, r(H, E, std=H**-0.5), None, k, RouterActFnType.SOFTMAX, True)
    tp, be, _ = build_token_blocks(ids, E, B, E)
    clamps = (0.8, -0.7, 0.9, -0.7)
    spec = MoECTESpec(MoECTEImplementation.shard_on_i_dropping, shard_on_I=ShardOnIConfig(checkpoint_activation=True))
    _, gate_up_T, _ = moe_cte(x, aff.reshape(-1, 1), wgu, wd, tp, be, B, spec, **_kwargs(clamps))
    codes, scales, clamped = pack_gate_up_checkpoint(gate_up_T, tp, T, **_kwargs(clamps), return_clamped=True)
    opts = dict(token_position_to_id=tp, n_tokens=T, **_kwargs(clamps))
    ones = torch.ones((be.numel() * B, I), device="cuda")
    got, tpn = values(glu_checkpoint_bwd(codes, scales, ones, **opts)[0]), tp.cpu().numpy()
    told, bits = values(glu_checkpoint_bwd(codes, scales, ones, **opts, clamped=clamped)[0]), _bits(clamped, I)
    xv, wv, seen = values(x), values(wgu), 0
    for e in range(E):
        rows = np.flatnonzero((tpn >= 0) & (tpn < T) & (np.repeat(be.cpu().numpy(), B) == e))
        pre = (xv[tpn[rows]] @ wv[e].reshape(H, 2 * I)).reshape(-1, 2, I)
        off = (np.abs(xv[tpn[rows]]) @ np.abs(wv[e].reshape(H, 2 * I))).reshape(-1, 2, I) * (H + 2) * 2.0**-24
        for half in (0, 1):
            hi, lo = clamps[2 * half : 2 * half + 2]
            p, o = pre[:, half], off[:, half]
            out = (p >= hi + o) | (p <= lo - o)
            # (half a step of bf16, half a step of e4m3 at the limit)
            inside = (p < hi * (1 - 2.0**-3) - o) & (p > lo * (1 - 2.0**-3) + o) & (np.abs(p) > 0.02)
            assert not got[rows, half][out].any()
            both = inside & (np.abs(pre[:, 1 - half]) > 0.02)
            assert got[rows, half][both].all()
            # with the bits: all that lies further inside than half a step of bf16 (2^-8, twice that here)
            near = (p < hi * (1 - 2.0**-7) - o) & (p > lo * (1 - 2.0**-7) + o)
            assert bits[rows, half][out].all() and not bits[rows, half][near].any() and not told[rows, half][out].any()
            assert told[rows, half][near & (np.abs(p) > 0.02) & (np.abs(pre[:, 1 - half]) > 0.02)].all()
            seen += out.sum()
    assert seen > 1000


def _bits(clamped, I):
    return np.unpackbits(clamped.cpu().numpy(), axis=-1, bitorder="little")[..., :I].astype(bool)


def _near_limits(rng, R, I, clamps):
    """Rows [R, 2, I] with values around, at and far beyond their limits."""
    x = rng.standard_normal((R, 2, I)) * np.exp2(rng.integers(-2, 5, (R, 2, 1)))
    for half in (0, 1):
        for limit in clamps[2 * half : 2 * half + 2]:
            if limit is not None:
                at = rng.random((R, I))
                x[:, half][at < 0.2] = limit * (1 + rng.uniform(-0.1, 0.1, np.count_nonzero(at < 0.2)))
                x[:, half][(at > 0.2) & (at < 0.25)] = limit
                x[:, half][(at > 0.25) & (at < 0.27)] = limit * 100
    return x


@pytest.mark.parametrize("clamps", LIMITS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("I", [1, 37, 200])
def test_kept_bits_tell_clamped_values_from_all_others(clamps, dtype, I):
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd

    rng = np.random.default_rng(I)
    R, T = 50, 20
    t = tensor(_near_limits(rng, R, I, clamps), dtype)
    v = values(t)
    h, codes, scales, clamped = glu_checkpoint(t, **_kwargs(clamps), return_clamped=True)
    assert all(torch.equal(a, b) for a, b in zip((h, codes, scales), glu_checkpoint(t, **_kwargs(clamps))))
    out = np.stack([_sides(v[:, half], *clamps[2 * half : 2 * half + 2])[0] for half in (0, 1)], 1)
    assert clamped.shape == (R, 2, -(-I // 8)) and np.array_equal(_bits(clamped, I), out)
    assert not (np.unpackbits(clamped.cpu().numpy(), axis=-1, bitorder="little")[..., I:]).any()
    d = torch.ones((R, I), device="cuda")
    d_gu, h2 = glu_checkpoint_bwd(codes, scales, d, **_kwargs(clamps), clamped=clamped)
    plain, h3 = glu_checkpoint_bwd(codes, scales, d, **_kwargs(clamps))
    got, was = values(d_gu), values(plain)
    assert torch.equal(h2, h3) and not got[out].any() and np.array_equal(got[was != 0], was[was != 0])
    rec = ot.record_values(codes.cpu().numpy(), scales.cpu().numpy())
    g, u = ot.clamp_glu(rec[:, 0], rec[:, 1], [None if l is None else float(np.float32(l)) for l in clamps])
    act, slope = ot.act(g, "silu")
    for half, factor in ((0, u * slope), (1, act)):
        assert got[:, half][~out[:, half] & (np.abs(factor) > 2.0**-100)].all()
    # padding rows: no bit, none looked at
    ids = rng.integers(-1, T + 2, R).astype(np.int32)
    on = (ids >= 0) & (ids < T)
    table = dict(token_position_to_id=tensor(ids, "int32"), n_tokens=T)
    got = glu_checkpoint(t, **_kwargs(clamps), **table, return_clamped=True)[3]
    assert np.array_equal(got.cpu().numpy(), clamped.cpu().numpy() * on[:, None, None])


@pytest.mark.parametrize("clamps", LIMITS)
@pytest.mark.parametrize("N,I,B", [(2, 96, 40), (3, 37, 1), (1, 130, 64), (2, 9, 200), (1, 1000, 3)])
def test_bits_of_a_layers_checkpoint(clamps, N, I, B):
    """Set where the checkpoint holds the limit's bf16 or more: for every clamped value, and for none further than a step of bf16 inside."""
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint_bwd, pack_gate_up_checkpoint

    rng = np.random.default_rng(N + I + B)
    x = _near_limits(rng, N * B, I, clamps).astype(np.float32)
    f32 = [None if l is None else float(np.float32(l)) for l in clamps]
    g, u = ot.clamp_glu(x[:, 0], x[:, 1], [None if l is None else np.float32(l) for l in clamps])
    kept = tensor(np.stack((g, u), 1).reshape(N, B, 2, I).transpose(0, 2, 3, 1), "bfloat16")
    codes, scales, clamped = pack_gate_up_checkpoint(kept, **_kwargs(clamps), return_clamped=True)
    assert all(torch.equal(a, b) for a, b in zip((codes, scales), pack_gate_up_checkpoint(kept)))
    got = _bits(clamped, I)
    rows = values(kept).transpose(0, 3, 1, 2).reshape(N * B, 2, I)
    for half in (0, 1):
        hi, lo = f32[2 * half : 2 * half + 2]
        want = (rows[:, half] >= (np.inf if hi is None else ot.bf16_value(hi))) | (rows[:, half] <= (-np.inf if lo is None else ot.bf16_value(lo)))
        assert np.array_equal(got[:, half], want)
        assert got[:, half][_sides(x[:, half].astype(np.float64), hi, lo)[0]].all()
    d_gu, _ = glu_checkpoint_bwd(codes, scales, torch.ones((N * B, I), device="cuda"), **_kwargs(clamps), clamped=clamped)
    assert not values(d_gu)[got].any()
    ids = rng.integers(-1, 3, N * B).astype(np.int32)
    on = (ids >= 0) & (ids < 2)
    got = pack_gate_up_checkpoint(kept, tensor(ids, "int32"), 2, **_kwargs(clamps), return_clamped=True)[2]
    assert np.array_equal(got.cpu().numpy(), clamped.cpu().numpy() * on[:, None, None])


def test_bits_of_infinities_and_nan_and_without_limits():
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, pack_gate_up_checkpoint

    x = torch.tensor([[[float("inf"), float("-inf"), float("nan"), 2.0, 1.0]] * 2], device="cuda").bfloat16()
    for kw, want in (({}, [[0] * 5] * 2), (dict(gate_clamp_upper_limit=2.0), [[1, 0, 0, 1, 0], [0] * 5]),
                     (dict(up_clamp_lower_limit=-3.0, up_clamp_upper_limit=1.0), [[0] * 5, [1, 1, 0, 1, 1]])):
        assert _bits(glu_checkpoint(x, **kw, return_clamped=True)[3], 5)[0].tolist() == want
        assert _bits(pack_gate_up_checkpoint(x.view(1, 2, 5, 1), **kw, return_clamped=True)[2], 5)[0].tolist() == want


def test_refusals():
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd, pack_gate_up_checkpoint

    x = torch.zeros((4, 2, 36), device="cuda")
    _, c, s, m = glu_checkpoint(x, return_clamped=True)
    d = torch.zeros((4, 36), device="cuda")
    for bad in (m[:3], m[:, :, :4], m.int(), m[:, 0], m.bool()):
        with pytest.raises(AssertionError, match="NCC_INKI016"):
            glu_checkpoint_bwd(c, s, d, clamped=bad)
    with pytest.raises(AssertionError, match="NCC_INKI016"):
        pack_gate_up_checkpoint(torch.zeros((1, 2, 8, 4), device="cuda").bfloat16(), gate_clamp_upper_limit=7.0)
    h, c, s, m = glu_checkpoint(x[:0], return_clamped=True)
    assert m.shape == (0, 2, 5) and glu_checkpoint_bwd(c, s, d[:0], clamped=m)[0].shape == (0, 2, 36)
