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
    codes, scales = pack_gate_up_checkpoint(gate_up_T, tp, T)
    d_gu, _ = glu_checkpoint_bwd(codes, scales, torch.ones((be.numel() * B, I), device="cuda"), token_position_to_id=tp,
                                 n_tokens=T, **_kwargs(clamps))
    got, tpn = values(d_gu), tp.cpu().numpy()
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
            seen += out.sum()
    assert seen > 1000
