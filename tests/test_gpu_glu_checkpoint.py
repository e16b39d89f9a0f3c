"""The gated activation with its inputs in 8 bits: records bit for bit, values and gradients against the oracle in 64 bits.

Tolerances: an error of z, the argument of the exponential (of erfc), is one of |z| times as much in the result, relative; z is
rounded once per product that makes it (``_steps``), and rows of 16 bits also round it to the exponent of the hardware's 2^x,
which rows of fp32 make good.  s(x) = act(x) / x is held in fp32: below 2^-126 its steps are 2^-149 and no longer relative, or it
is zero, so what it multiplies counts 2^-126 times (erfc(7.1) = 1e-23, erfc(9.4) = 2.5e-40: x = -13.3 among normal values times
8).  The slope is a sum of two parts, whose magnitudes count, as they may cancel.
"""

import numpy as np
import pytest

from oracle import train as ot
from train_helpers import assert_within, bound, tensor, values

pytestmark = pytest.mark.gpu

ACTS = {"silu": "SiLU", "gelu": "GELU", "gelu_tanh": "GELU_Tanh_Approx", "swish": "Swish"}
DTYPES = ["bfloat16", "float16", "float32"]
# R, I: one value, short groups, rows whose length is no multiple of 8 (of 4, of 2), more than a workgroup's pieces in a row
SHAPES = [(1, 1), (3, 31), (2, 32), (5, 33), (17, 100), (40, 192), (9, 1030), (3, 2048), (2, 14337)]


def _act(kind):
    from nkilib.core.utils.common_types import ActFnType

    return ActFnType[ACTS[kind]]


def _steps(x, kind, dtype):
    """Error of the activation in units of 2^-24 of its magnitude: 16 for the arithmetic (erfc, exponential, reciprocal, products),
    and what the roundings of z cost (beyond |z| = 130 the value is 0 or x)."""
    x = np.abs(x)
    z = {"silu": x, "swish": 1.702 * x, "gelu": x * x, "gelu_tanh": 1.6 * (x + 0.0448 * x**3)}[kind]
    return 16 + (0 if kind == "silu" and dtype == "float32" else 4) * np.minimum(z, 130.0)


def _slope_magnitude(g, kind):
    a, da = ot.act(g, kind)
    with np.errstate(invalid="ignore", divide="ignore"):
        s = np.where(g == 0, 0.5, a / g)
    return np.abs(s) + np.abs(da - s)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", list(ACTS))
def test_forward(shape, dtype, kind):
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint

    R, I = shape
    rng = np.random.default_rng(R + I)
    x = tensor(rng.standard_normal((R, 2, I)) * np.exp2(rng.integers(-4, 3, (R, 2, 1))), dtype)
    h, codes, scales = glu_checkpoint(x, _act(kind))
    v = values(x)
    want_c, want_s = ot.record(v)
    assert np.array_equal(codes.cpu().numpy(), want_c) and np.array_equal(scales.cpu().numpy(), want_s)
    a, _ = ot.act(v[:, 0], kind)
    want = a * v[:, 1]
    limit = bound(want, np.abs(want) * _steps(v[:, 0], kind, dtype), dtype, 1) + 2.0**-126 * np.abs(v[:, 0] * v[:, 1])
    assert_within(h, want, limit, f"{shape} {dtype} {kind}")
    assert np.array_equal(values(dequantize_checkpoint(codes, scales)), ot.record_values(want_c, want_s))
    import torch

    assert np.array_equal(values(dequantize_checkpoint(codes, scales, torch.float32)), ot.record_values(want_c, want_s))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", list(ACTS))
@pytest.mark.parametrize("clamped", [False, True])
def test_backward(shape, dtype, kind, clamped):
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint_bwd

    R, I = shape
    rng = np.random.default_rng(R + 2 * I)
    codes, scales = ot.record((rng.standard_normal((R, 2, I)) * 3).astype(np.float32))
    v = ot.record_values(codes, scales)
    d = tensor(rng.standard_normal((R, I)), dtype)
    clamps = (2.0, None, 1.5, -1.0) if clamped else (None,) * 4
    names = ("gate_clamp_upper_limit", "gate_clamp_lower_limit", "up_clamp_upper_limit", "up_clamp_lower_limit")
    import torch

    d_gu, h = glu_checkpoint_bwd(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), d, _act(kind),
                                 **{n: c for n, c in zip(names, clamps) if c is not None})
    dv = values(d)
    dg, du, want_h = ot.glu_bwd(v[:, 0], v[:, 1], dv, kind, clamps)
    g, u = ot.clamp_glu(v[:, 0], v[:, 1], clamps)
    steps, small = _steps(g, kind, dtype), 2.0**-126
    what = f"{shape} {dtype} {kind} {clamped}"
    assert_within(h, want_h, bound(want_h, np.abs(want_h) * steps, dtype, 1) + small * np.abs(g * u), "h " + what)
    assert_within(d_gu[:, 1].contiguous(), du, bound(du, np.abs(du) * steps, dtype, 1) + small * np.abs(dv * g), "du " + what)
    mag = np.abs(dv * u) * _slope_magnitude(g, kind) * steps
    assert_within(d_gu[:, 0].contiguous(), dg, bound(dg, mag, dtype, 1) + small * np.abs(dv * u) * (1 + np.abs(g)), "dg " + what)
    only, none = glu_checkpoint_bwd(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), d, _act(kind),
                                    **{n: c for n, c in zip(names, clamps) if c is not None}, return_intermediate=False)
    assert none is None and torch.equal(only, d_gu)


@pytest.mark.parametrize("N,I,B", [(1, 1, 1), (3, 33, 1), (2, 64, 4), (3, 100, 16), (2, 1024, 60), (2, 130, 64), (1, 96, 200), (3, 256, 128),
                                   (1, 9000, 1), (2, 513, 512)])
def test_pack(N, I, B):
    from nkilib.core.moe.glu_checkpoint import pack_gate_up_checkpoint

    rng = np.random.default_rng(N + I + B)
    x = tensor(rng.standard_normal((N, 2, I, B)) * np.exp2(rng.integers(-9, 9, (N, 2, 1, B))), "bfloat16")
    rows = values(x).transpose(0, 3, 1, 2).reshape(N * B, 2, I)
    want_c, want_s = ot.record(rows)
    codes, scales = pack_gate_up_checkpoint(x)
    assert np.array_equal(codes.cpu().numpy(), want_c) and np.array_equal(scales.cpu().numpy(), want_s)
    ids = rng.integers(-1, 3, N * B).astype(np.int32)
    on = ((ids >= 0) & (ids < 2))[:, None, None]
    codes, scales = pack_gate_up_checkpoint(x, tensor(ids, "int32"), 2)
    assert np.array_equal(codes.cpu().numpy(), want_c * on) and np.array_equal(scales.cpu().numpy(), want_s * on)
    # the same bits begun at an address that is aligned to an element only
    import torch

    flat = torch.empty(x.numel() + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x.reshape(-1)
    c2, s2 = pack_gate_up_checkpoint(flat[1:].view(x.shape))
    assert np.array_equal(c2.cpu().numpy(), want_c) and np.array_equal(s2.cpu().numpy(), want_s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_values(dtype):
    """Infinities and NaN: in the record as NaN, without a part in their neighbours' scale; slopes of values far out; zeros,
    subnormals, the borders of the scale rule."""
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd, pack_gate_up_checkpoint

    rng = np.random.default_rng(7)
    x = rng.standard_normal((8, 2, 70)).astype(np.float32)
    x[0, 0, 3], x[0, 0, 40], x[0, 1, 69] = np.inf, -np.inf, np.nan
    x[1] = 0
    x[1, 0, 0] = -0.0
    x[2] *= 1e-38 if dtype != "float16" else 1e-7
    x[3] *= 1e30 if dtype != "float16" else 2e4
    x[4, 0, :32], x[4, 1, :32], x[4, 1, 5] = 448.0, 7.0, 450.0
    x[5, 0] = np.linspace(-200, 200, 70)
    t = tensor(x, dtype)
    v = values(t)
    want_c, want_s = ot.record(v)
    h, codes, scales = glu_checkpoint(t)
    nan = (want_c & 0x7F) == 0x7F  # (a NaN has no sign)
    assert np.array_equal(np.where(nan, codes.cpu().numpy() | 0x80, codes.cpu().numpy()), np.where(nan, 0xFF, want_c))
    assert np.array_equal(scales.cpu().numpy(), want_s)
    with np.errstate(all="ignore"):
        a, _ = ot.act(v[:, 0], "silu")
        want = a * v[:, 1]
    fits = np.abs(want) < (6e4 if dtype == "float16" else 3e38)
    ok = fits & np.isfinite(v[:, 0]) & np.isfinite(v[:, 1])
    # (a sigmoid below 2^-126 may become zero, and so may a product)
    with np.errstate(all="ignore"):
        limit = bound(want, np.abs(want) * 700, dtype, 1) + 2.0**-126 * (1 + np.abs(v[:, 0] * v[:, 1]))
    assert (np.abs(values(h) - want)[ok] <= limit[ok]).all()
    # an infinite gate: act(inf) = inf; the slope there is one, at -inf zero
    assert np.isinf(values(h)[0, 3]) and np.isnan(values(h)[0, 69])
    # large recorded values have slopes 0 and 1
    big = torch.tensor([[[-3e38, -1e20, -200.0, 200.0, 1e20, 3e38] + [0.0] * 26] * 2], device="cuda")
    big[:, 1] = 1.0
    for kind in ACTS:
        for i in range(6):
            one = torch.zeros_like(big)
            one[:, 0, i], one[:, 1] = big[:, 0, i], 1.0
            _, c, s = glu_checkpoint(one, _act(kind))
            d_gu, _ = glu_checkpoint_bwd(c, s, torch.ones((1, 32), device="cuda"), _act(kind))
            assert float(d_gu[0, 0, i]) == (1.0 if i >= 3 else 0.0), (kind, i)
    if dtype == "bfloat16":
        c2, s2 = pack_gate_up_checkpoint(t.permute(1, 2, 0).reshape(1, 2, 70, 8).contiguous())
        assert torch.equal(c2, codes) and torch.equal(s2, scales)


@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_rows(dtype):
    """Rows whose id is no token: not read (they hold NaN here), zero in every output."""
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd
    from nkilib.core.utils.common_types import ActFnType

    rng = np.random.default_rng(8)
    R, I, T = 50, 77, 20
    ids = rng.integers(-1, T + 2, R).astype(np.int32)
    on = torch.from_numpy((ids >= 0) & (ids < T)).cuda()
    x = tensor(rng.standard_normal((R, 2, I)) * 3, dtype)
    opts = dict(activation_function=ActFnType.Swish, gate_clamp_upper_limit=2.0, gate_clamp_lower_limit=0.5, up_clamp_lower_limit=1.0)
    want = glu_checkpoint(x, **opts)
    d = tensor(rng.standard_normal((R, I)), dtype)
    want_b = glu_checkpoint_bwd(*want[1:], d, **opts)
    x[~on], d[~on] = float("nan"), float("nan")
    codes, scales = want[1].clone(), want[2].clone()
    codes[~on] = 0x7F
    table = dict(token_position_to_id=tensor(ids, "int32"), n_tokens=T)
    got = (*glu_checkpoint(x, **opts, **table), *glu_checkpoint_bwd(codes, scales, d, **opts, **table))
    for g, w in zip(got, (*want, *want_b)):
        w = w.clone()
        w[~on] = 0
        assert torch.equal(g, w)


def test_clamped_values_have_no_gradient():
    """A gate of 7 with a limit of 7 has been clamped: forward keeps the clamped value, backward passes nothing through."""
    import torch
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd

    x = torch.tensor([[[9.0, 7.0, 3.0, -9.0] * 8, [1.0, -8.0, 7.0, 2.0] * 8]], device="cuda")
    opts = dict(gate_clamp_upper_limit=7.0, up_clamp_upper_limit=7.0, up_clamp_lower_limit=-7.0)
    _, c, s = glu_checkpoint(x, **opts)
    assert dequantize_checkpoint(c, s)[0, :, :4].tolist() == [[7.0, 7.0, 3.0, -9.0], [1.0, -7.0, 7.0, 2.0]]
    d_gu, _ = glu_checkpoint_bwd(c, s, torch.ones((1, 32), device="cuda"), **opts)
    assert (d_gu[0, :, :4] != 0).tolist() == [[False, False, True, True], [True, False, False, True]]


def test_records_beyond_32_bit_offsets():
    import torch
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd

    I, R = 131072, 8200  # 2.15 G values; the last row is looked at
    x = torch.zeros((R, 2, I), dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn((2, I), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").bfloat16()
    h, c, s = glu_checkpoint(x)
    h1, c1, s1 = glu_checkpoint(x[-1:].contiguous())
    assert torch.equal(h[-1:], h1) and torch.equal(c[-1:], c1) and torch.equal(s[-1:], s1)
    assert not h[:-1].any()
    v = dequantize_checkpoint(c[-1:], s[-1:])
    del x
    d_gu, h2 = glu_checkpoint_bwd(c, s, h)
    d1, h3 = glu_checkpoint_bwd(c1, s1, h1)
    assert torch.equal(d_gu[-1:], d1) and torch.equal(h2[-1:], h3) and v.any()


def test_refusals():
    import torch
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd, pack_gate_up_checkpoint

    x = torch.zeros((4, 2, 64), device="cuda")
    _, c, s = glu_checkpoint(x)
    d = torch.zeros((4, 64), device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [
        lambda: glu_checkpoint(x.double()), lambda: glu_checkpoint(x.view(4, 128)), lambda: glu_checkpoint(x, activation_function=0),
        lambda: glu_checkpoint(x, token_position_to_id=ids), lambda: glu_checkpoint(x, token_position_to_id=ids[:3], n_tokens=4),
        lambda: glu_checkpoint(x, token_position_to_id=ids.long(), n_tokens=4),
        lambda: glu_checkpoint_bwd(c, s[:, :, :1], d), lambda: glu_checkpoint_bwd(c.int(), s, d), lambda: glu_checkpoint_bwd(c, s, d[:3]),
        lambda: glu_checkpoint_bwd(c, s, d.double()), lambda: pack_gate_up_checkpoint(x.view(1, 2, 64, 4)),
        lambda: pack_gate_up_checkpoint(x.bfloat16()), lambda: dequantize_checkpoint(c, s, torch.float64),
        lambda: glu_checkpoint(torch.zeros((1, 2, 131073), device="cuda")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError, match="NCC_INKI016"):
            call()
            pytest.fail(f"call {i} was not refused")
    # no rows: nothing is launched
    h, c0, s0 = glu_checkpoint(x[:0])
    assert h.shape == (0, 64) and c0.shape == (0, 2, 64) and glu_checkpoint_bwd(c0, s0, d[:0])[0].shape == (0, 2, 64)
