"""The norm into 8-bit rows and its gradient against their formulas in 64 bits.

Tolerances, in units u = 2^-24 (half a step of fp32, relative): y takes three roundings (1/sqrt, its product with s, gamma), the scale two
more (of the largest y: the division by M; the clamp rounds nothing), M / largest one and the product with y one.  So a scale is within
5 u of the formula's, and a code is the nearest to a number within 9 u of the formula's; the nearest int8 lies within 1/2, the
nearest e4m3 within 2^-4 of the value or 2^-10 (half the step below 2^-6).
"""

import pytest
import torch

from group_helpers import assert_near
from train_helpers import HALF, TINY

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = ["bfloat16", "float16", "float32"]
# one value, rows shorter than a vector, odd rows, every number of pieces per thread for a wave and for a workgroup per row, the longest
SHAPES = [(1, 1), (3, 5), (2, 64), (1, 7168), (8, 7168), (33, 1030), (5, 2049), (130, 4096), (3, 16384), (4, 16383), (2100, 130),
          (2048, 515), (2300, 1024), (2049, 2048), (2050, 2040), (2100, 4100)]


def _case(rows, H, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + H)
    dt = getattr(torch, dtype)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    wide = 1 + 20 * (torch.rand(H, generator=g, device="cuda") < 0.02)
    return (r(rows, H) * wide).to(dt), (r(rows, H) * wide).to(dt), (1 + 0.2 * r(H)).to(dt), r(rows, H).to(dt), r(rows, H).to(dt)


def _check_codes(codes, scales, y, what=""):
    M = 127.0 if codes.dtype == torch.int8 else 448.0
    scale = y.abs().amax(-1).clamp(min=2.0**-100) / M
    assert bool(((scales.double() - scale).abs() <= 5.1 * U * scale).all()), what
    v = y / scale[..., None]
    half = 0.5 if codes.dtype == torch.int8 else torch.clamp(2.0**-4 * v.abs(), min=2.0**-10)
    err = (codes.double() - v).abs()
    limit = half + 9.1 * U * v.abs()
    assert bool((err <= limit).all()), f"{what}: {(err - limit).max().item()} past"
    assert bool((codes.double().abs() <= M).all()), what


def _formula(s, gamma, eps):
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return y if gamma is None else y * gamma.double()


@pytest.mark.parametrize("rows,H", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code_dtype", ["int8", "float8_e4m3fn"])
def test_norm(rows, H, dtype, code_dtype):
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows

    x, r, gamma, _, _ = _case(rows, H, dtype)
    cd = getattr(torch, code_dtype)
    for res in (None, r):
        for gm, norm in ((gamma, True), (None, True), (None, False)):
            out = rmsnorm_quant_rows(x, gm, eps=1e-5, do_norm=norm, residual=res, code_dtype=cd)
            s = x.double()
            if res is not None:
                want = (x.float() + res.float()).to(x.dtype)  # (one addition of two values, rounded twice at most as torch does it)
                assert torch.equal(out[2], want)
                s = want.double()
            y = _formula(s, gm, 1e-5) if norm else s
            _check_codes(out[0], out[1], y, f"{rows} {H} {dtype} {code_dtype} {res is not None} {norm}")
            assert len(out) == (2 if res is None else 3) and out[0].dtype == cd and out[1].shape == (rows,)
    for dt in DTYPES:
        got = dequantize_rows(out[0], out[1], getattr(torch, dt))
        want = out[0].double() * out[1].double()[:, None]
        assert_near(got, want, want.abs(), 1, dt)


def test_gamma_of_another_type_and_shapes():
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

    x, r, gamma, d, _ = _case(6, 1032, "bfloat16")
    for g in (gamma.float(), gamma.half(), gamma.view(1, -1)):
        _check_codes(*rmsnorm_quant_rows(x, g), _formula(x.double(), g.reshape(-1), 1e-6))
        dx, dg = rmsnorm_quant_rows_bwd(d, x, g)
        assert dg.dtype == g.dtype and dg.shape == g.shape
    c, s, t = rmsnorm_quant_rows(x.view(2, 3, -1), gamma, residual=r.view(2, 3, -1))
    c2, s2, t2 = rmsnorm_quant_rows(x, gamma, residual=r)
    assert c.shape == (2, 3, 1032) and s.shape == (2, 3) and torch.equal(c.view(6, -1), c2) and torch.equal(s.view(6), s2)
    assert torch.equal(dequantize_rows(c, s).view(6, -1), dequantize_rows(c2, s2))
    c1, s1 = rmsnorm_quant_rows(t2[4], gamma)  # a row alone, and its sum as input: the same bits
    assert c1.shape == (1032,) and s1.shape == () and torch.equal(c1, c2[4]) and torch.equal(s1, s2[4])
    assert torch.equal(rmsnorm_quant_rows(x.t().contiguous().t(), gamma)[0], rmsnorm_quant_rows(x, gamma)[0])
    assert rmsnorm_quant_rows(x[:0], gamma)[0].shape == (0, 1032)


def test_a_row_does_not_depend_on_the_others():
    """A wave or a workgroup per row, one or several rounds: the same bits."""
    from nkilib.core.rmsnorm import rmsnorm_quant_rows

    x, r, gamma, _, _ = _case(5000, 1024, "bfloat16")
    many = rmsnorm_quant_rows(x, gamma, residual=r)
    few = rmsnorm_quant_rows(x[:100].contiguous(), gamma, residual=r[:100].contiguous())
    # (sums of 64-bit products taken in another order may round 1 / sqrt otherwise, once in 2^29 rows; these 100 do not)
    assert all(torch.equal(a[:100], b) for a, b in zip(many, few))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code_dtype", ["int8", "float8_e4m3fn"])
def test_rows_of_zeros_tiny_huge_and_not_finite(dtype, code_dtype):
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows

    dt, cd = getattr(torch, dtype), getattr(torch, code_dtype)
    top = torch.finfo(dt).max
    x = torch.randn((9, 130), device="cuda").to(dt)
    x[0] = 0
    x[1] = torch.finfo(dt).tiny
    x[2] = top
    x[3, 7] = float("nan")
    x[4, 129] = float("inf")
    x[5, 0] = -float("inf")
    x[6] = 0
    x[6, 128] = -top
    gamma = torch.ones(130, device="cuda").to(dt)
    for norm in (True, False):
        c, s = rmsnorm_quant_rows(x, gamma if norm else None, do_norm=norm, code_dtype=cd)
        assert torch.isnan(s[3:6]).all() and not c[3:6].double().any()
        ok = [0, 1, 2, 6, 7, 8]
        y = _formula(x.double(), gamma, 1e-6) if norm else x.double()
        assert bool((s[0] > 0).all()) and not c[0].double().any()
        if norm or dtype != "bfloat16":
            _check_codes(c[ok], s[ok], y[ok], f"{dtype} {norm}")
        else:  # (1e-38 without a norm lies below the least magnitude: codes 0)
            _check_codes(c[[2, 6, 7, 8]], s[[2, 6, 7, 8]], y[[2, 6, 7, 8]], f"{dtype} {norm}")
        assert torch.isnan(dequantize_rows(c, s)[3:6]).all()
    c, s, t = rmsnorm_quant_rows(x[2:3], gamma, residual=x[2:3], code_dtype=cd)  # the sum passes the type
    if dtype != "bfloat16":
        assert torch.isinf(t).all() and torch.isnan(s).all()


@pytest.mark.parametrize("rows,H", SHAPES + [(1030, 256), (3000, 4096)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(rows, H, dtype):
    from nkilib.core.rmsnorm import rmsnorm_quant_rows_bwd

    x, _, gamma, d, res = _case(rows, H, dtype, 1)
    for gm, rs in ((gamma, res), (gamma, None), (None, res)):
        dx, dg = rmsnorm_quant_rows_bwd(d, x, gm, eps=1e-5, d_residual=rs)
        x64 = x.double().requires_grad_()
        g64 = (gamma.double() if gm is not None else torch.ones(H, dtype=torch.float64, device="cuda")).requires_grad_()
        want, want_g = torch.autograd.grad(_formula(x64, g64, 1e-5), (x64, g64), d.double())
        inv = 1 / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-5)
        n, dn = x.double() * inv, d.double() * g64.detach()
        mag = inv * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True))
        if rs is not None:
            want, mag = want + rs.double(), mag + rs.double().abs()
        # 1/sqrt, n, dn, the mean's terms and the mean, its product, the difference, the product with 1/sqrt, the sum with the residual's
        assert_near(dx, want, mag, 9, f"{rows} {H} {dtype}")
        if gm is None:
            assert dg is None
        else:  # two roundings of n, its product, a chain of at most 1 + rows / 512 additions and three more; the parts' sum is in 64
            # bits, rounded to 32
            assert_near(dg, want_g, (d.double() * n).abs().sum(0), 8 + rows // 512, f"gamma {rows} {H} {dtype}")


def test_gradient_against_differences():
    """The loss sum(y d) of the formula in 64 bits changes with hidden and gamma as the gradients say."""
    from nkilib.core.rmsnorm import rmsnorm_quant_rows_bwd

    x, _, gamma, d, _ = _case(4, 66, "float32", 2)
    dx, dg = rmsnorm_quant_rows_bwd(d, x, gamma, eps=1e-3)
    loss = lambda x, g: (_formula(x, g, 1e-3) * d.double()).sum()
    h = 1e-4
    for i, j in ((0, 0), (3, 65), (1, 33)):
        e = torch.zeros_like(x, dtype=torch.float64)
        e[i, j] = h
        diff = (loss(x.double() + e, gamma) - loss(x.double() - e, gamma)) / (2 * h)
        assert abs(diff - dx[i, j]) <= 1e-5 * dx.abs().max()
        diff = (loss(x.double(), gamma.double() + e[i]) - loss(x.double(), gamma.double() - e[i])) / (2 * h)
        assert abs(diff - dg[j]) <= 1e-5 * dg.abs().max()


def test_addresses_in_a_graph_and_on_a_stream():
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

    x, r, gamma, d, res = _case(40, 516, "bfloat16", 3)
    want = rmsnorm_quant_rows(x, gamma, residual=r)
    buf = torch.zeros(40 * 516 + 3, dtype=torch.bfloat16, device="cuda")
    for shift in (1, 3):
        moved = buf[shift:][: 40 * 516].view(40, 516)
        moved.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(rmsnorm_quant_rows(moved, gamma, residual=r), want))

    def step():
        c, s, t = rmsnorm_quant_rows(x, gamma, residual=r)
        return (c, s, t, dequantize_rows(c, s), *rmsnorm_quant_rows_bwd(d, t, gamma, d_residual=res))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(torch.randn_like(x))
        d.copy_(torch.randn_like(d))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_refusals():
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, device="cuda", dtype=dt)
    x, g, c, s = z(4, 8), z(8), z(4, 8, dt=torch.int8), z(4, dt=torch.float32)
    bad = [
        lambda: rmsnorm_quant_rows(x.double(), g), lambda: rmsnorm_quant_rows(z(2, 16385), None), lambda: rmsnorm_quant_rows(z(2, 0), None),
        lambda: rmsnorm_quant_rows(x, z(7)), lambda: rmsnorm_quant_rows(x, g.double()), lambda: rmsnorm_quant_rows(x, g, do_norm=False),
        lambda: rmsnorm_quant_rows(x, g, residual=z(4, 7)), lambda: rmsnorm_quant_rows(x, g, residual=x.half()),
        lambda: rmsnorm_quant_rows(x, g, eps=-1.0), lambda: rmsnorm_quant_rows(x, g, eps=float("nan")),
        lambda: rmsnorm_quant_rows(x, g, code_dtype=torch.uint8), lambda: rmsnorm_quant_rows_bwd(z(4, 7), x, g),
        lambda: rmsnorm_quant_rows_bwd(x.half(), x, g), lambda: rmsnorm_quant_rows_bwd(x, x, z(9)),
        lambda: rmsnorm_quant_rows_bwd(x, x, g, d_residual=z(3, 8)), lambda: rmsnorm_quant_rows_bwd(x, x, g, eps=-1),
        lambda: dequantize_rows(x, s), lambda: dequantize_rows(c, s[:3]), lambda: dequantize_rows(c, s.half()),
        lambda: dequantize_rows(c, s, torch.float64), lambda: dequantize_rows(c, s[:, None]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was not refused")
