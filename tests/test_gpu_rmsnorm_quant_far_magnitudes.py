"""The norm of rows whose values lie at the ends of what 32 bits hold: 1 / sqrt of their mean square is above the largest float, or no normal one.

Tolerances as in test_gpu_rmsnorm_quant_rows.py: the roundings are the same ones.
"""

import pytest
import torch

from group_helpers import assert_near
from test_gpu_rmsnorm_quant_rows import _check_codes, _formula

pytestmark = pytest.mark.gpu

# the root of the mean square: denormal values; around the least one whose inverse is a float (2^-128); ordinary; around the largest whose
# inverse is a normal one (2^126); the largest values there are
MAGNITUDES = [2.0**-138, 2.0**-130, 2.0**-128, 2.0**-127, 1.0, 2.0**125, 2.0**126, 1.9 * 2.0**126]


def _rows(dtype, H):
    g = torch.Generator(device="cuda").manual_seed(H)
    r = torch.rand((len(MAGNITUDES), 7, H), generator=g, device="cuda", dtype=torch.float64) + 0.4  # (none beyond 2^128)
    r *= torch.randint(0, 2, r.shape, generator=g, device="cuda") * 2 - 1
    r *= torch.tensor(MAGNITUDES, device="cuda", dtype=torch.float64)[:, None, None]
    gamma = (1 + 0.2 * torch.randn(H, generator=g, device="cuda")).to(dtype)
    d = torch.randn(r.shape, generator=g, device="cuda", dtype=torch.float64)
    return r.to(dtype).view(-1, H), gamma, d.view(-1, H)


@pytest.mark.parametrize("H", [129, 1024, 4096])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("code_dtype", ["int8", "float8_e4m3fn"])
def test_codes(dtype, H, code_dtype):
    from nkilib.core.rmsnorm import rmsnorm_quant_rows

    dt, cd = getattr(torch, dtype), getattr(torch, code_dtype)
    x, gamma, _ = _rows(dt, H)
    assert torch.isfinite(x).all()
    for eps in (0.0, 1e-90, 1e-6):
        for gm in (gamma, None):
            y = _formula(x.double(), gm, eps)
            c, s = rmsnorm_quant_rows(x, gm, eps=eps, code_dtype=cd)
            ok = torch.isfinite(y).all(1)  # (2^-138 is 0 in bf16, and without eps 0 / 0)
            assert bool((ok | (x == 0).all(1)).all()) and torch.isnan(s[~ok]).all() and not c[~ok].double().any()
            _check_codes(c[ok], s[ok], y[ok], f"eps {eps}")
            many = rmsnorm_quant_rows(x.repeat(40, 1), gm, eps=eps, code_dtype=cd)
            assert torch.equal(many[1][-len(x) :][ok], s[ok]) and torch.equal(many[0][-len(x) :].double(), c.double())


@pytest.mark.parametrize("H", [129, 1024, 4096])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_gradient(dtype, H):
    from nkilib.core.rmsnorm import rmsnorm_quant_rows_bwd

    dt = getattr(torch, dtype)
    x, gamma, d = _rows(dt, H)
    some = (x != 0).any(1)  # (2^-138 is 0 in bf16)
    x, d = x[some], d[some]
    # (the gradient is that of the values over their magnitude: it stays a float where that of the values is as small or as large)
    rms = (x.double() ** 2).mean(1, keepdim=True).sqrt()
    d = (d * rms.clamp(2.0**-100, 2.0**20)).to(dt)
    x64, g64 = x.double().requires_grad_(), gamma.double().requires_grad_()
    want, want_g = torch.autograd.grad(_formula(x64, g64, 0.0), (x64, g64), d.double())
    dx, dg = rmsnorm_quant_rows_bwd(d, x, gamma, eps=0.0)
    n, dn = x.double() / rms, d.double() * gamma.double()
    mag = (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True)) / rms
    assert_near(dx, want, mag, 9, "d_x")
    assert_near(dg, want_g, (d.double() * n).abs().sum(0), 9, "d_gamma")


def test_zeros_without_eps():
    """0 / 0 is no number, in either type."""
    from nkilib.core.rmsnorm import rmsnorm_quant_rows

    for dt in (torch.bfloat16, torch.float16, torch.float32):
        c, s = rmsnorm_quant_rows(torch.zeros((3, 70), device="cuda", dtype=dt), None, eps=0.0)
        assert torch.isnan(s).all() and not c.any()
