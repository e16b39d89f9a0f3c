"""A row's codes and scale go by the row, not by the rows beside it: launches of few rows and of many add a row's squares in one order.

Sums of 64 bits in another order agree to a few of their last bits, and 1 / sqrt rounded to 32 bits differs only where it lies that near the
middle between two floats, once in 2^29 rows of random values.  So the rows are made: a few of their values bring the exact sum to
where 1 / sqrt is such a middle, and the two orders that a wave or a workgroup per row would take without care (a thread's pieces
one after the other, then the threads; or every piece by itself) are worked out on the host.
"""

from fractions import Fraction

import numpy as np
import pytest
import torch


def _wave_sum(v):
    v = v.reshape(*v.shape[:-1], 4, 16)
    for n in (8, 4, 2, 1):
        v = v + np.roll(v, n, -1)
    v = v[..., 0]
    return (v[..., 0] + v[..., 1]) + (v[..., 2] + v[..., 3])


def _threads(x, N, threads):
    """Every thread's sum of squares over its pieces of N values, one after the other."""
    rows, H = x.shape
    P = -(-H // (threads * N))
    p = np.zeros((rows, P * threads * N))
    p[:, :H] = x
    p = p.reshape(rows, P, threads, N)
    s = np.zeros((rows, threads))
    for a in range(P):
        for i in range(N):
            s = p[:, a, :, i] ** 2 + s  # (squares of 32-bit values are exact)
    return s


def _two_orders(x, N):
    w = _wave_sum(_threads(x, N, 256).reshape(len(x), 4, 64))
    return _wave_sum(_threads(x, N, 64)), ((w[:, 0] + w[:, 1]) + w[:, 2]) + w[:, 3]


def _made_rows(H, rows, steps, seed, dtype):
    """Rows of `dtype` ("float32", "bfloat16"), the last `steps` values of each (at places of their own) chosen so that
    1 / sqrt(mean of squares) is the middle between two floats, as near as the type lets it."""
    rng = np.random.default_rng(seed)
    cut = (lambda v: np.float32(v)) if dtype == "float32" else (lambda v: (np.float32(v).view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32))
    out = np.zeros((rows, H), np.float32)
    for x in out:
        x[:] = rng.standard_normal(H)
        if dtype != "float32":  # (squares of 16 bits: magnitudes wide enough that 64 bits do not hold every sum of them)
            x *= 2.0 ** -rng.integers(0, 28, H).astype(np.float32)
            x[:] = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        at = rng.permutation(H)[:steps]
        x[at] = 0
        s = sum(Fraction(float(v)) ** 2 for v in x)
        m = np.float32((float(s) * 1.01 / H) ** -0.5)
        middle = (Fraction(float(m)) + Fraction(float(np.nextafter(m, np.float32(9))))) / 2
        want = H / middle**2
        for j in at:
            v = cut(float(want - s) ** 0.5)
            while Fraction(float(v)) ** 2 > want - s:
                v = cut(np.nextafter(v, np.float32(0)))
            x[j] = v
            s += Fraction(float(v)) ** 2
    return out


# (fp32: a wave has four pieces a thread, three with a short one, two; bf16 with eight values a piece)
CASES = [("float32", 1024, 6, 4), ("float32", 700, 6, 4), ("float32", 515, 6, 4), ("float32", 412, 6, 4), ("bfloat16", 1030, 14, 8)]


def _case(dtype, H, steps, N):
    x = _made_rows(H, 96, steps, H, dtype)
    a, b = (1 / np.sqrt(s / H) for s in _two_orders(x.astype(np.float64), N))
    return x, a.astype(np.float32) != b.astype(np.float32)


@pytest.mark.parametrize("dtype,H,steps,N", CASES)
def test_the_rows_tell_the_orders_apart(dtype, H, steps, N):
    assert _case(dtype, H, steps, N)[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H,steps,N", CASES)
@pytest.mark.parametrize("code_dtype", ["int8", "float8_e4m3fn"])
def test_few_rows_and_many(dtype, H, steps, N, code_dtype):
    from nkilib.core.rmsnorm import rmsnorm_quant_rows

    x = torch.from_numpy(_case(dtype, H, steps, N)[0]).to(getattr(torch, dtype)).cuda()
    few = rmsnorm_quant_rows(x, None, eps=0.0, code_dtype=getattr(torch, code_dtype))
    many = rmsnorm_quant_rows(x.repeat(30, 1), None, eps=0.0, code_dtype=getattr(torch, code_dtype))
    for i in (0, 13, 29):
        assert torch.equal(many[1][96 * i :][:96], few[1]), f"scales, copy {i}"
        assert torch.equal(many[0][96 * i :][:96].view(torch.uint8), few[0].view(torch.uint8)), f"codes, copy {i}"
    alone = [rmsnorm_quant_rows(r, None, eps=0.0, code_dtype=getattr(torch, code_dtype)) for r in x[:8]]
    assert torch.equal(torch.stack([s for _, s in alone]), few[1][:8])
