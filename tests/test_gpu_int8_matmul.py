"""Products in 8-bit integers against whole numbers in 64 bits.

Tolerance: the sum is exact; its conversion to fp32, the product with each scale and the addition of the bias round once each (2^-24
of what they round), and the result is rounded once to its type.
"""

import pytest
import torch

from group_helpers import assert_near, groups, offsets_of

pytestmark = pytest.mark.gpu

OUT = ["bfloat16", "float16", "float32"]


def _codes(g, *shape, full=False):
    if full:
        return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    return (torch.randn(shape, generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)


def _scales(g, *shape):
    return torch.rand(shape, generator=g, device="cuda") * 0.02 + 0.001


def _want(x, xs, w, ws):
    return (x.double() @ w.double().t().contiguous()) * xs.double()[:, None] * ws.double()


@pytest.mark.parametrize("S,K,N", [(1, 64, 64), (1, 7168, 4096), (2, 1, 1), (3, 7, 5), (5, 16, 1),
                                   (16, 128, 136), (17, 129, 515), (33, 1030, 77),
                                   (64, 2048, 256), (100, 200, 264), (257, 384, 512), (300, 1040, 1030), (1000, 14336, 320), (7, 131071, 24)])
@pytest.mark.parametrize("out", OUT)
def test_dense(S, K, N, out):
    from nkilib.core.int8_matmul import int8_matmul

    g = torch.Generator(device="cuda").manual_seed(S + K)
    dt = getattr(torch, out)
    x, w, xs, ws = _codes(g, S, K, full=True), _codes(g, N, K, full=True), _scales(g, S), _scales(g, N)
    want = _want(x, xs, w, ws)
    got = int8_matmul(x, xs, w, ws, out_dtype=dt)
    assert got.dtype == dt
    if out != "float16" or K < 2000:  # (codes of 128 at every place: past what 16 bits hold)
        assert_near(got, want, want.abs(), 4, f"{S} {K} {N}")
    bias = (torch.randn(N, generator=g, device="cuda") * 10).to(dt)
    got = int8_matmul(x, xs[:, None], w, ws, bias=bias, out_dtype=dt)
    if out != "float16" or K < 2000:
        assert_near(got, want + bias.double(), want.abs() + bias.double().abs(), 5, f"bias {S} {K} {N}")


def test_extreme_codes_are_exact():
    """-128 by -128 over the longest rows: the largest sum there is."""
    from nkilib.core.int8_matmul import int8_matmul

    for K in (131071, 131056):
        x = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
        w = torch.full((20, K), -128, dtype=torch.int8, device="cuda")
        w[1] = 127
        one = lambda n: torch.ones(n, device="cuda")
        got = int8_matmul(x, one(3), w, one(20), out_dtype=torch.float32)
        want = torch.full((3, 20), 16384.0 * K, device="cuda")
        want[:, 1] = -128.0 * 127 * K
        assert torch.equal(got, want)


@pytest.mark.parametrize("counts,ahead,behind,K,N", [([1], 0, 0, 64, 64), ([0] * 60 + [1, 2, 0, 1], 0, 0, 2048, 768),
                                                        ([3, 0, 20, 1], 2, 3, 77, 39),
                                                    ([40, 0, 129, 300, 16], 1, 9, 256, 520), ([512, 256, 255, 257], 0, 0, 512, 512),
                                                    ([0, 0], 3, 4, 128, 128), ([700, 2, 90], 0, 0, 1030, 515)])
@pytest.mark.parametrize("out", OUT)
def test_grouped(counts, ahead, behind, K, N, out):
    from nkilib.core.int8_matmul import grouped_int8_matmul

    g = torch.Generator(device="cuda").manual_seed(K + N)
    S, E, o = ahead + sum(counts) + behind, len(counts), offsets_of(counts, ahead)
    x, w, xs, ws = _codes(g, S, K), _codes(g, E, N, K), _scales(g, S), _scales(g, E, N)
    want = torch.zeros((S, N), dtype=torch.float64, device="cuda")
    for e, a, b in groups(o, S):
        want[a:b] = _want(x[a:b], xs[a:b], w[e], ws[e])
    got = grouped_int8_matmul(x, xs, w, ws, torch.from_numpy(o).cuda(), out_dtype=getattr(torch, out))
    assert_near(got, want, want.abs(), 4)
    assert not got[:ahead].any() and not got[S - behind :].any()


def test_scales_that_are_not_finite_and_rows_of_none():
    """A row whose scale is NaN comes out as NaN, alone; rows of no expert are zero whatever their scales are."""
    from nkilib.core.int8_matmul import grouped_int8_matmul, int8_matmul

    g = torch.Generator(device="cuda").manual_seed(2)
    x, w, xs, ws = _codes(g, 40, 96), _codes(g, 2, 48, 96), _scales(g, 40), _scales(g, 2, 48)
    o = torch.tensor([5, 20, 30], dtype=torch.int32, device="cuda")
    clean = grouped_int8_matmul(x, xs, w, ws, o)
    xs1 = xs.clone()
    xs1[0], xs1[35], xs1[8] = float("nan"), float("inf"), float("nan")
    got = grouped_int8_matmul(x, xs1, w, ws, o)
    assert not got[:5].any() and not got[30:].any() and torch.isnan(got[8]).all()
    keep = torch.arange(40, device="cuda") != 8
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(int8_matmul(x, xs1, w[0], ws[0])[8]).all()


def test_leading_dimensions_views_and_addresses():
    from nkilib.core.int8_matmul import int8_matmul

    g = torch.Generator(device="cuda").manual_seed(3)
    x, w, xs, ws = _codes(g, 6, 160), _codes(g, 72, 160), _scales(g, 6), _scales(g, 72)
    want = int8_matmul(x, xs, w, ws)
    assert torch.equal(int8_matmul(x.view(2, 3, 160), xs.view(2, 3), w, ws), want.view(2, 3, 72))
    assert torch.equal(int8_matmul(x.view(2, 3, 160), xs.view(2, 3, 1), w, ws), want.view(2, 3, 72))
    assert torch.equal(int8_matmul(x[4], xs[4], w, ws), want[4])
    assert int8_matmul(x[:0], xs[:0], w, ws).shape == (0, 72) and int8_matmul(x, xs, w[:0], ws[:0]).shape == (6, 0)
    for shift in (1, 2, 7, 16):
        buf = torch.zeros(6 * 160 + 16, dtype=torch.int8, device="cuda")
        moved = buf[shift:][: 6 * 160].view(6, 160)
        moved.copy_(x)
        assert torch.equal(int8_matmul(moved, xs, w, ws), want)
    assert torch.equal(int8_matmul(x.t().contiguous().t(), xs, w, ws), want)
    bias = torch.ones(72, device="cuda").bfloat16()
    assert torch.equal(int8_matmul(x[:, :0], xs, w[:, :0], ws, bias), bias.expand(6, 72))
    assert not int8_matmul(x[:, :0], xs, w[:, :0], ws, bias.clone().requires_grad_()).requires_grad
    assert not int8_matmul(x[:, :0], xs, w[:, :0], ws).any()


def test_in_a_graph():
    from nkilib.core.int8_matmul import grouped_int8_matmul, int8_matmul

    g = torch.Generator(device="cuda").manual_seed(4)
    x, w, xs, ws = _codes(g, 64, 256), _codes(g, 4, 136, 256), _scales(g, 64), _scales(g, 4, 136)
    o = torch.tensor([0, 10, 10, 40, 60], dtype=torch.int32, device="cuda")
    step = lambda: (int8_matmul(x, xs, w[0], ws[0]), grouped_int8_matmul(x, xs, w, ws, o))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i, bounds in enumerate(([0, 10, 10, 40, 60], [0, 64, 64, 64, 64], [3, 4, 5, 6, 7])):
        o.copy_(torch.tensor(bounds, dtype=torch.int32))
        x.copy_(_codes(g, 64, 256))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_refusals():
    from nkilib.core.int8_matmul import grouped_int8_matmul, int8_matmul

    z = lambda *s, dt=torch.int8: torch.zeros(s, device="cuda", dtype=dt)
    f = lambda *s: torch.zeros(s, device="cuda")
    x, w, xs, ws, o = z(4, 8), z(6, 8), f(4), f(6), z(3, dt=torch.int32)
    bad = [
        lambda: int8_matmul(x.float(), xs, w, ws), lambda: int8_matmul(x, xs, w.float(), ws), lambda: int8_matmul(x, xs.half(), w, ws),
        lambda: int8_matmul(x, xs, w, ws.double()), lambda: int8_matmul(x, f(5), w, ws), lambda: int8_matmul(x, xs, w, f(7)),
        lambda: int8_matmul(x, xs, z(6, 9), ws), lambda: int8_matmul(x, xs, z(1, 6, 8), ws),
        lambda: int8_matmul(x, xs, w, ws, out_dtype=torch.float64),
        lambda: int8_matmul(x, xs, w, ws, bias=f(6)), lambda: int8_matmul(x, xs, w, ws, bias=f(5), out_dtype=torch.float32),
        lambda: int8_matmul(z(1, 2**17), f(1), z(2, 2**17), f(2)), lambda: grouped_int8_matmul(x, xs, z(2, 6, 8), f(2, 6), o.long()),
        lambda: grouped_int8_matmul(x, xs, z(2, 6, 8), f(2, 6), o[:2]), lambda: grouped_int8_matmul(x, xs, z(2, 6, 8), f(6, 2), o),
        lambda: grouped_int8_matmul(x, xs, z(2, 8, 6), f(2, 8), o), lambda: grouped_int8_matmul(z(2, 2, 8), f(2, 2), z(2, 6, 8), f(2, 6), o),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("N", [144, 1040, 8208, 131, 1027, 8195])
@pytest.mark.parametrize("K", [64, 160, 1040, 77, 1030, 68, 124, 1028])
@pytest.mark.parametrize("out", OUT)
def test_every_kind_of_tile(K, N, out):
    """As for the 16-bit products: few columns, some and many, aligned or not, one step and several; and a dense product of as many rows."""
    from nkilib.core.int8_matmul import grouped_int8_matmul, int8_matmul
    from test_gpu_grouped_matmul import EVERY_TILE

    g = torch.Generator(device="cuda").manual_seed(K + N)
    S, E, o = sum(EVERY_TILE), len(EVERY_TILE), offsets_of(EVERY_TILE)
    x, w, xs, ws = _codes(g, S, K), _codes(g, E, N, K), _scales(g, S), _scales(g, E, N)
    want = torch.zeros((S, N), dtype=torch.float64, device="cuda")
    for e, a, b in groups(o, S):
        want[a:b] = _want(x[a:b], xs[a:b], w[e], ws[e])
    dt = getattr(torch, out)
    assert_near(grouped_int8_matmul(x, xs, w, ws, torch.from_numpy(o).cuda(), out_dtype=dt), want, want.abs(), 4)
    bias = torch.randn(N, generator=g, device="cuda").to(dt)
    want = _want(x, xs, w[0], ws[0])
    assert_near(int8_matmul(x, xs, w[0], ws[0], bias, dt), want + bias.double(), want.abs() + bias.double().abs(), 5, "dense")
