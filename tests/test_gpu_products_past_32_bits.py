"""Tensors of more than 4 GB: rows, weights and columns behind 2^31 elements or 2^32 bytes, checked where they end.

Tolerances as in test_gpu_grouped_matmul.py, test_gpu_int8_matmul.py and test_gpu_rmsnorm_quant_rows.py.
"""

import pytest
import torch

from group_helpers import assert_near

pytestmark = pytest.mark.gpu


def _fill(t, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat, part = t.view(-1), 1 << 28
    for i in range(0, flat.numel(), part):
        n = min(part, flat.numel() - i)
        flat[i : i + n] = torch.randn(n, generator=g, device="cuda").mul_(scale)
    return t


def test_rows():
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    S, K, N = 2_200_000, 1024, 72
    x = _fill(torch.empty((S, K), dtype=torch.bfloat16, device="cuda"), 1)
    w = _fill(torch.empty((3, K, N), dtype=torch.bfloat16, device="cuda"), 2, K**-0.5)
    o = torch.tensor([0, 1_000_000, 2_199_000, S - 10], dtype=torch.int32, device="cuda")
    out = grouped_matmul(x, w, o)
    for a, b, e in ((0, 300, 0), (999_800, 1_000_000, 0), (1_000_000, 1_000_100, 1), (2_198_900, 2_199_000, 1), (2_199_000, S - 10, 2)):
        xe, we = x[a:b].double(), w[e].double()
        assert_near(out[a:b], xe @ we, xe.abs() @ we.abs(), K, f"rows {a}")
    assert not out[S - 10 :].any()
    # the gradients: rows of the last group alone carry one, so that the weights' is a sum of few terms
    d = torch.zeros((S, N), dtype=torch.bfloat16, device="cuda")
    d[2_199_000:] = _fill(torch.empty((S - 2_199_000, N), dtype=torch.bfloat16, device="cuda"), 3)
    dx, dw = grouped_matmul_bwd(d, x, w, o)
    de, wt = d[2_199_000 : S - 10].double(), w[2].double().t().contiguous()
    assert_near(dx[2_199_000 : S - 10], de @ wt, de.abs() @ wt.abs(), N, "d_x")
    assert not dx[:2_199_000].any() and not dx[S - 10 :].any()
    xt = x[2_199_000 : S - 10].double().t().contiguous()
    assert_near(dw[2], xt @ de, xt.abs() @ de.abs(), 1000, "d_w")
    assert not dw[:2].any()


def test_weights():
    from nkilib.core.int8_matmul import grouped_int8_matmul
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    E, K, N, S = 600, 2048, 2048, 40
    w = _fill(torch.empty((E, K, N), dtype=torch.bfloat16, device="cuda"), 4, K**-0.5)
    x = _fill(torch.empty((S, K), dtype=torch.bfloat16, device="cuda"), 5)
    bounds = [0] * 550 + [10] * 49 + [10, S]  # rows of experts 549 and 599
    o = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    out = grouped_matmul(x, w, o)
    dx, dw = grouped_matmul_bwd(x, x, w, o)
    for a, b, e in ((0, 10, 549), (10, S, 599)):
        xe, we = x[a:b].double(), w[e].double()
        assert_near(out[a:b], xe @ we, xe.abs() @ we.abs(), K, f"expert {e}")
        wt = we.t().contiguous()
        assert_near(dx[a:b], xe @ wt, xe.abs() @ wt.abs(), N, f"d_x of {e}")
        assert_near(dw[e], xe.t().contiguous() @ xe, xe.abs().t().contiguous() @ xe.abs(), 30, f"d_w of {e}")
    assert not dw[:549].any() and not dw[550:599].any()
    del dw, w
    w8 = torch.randint(-128, 128, (E, 4096, K), dtype=torch.int8, device="cuda")
    x8 = torch.randint(-128, 128, (S, K), dtype=torch.int8, device="cuda")
    xs, ws = torch.rand(S, device="cuda"), torch.rand((E, 4096), device="cuda")
    out = grouped_int8_matmul(x8, xs, w8, ws, o, out_dtype=torch.float32)
    for a, b, e in ((0, 10, 549), (10, S, 599)):
        want = (x8[a:b].double() @ w8[e].double().t().contiguous()) * xs[a:b, None].double() * ws[e].double()
        assert_near(out[a:b], want, want.abs(), 4, f"int8 expert {e}")


def test_norm():
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

    rows, H = 300_000, 8192
    x = _fill(torch.empty((rows, H), dtype=torch.bfloat16, device="cuda"), 6)
    codes, scales, stream = rmsnorm_quant_rows(x, None, residual=x)
    few = rmsnorm_quant_rows(x[-50:].clone(), None, residual=x[-50:].clone())
    assert torch.equal(codes[-50:], few[0]) and torch.equal(scales[-50:], few[1]) and torch.equal(stream[-50:], few[2])
    values = dequantize_rows(codes, scales)
    assert torch.equal(values[-50:], dequantize_rows(*few[:2]))
    dx, _ = rmsnorm_quant_rows_bwd(values, stream, None)
    assert torch.equal(dx[-50:], rmsnorm_quant_rows_bwd(values[-50:].clone(), few[2], None)[0])
