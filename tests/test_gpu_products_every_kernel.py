"""Every kernel of the products by expert, at sizes that the rule sends to it (``grouped_kernels``, asserted without a GPU): few rows of 16 and of
32, tiles of 128 and of 256, each of rows of whole pieces and of rows that begin at 4 bytes, and tiles at any address.

Against sums in 64 bits; what is not finite stays with its rows, columns and expert; offsets that are no bounds.  Tolerances as in
test_gpu_grouped_matmul.py and test_gpu_int8_matmul.py.
"""

import pytest
import torch

import grouped_kernels as rule
from group_helpers import assert_near, offsets_of, outer_products, products

# groups of one tile and of several, whole and ending inside a tile, of one row and of none; rows ahead of the first and behind the last
MANY = ([1100, 3, 0, 700, 257, 1, 1500, 520], 5, 10)
FEW = ([20, 0, 14, 3], 2, 1)
MIDDLE = ([300, 250, 512, 190, 0, 130, 97, 60, 1, 34, 400, 225], 0, 0)

# kernel, groups, terms of a sum, columns, bytes by which the operands begin behind an aligned address
ROWS = [("few1", FEW, 200, 264, 0), ("few1", FEW, 201, 263, 0), ("few2", MIDDLE, 72, 131, 0), ("few2", MIDDLE, 520, 136, 2),
        ("any", MANY, 331, 1025, 0), ("any", MANY, 2049, 1025, 0), ("any", MANY, 57, 1027, 0), ("any", MANY, 330, 1031, 0),
        ("any", MANY, 328, 1032, 2), ("any", MANY, 64, 4104, 6),
        ("small", MANY, 328, 1032, 0), ("small", MANY, 64, 1024, 0), ("small_cut", MANY, 330, 1030, 0), ("small_cut", MANY, 58, 1032, 0),
        ("small_cut", MANY, 328, 1032, 4), ("large", MANY, 328, 4104, 0), ("large", MANY, 56, 4096, 0),
        ("large_cut", MANY, 330, 4102, 0), ("large_cut", MANY, 62, 4104, 0), ("large_cut", MANY, 328, 4104, 12)]
# (the gradient of the rows: other times per step, weights that lie along their terms)
ROWS_GRADIENT = [c for c in ROWS if c[0] != "few2" and c[2:4] != (330, 1031)] + [
    ("few2", MIDDLE, 72, 136, 0), ("few2", MIDDLE, 515, 131, 0), ("any", MANY, 331, 1032, 0)]
# kernel, groups, columns of x, columns of d
WEIGHTS = [("any", MANY, 331, 1025, 0), ("any", MANY, 9, 70, 0), ("any", MANY, 328, 1032, 2), ("small", MANY, 328, 1032, 0),
           ("small_cut", MANY, 330, 1030, 0), ("small_cut", MANY, 328, 1032, 4), ("large", MANY, 1024, 2048, 0), ("large", MANY, 1032, 2056, 0),
           ("large_cut", MANY, 1026, 2050, 0), ("large_cut", MANY, 1024, 2048, 8)]
INT8 = [("few1", FEW, 200, 264, 0), ("few2", MIDDLE, 77, 131, 0), ("any", MANY, 331, 1025, 0), ("any", MANY, 2050, 1027, 0), ("any", MANY, 64, 1032, 1),
        ("small", MANY, 656, 1032, 0), ("small_cut", MANY, 332, 1030, 0), ("small_cut", MANY, 656, 1032, 4), ("large", MANY, 656, 4104, 0),
        ("large_cut", MANY, 332, 4102, 0)]


def _sizes(groups):
    counts, ahead, behind = groups
    return ahead + sum(counts) + behind, len(counts)


@pytest.mark.parametrize("cases,of", [(ROWS, rule.forward), (ROWS_GRADIENT, lambda S, E, K, N, m: rule.rows_gradient(S, E, N, K, m)),
                                      (WEIGHTS, rule.weights_gradient), (INT8, rule.int8)], ids=["forward", "rows", "weights", "int8"])
def test_the_rule_sends_the_sizes_there(cases, of):
    for kernel, groups, K, N, moved in cases:
        assert of(*_sizes(groups), K, N, moved) == kernel, (kernel, K, N, moved)
    want = {"any", "small", "small_cut", "large", "large_cut"} | (set() if cases is WEIGHTS else {"few1", "few2"})
    assert {c[0] for c in cases} == want


def _moved(t, nbytes):
    """A copy that begins nbytes behind an aligned address."""
    n = nbytes // t.element_size()
    buf = torch.empty(t.numel() + n, dtype=t.dtype, device=t.device)
    assert buf.data_ptr() % 256 == 0
    out = buf[n:].view(t.shape)
    out.copy_(t)
    return out


def _case(groups, K, N, moved, dtype, seed):
    counts, ahead, _ = groups
    S, E = _sizes(groups)
    g = torch.Generator(device="cuda").manual_seed(seed + K + N)
    r = lambda *s: _moved(torch.randn(s, generator=g, device="cuda").to(getattr(torch, dtype)), moved)
    return r, S, E, offsets_of(counts, ahead)


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,groups,K,N,moved", ROWS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_forward(kernel, groups, K, N, moved, dtype):
    from nkilib.core.moe.grouped_matmul import grouped_matmul

    r, S, E, o = _case(groups, K, N, moved, dtype, 1)
    x, w, od = r(S, K), r(E, K, N), torch.from_numpy(o).cuda()
    want, mag = products(x, w, o)
    got = grouped_matmul(x, w, od)
    assert_near(got, want, mag, K)
    assert torch.equal(got, grouped_matmul(x, w, od))


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,groups,K,N,moved", ROWS_GRADIENT)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_rows_gradient(kernel, groups, K, N, moved, dtype):
    from nkilib.core.moe.grouped_matmul import grouped_matmul_bwd

    r, S, E, o = _case(groups, K, N, moved, dtype, 2)
    d, w = r(S, K), r(E, N, K)
    want, mag = products(d, w.transpose(1, 2).contiguous(), o)
    assert_near(grouped_matmul_bwd(d, None, w, torch.from_numpy(o).cuda(), need_weight=False)[0], want, mag, K)


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,groups,K,N,moved", WEIGHTS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_weights_gradient(kernel, groups, K, N, moved, dtype):
    from nkilib.core.moe.grouped_matmul import grouped_matmul_bwd

    r, S, E, o = _case(groups, K, N, moved, dtype, 3)
    x, d, w = r(S, K), r(S, N), r(E, K, N)
    want, mag = outer_products(x, d, o)
    for wdt in (x.dtype, torch.float32):
        _, dw = grouped_matmul_bwd(d, x, w, torch.from_numpy(o).cuda(), weight_grad_dtype=wdt, need_x=False)
        assert_near(dw, want, mag, max(groups[0]), str(wdt))


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,groups,K,N,moved", INT8)
@pytest.mark.parametrize("out", ["bfloat16", "float16", "float32"])
def test_int8(kernel, groups, K, N, moved, out):
    from group_helpers import groups as ranges
    from nkilib.core.int8_matmul import grouped_int8_matmul

    counts, ahead, behind = groups
    (S, E), o = _sizes(groups), offsets_of(counts, ahead)
    g = torch.Generator(device="cuda").manual_seed(K + N)
    c = lambda *s: _moved(torch.randint(-128, 128, s, generator=g, device="cuda", dtype=torch.int8), moved)
    f = lambda *s: torch.rand(s, generator=g, device="cuda") * 0.02 + 0.001
    x, w, xs, ws = c(S, K), c(E, N, K), f(S), f(E, N)
    want = torch.zeros((S, N), dtype=torch.float64, device="cuda")
    for e, a, b in ranges(o, S):
        want[a:b] = (x[a:b].double() @ w[e].double().t().contiguous()) * xs[a:b, None].double() * ws[e].double()
    got = grouped_int8_matmul(x, xs, w, ws, torch.from_numpy(o).cuda(), out_dtype=getattr(torch, out))
    assert_near(got, want, want.abs(), 4)


def _bad_rows(o, S):
    """Rows that are to hold what is not finite: those of none, all of an expert between two others, and single ones of the other experts: the
    first, the last, ones at and beside the end of a tile.  Returns (rows of none, rows of the expert, the expert, single rows)."""
    lengths = [int(o[e + 1] - o[e]) for e in range(len(o) - 1)]
    expert = next(e for e in range(1, len(lengths) - 1) if lengths[e] > 1 and lengths[e - 1] + lengths[e + 1] > 0)
    single = []
    for e, n in enumerate(lengths):
        if e != expert:
            single += [int(o[e]) + i for i in (0, 17, 127, 128, 255, 257, n - 1) if 0 <= i < n and n > 4]
    none = [*range(int(o[0])), *range(int(o[-1]), S)]
    return none, [*range(int(o[expert]), int(o[expert + 1]))], expert, sorted(set(single))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("direction,kernel,groups,K,N,moved",
                         [("forward", *c) for c in ROWS] + [("rows", *c) for c in ROWS_GRADIENT])
def test_rows_that_are_not_finite_keep_to_themselves(direction, kernel, groups, K, N, moved, bad):
    """A row's end lies beside the next row's first terms, a matrix' end beside the next one's: neither has a part in its sums."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    r, S, E, o = _case(groups, K, N, moved, "bfloat16", 4)
    od = torch.from_numpy(o).cuda()
    x, w = r(S, K), (r(E, K, N) if direction == "forward" else r(E, N, K))
    want, mag = products(x, w if direction == "forward" else w.transpose(1, 2).contiguous(), o)
    none, of_expert, expert, single = _bad_rows(o, S)
    x[none + of_expert + single] = bad
    w[expert] = bad
    got = grouped_matmul(x, w, od) if direction == "forward" else grouped_matmul_bwd(x, None, w, od, need_weight=False)[0]
    clean = torch.ones(S, dtype=torch.bool, device="cuda")
    clean[none + of_expert + single] = False
    assert_near(got[clean], want[clean], mag[clean], K)
    assert not got[none].any()
    assert not torch.isfinite(got[of_expert + single]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("kernel,groups,K,N,moved", WEIGHTS)
def test_columns_that_are_not_finite_keep_to_themselves(kernel, groups, K, N, moved, bad):
    """The gradient of the weights: rows of another expert and of none, and single columns of either side, the first ones among them, which
    lie behind the end of the row before."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul_bwd

    r, S, E, o = _case(groups, K, N, moved, "bfloat16", 5)
    x, d, w = r(S, K), r(S, N), r(E, K, N)
    want, mag = outer_products(x, d, o)
    none, of_expert, expert, _ = _bad_rows(o, S)
    ks, ns = sorted({0, min(K - 1, 128), K - 2}), sorted({0, min(N - 1, 65), N - 1})
    x[none + of_expert], d[none + of_expert] = bad, bad
    x[:, ks] = bad
    d[:, ns] = bad
    _, dw = grouped_matmul_bwd(d, x, w, torch.from_numpy(o).cuda(), need_x=False)
    k = [i for i in range(K) if i not in ks]
    n = [i for i in range(N) if i not in ns]
    for e, rows in enumerate(groups[0]):
        if e == expert:
            assert not torch.isfinite(dw[e]).any()
        elif rows == 0:
            assert not dw[e].any()
        else:
            assert_near(dw[e][k][:, n], want[e][k][:, n], mag[e][k][:, n], rows, f"expert {e}")
            assert not torch.isfinite(dw[e][ks]).any() and not torch.isfinite(dw[e][:, ns]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[700, 4000, 900, -5, 2**31 - 1, 3000, 4096, 100, 50], [-9, 0, 513, 300, 2000, 1999, 4000, 4090, 4095],
                                     [-(2**31), 5000, 0, 0, 0, 0, 0, 0, 0], [4096] * 9, [0, 0, 0, 4096, 4095, 0, 0, 0, 9999]])
@pytest.mark.parametrize("K,N", [(331, 1025), (328, 1032), (330, 1030), (328, 4104), (330, 4102)])
def test_offsets_that_are_no_bounds(offsets, K, N):
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    r, S, E, _ = _case(MANY, K, N, 0, "bfloat16", 6)
    x, w, d = r(S, K), r(E, K, N), r(S, N)
    od = torch.tensor(offsets, dtype=torch.int64).to(torch.int32).cuda()
    want, mag = products(x, w, offsets)
    assert_near(grouped_matmul(x, w, od), want, mag, K)
    dx, dw = grouped_matmul_bwd(d, x, w, od)
    want, mag = products(d, w.transpose(1, 2).contiguous(), offsets)
    assert_near(dx, want, mag, N, "d_x")
    want, mag = outer_products(x, d, offsets)
    assert_near(dw, want, mag, S, "d_w")


# both gradients in one launch: large tiles of either, of the rows' gradient fewer than there are workgroups and more
BOTH = [(4096, 512), (8192, 256), (8200, 520)]


def test_the_rule_sends_both_gradients_to_large_tiles():
    S, E = _sizes(MIDDLE)
    for K, N in BOTH:
        assert rule.rows_gradient(S, E, K, N) == rule.weights_gradient(S, E, K, N) == "large"
    tiles = [sum(-(-n // 256) for n in MIDDLE[0]) * -(-K // 256) for K, _ in BOTH]
    assert tiles[0] < 256 < tiles[1]


@pytest.mark.gpu
@pytest.mark.parametrize("K,N", BOTH)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_both_gradients_in_one_launch(K, N, dtype):
    from nkilib.core.moe.grouped_matmul import grouped_matmul_bwd

    r, S, E, o = _case(MIDDLE, K, N, 0, dtype, 7)
    x, d, w, od = r(S, K), r(S, N), r(E, K, N), torch.from_numpy(o).cuda()
    for wdt in (x.dtype, torch.float32):
        dx, dw = grouped_matmul_bwd(d, x, w, od, weight_grad_dtype=wdt)
        want, mag = products(d, w.transpose(1, 2).contiguous(), o)
        assert_near(dx, want, mag, N, "d_x")
        want, mag = outer_products(x, d, o)
        assert_near(dw, want, mag, max(MIDDLE[0]), "d_w")
        assert torch.equal(dx, grouped_matmul_bwd(d, None, w, od, need_weight=False)[0])
        assert torch.equal(dw, grouped_matmul_bwd(d, x, w, od, weight_grad_dtype=wdt, need_x=False)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("S,K,N", [(1, 7168, 4096), (64, 2048, 256), (1000, 14336, 320), (7, 131071, 24)])
def test_int8_long_rows_to_fp16(S, K, N):
    """Codes at random, scales of at most 0.021: the standard deviation of a result is below 74^2 * K^0.5 * 0.021^2, 875 for the longest rows, so that
    all of them are inside of what 16 bits hold."""
    from nkilib.core.int8_matmul import int8_matmul

    g = torch.Generator(device="cuda").manual_seed(S + K)
    c = lambda *s: torch.randint(-128, 128, s, generator=g, device="cuda", dtype=torch.int8)
    f = lambda *s: torch.rand(s, generator=g, device="cuda") * 0.02 + 0.001
    x, w, xs, ws, bias = c(S, K), c(N, K), f(S), f(N), (torch.randn(N, generator=g, device="cuda") * 10).half()
    want = (x.double() @ w.double().t().contiguous()) * xs.double()[:, None] * ws.double()
    assert want.abs().max() < 60000
    assert_near(int8_matmul(x, xs, w, ws, out_dtype=torch.float16), want, want.abs(), 4)
    assert_near(int8_matmul(x, xs, w, ws, bias=bias, out_dtype=torch.float16), want + bias.double(), want.abs() + bias.double().abs(), 5)
