"""Products by expert and their gradients against sums in 64 bits.

Tolerance (``group_helpers.assert_near``): products of two 16-bit values are exact in fp32, a sum of n of them is off by at most n
roundings of 2^-24 of the terms' magnitudes, and the result is rounded once.
"""

import numpy as np
import pytest
import torch

from group_helpers import assert_near, offsets_of, outer_products, products

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16"]
# rows of every expert, rows ahead of the first and behind the last, K, N: one row; experts without rows; rows, terms and columns of
# no multiple of a tile or of a vector; rows of fewer than 16 bytes; more than one tile each way; more experts than rows
CASES = {
    "one": ([1], 0, 0, 64, 64),
    "one_of_many": ([0] * 100 + [1] + [0] * 27, 0, 0, 256, 192),
    "tiny": ([3, 0, 2], 1, 2, 3, 5),
    "one_column": ([4, 7], 0, 0, 9, 1),
    "one_term": ([5, 130], 0, 3, 1, 24),
    "odd": ([0, 33, 1, 0, 200, 77], 3, 9, 131, 515),
    "odd_terms": ([64, 129], 0, 0, 1030, 136),
    "ragged": ([16, 17, 0, 5, 128, 127, 1], 0, 40, 200, 264),
    "wide": ([300, 0, 260, 129], 7, 0, 448, 776),
    "long": ([513, 1], 0, 0, 2056, 320),
    "no_rows": ([0, 0, 0], 5, 6, 128, 128),
    "large_tiles": ([512, 256, 255, 257], 0, 0, 512, 512),
    "most_experts": ([1, 0, 2] * 341 + [1], 0, 0, 72, 40),
}


def _case(name, dtype, seed=0):
    counts, ahead, behind, K, N = CASES[name]
    g = torch.Generator(device="cuda").manual_seed(seed + len(name))
    dt = getattr(torch, dtype)
    S = ahead + sum(counts) + behind
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
    o = offsets_of(counts, ahead)
    return r(S, K), (r(len(counts), K, N).float() * K**-0.5).to(dt), r(S, N), o, torch.from_numpy(o).cuda()


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward(name, dtype):
    from nkilib.core.moe.grouped_matmul import grouped_matmul

    x, w, _, o, od = _case(name, dtype)
    want, mag = products(x, w, o)
    got = grouped_matmul(x, w, od)
    assert got.dtype == x.dtype
    assert_near(got, want, mag, x.shape[1], f"{name} {dtype}")
    assert torch.equal(got, grouped_matmul(x, w, od))  # the same bits each time


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(name, dtype):
    from nkilib.core.moe.grouped_matmul import grouped_matmul_bwd

    x, w, d, o, od = _case(name, dtype, 1)
    counts = CASES[name][0]
    dx, dw = grouped_matmul_bwd(d, x, w, od)
    want, mag = products(d, w.transpose(1, 2).contiguous(), o)
    assert_near(dx, want, mag, w.shape[2], f"d_x {name} {dtype}")
    want, mag = outer_products(x, d, o)
    assert_near(dw, want, mag, max(counts), f"d_w {name} {dtype}")
    dw32 = grouped_matmul_bwd(d, x, w, od, weight_grad_dtype=torch.float32, need_x=False)
    assert dw32[0] is None and dw32[1].dtype == torch.float32
    assert_near(dw32[1], want, mag, max(counts), f"d_w fp32 {name} {dtype}")
    only = grouped_matmul_bwd(d, None, w, od, need_weight=False)
    assert only[1] is None and torch.equal(only[0], dx)


def test_gradient_against_differences():
    """The loss sum(out * d) changes with x and w as the gradients say (values of few bits: the sums are exact)."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randint(-3, 4, s, generator=g, device="cuda").half()
    o = torch.tensor([0, 3, 3, 8], dtype=torch.int32, device="cuda")
    x, w, d = r(8, 16), r(3, 16, 24), r(8, 24)
    dx, dw = grouped_matmul_bwd(d, x, w, o)
    loss = lambda x, w: (grouped_matmul(x, w, o).double() * d.double()).sum().item()
    base = loss(x, w)
    for s, k in ((0, 0), (2, 15), (7, 3)):
        x1 = x.clone()
        x1[s, k] += 1
        assert loss(x1, w) - base == dx[s, k].item()
    for e, k, n in ((0, 0, 0), (0, 15, 23), (1, 2, 2), (2, 8, 16)):
        w1 = w.clone()
        w1[e, k, n] += 1
        assert loss(x, w1) - base == dw[e, k, n].item()


@pytest.mark.parametrize("offsets", [[0, 100, 40, 90], [-5, 10, 2**31 - 1, 20], [50, 30, 20, 10], [-(2**31), 0, 0, 0], [200, 300, 300, 300],
                                     [7, 7, 7, 7], [120, 0, 0, 120]])
@pytest.mark.parametrize("K,N", [(128, 128), (33, 77)])
def test_offsets_that_are_no_bounds(offsets, K, N):
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    x, w, d = r(120, K), r(3, K, N), r(120, N)
    od = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    want, mag = products(x, w, offsets)
    assert_near(grouped_matmul(x, w, od), want, mag, K)
    dx, dw = grouped_matmul_bwd(d, x, w, od)
    want, mag = products(d, w.transpose(1, 2).contiguous(), offsets)
    assert_near(dx, want, mag, N)
    want, mag = outer_products(x, d, offsets)
    assert_near(dw, want, mag, 120)


@pytest.mark.parametrize("K,N", [(64, 256), (200, 264), (40, 72), (35, 39)])
def test_what_is_not_finite_stays_with_its_group(K, N):
    """Rows of another expert, of none, and terms and columns behind a row's end (the next row's values) have no part in a result."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    o = offsets_of([20, 30, 14], 4)
    x, w, d = r(80, K), r(3, K, N), r(80, N)
    for bad in (float("nan"), float("inf")):
        x1, w1, d1 = x.clone(), w.clone(), d.clone()
        x1[:4], x1[68:], x1[24:54] = bad, bad, bad  # (rows of none, rows of expert 1)
        d1[:4], d1[68:], d1[24:54] = bad, bad, bad
        w1[1] = bad
        x1[10, 3] = bad  # one row of expert 0
        od = torch.from_numpy(o).cuda()
        out = grouped_matmul(x1, w1, od)
        want, mag = products(x, w, o)
        keep = torch.ones(80, dtype=torch.bool, device="cuda")
        keep[24:54], keep[10] = False, False
        assert_near(out[keep], want[keep], mag[keep], K)
        assert not out[:4].any() and not out[68:].any() and not torch.isfinite(out[10]).any() and not torch.isfinite(out[24:54]).any()
        dx, dw = grouped_matmul_bwd(d1, x1, w1, od)
        want, mag = products(d, w.transpose(1, 2).contiguous(), o)
        keep[10] = True
        assert_near(dx[keep], want[keep], mag[keep], N)
        want, mag = outer_products(x, d, o)
        assert_near(dw[2], want[2], mag[2], 30)
        rest = [k for k in range(K) if k != 3]
        assert_near(dw[0][rest], want[0][rest], mag[0][rest], 30)
        assert not torch.isfinite(dw[1]).any() and not torch.isfinite(dw[0, 3]).any()


@pytest.mark.parametrize("K,N", [(128, 256), (136, 72)])
def test_views_addresses_and_strides(K, N):
    """Tensors that begin at any element, and ones that are not contiguous (copied)."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda n: torch.randn(n, generator=g, device="cuda").half()
    o = offsets_of([40, 0, 31])
    od = torch.from_numpy(o).cuda()
    for shift in (1, 3, 8):
        x, w, d = r(71 * K + 8)[shift:][: 71 * K].view(71, K), r(3 * K * N + 8)[shift:][: 3 * K * N].view(3, K, N), \
            r(71 * N + 8)[shift:][: 71 * N].view(71, N)
        want, mag = products(x, w, o)
        assert_near(grouped_matmul(x, w, od), want, mag, K, f"shift {shift}")
        dx, dw = grouped_matmul_bwd(d, x, w, od)
        want, mag = products(d, w.transpose(1, 2).contiguous(), o)
        assert_near(dx, want, mag, N, f"shift {shift}")
        want, mag = outer_products(x, d, o)
        assert_near(dw, want, mag, 40, f"shift {shift}")
    x, w = r(K * 71).view(K, 71).t(), r(3 * K * N).view(3, N, K).transpose(1, 2)
    want, mag = products(x, w, o)
    assert_near(grouped_matmul(x, w, od), want, mag, K, "strided")


def test_no_rows_no_terms_no_columns():
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    z = lambda *s: torch.ones(s, device="cuda", dtype=torch.bfloat16)
    o = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert grouped_matmul(z(0, 64), z(2, 64, 32), o).shape == (0, 32)
    dx, dw = grouped_matmul_bwd(z(0, 32), z(0, 64), z(2, 64, 32), o)
    assert dx.shape == (0, 64) and dw.shape == (2, 64, 32) and not dw.any()
    assert not grouped_matmul(z(4, 0), z(2, 0, 32), o).any() and grouped_matmul(z(4, 8), z(2, 8, 0), o).shape == (4, 0)
    dx, dw = grouped_matmul_bwd(z(4, 0), z(4, 8), z(2, 8, 0), o)
    assert not dx.any() and dw.shape == (2, 8, 0)


def test_a_long_group_and_its_neighbours():
    """More tiles than workgroups, groups of very different lengths."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    counts = [9000, 3, 0, 700, 1, 2047]
    o = offsets_of(counts, 2)
    S = 2 + sum(counts) + 5
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    x, w, d = r(S, 320), r(len(counts), 320, 1536), r(S, 1536)
    od = torch.from_numpy(o).cuda()
    want, mag = products(x, w, o)
    assert_near(grouped_matmul(x, w, od), want, mag, 320)
    dx, dw = grouped_matmul_bwd(d, x, w, od)
    want, mag = products(d, w.transpose(1, 2).contiguous(), o)
    assert_near(dx, want, mag, 1536)
    want, mag = outer_products(x, d, o)
    assert_near(dw, want, mag, 9000)


@pytest.mark.parametrize("T,E,k,B", [(1, 4, 1, 1), (70, 8, 3, 16), (3000, 60, 4, 32), (500, 256, 8, 1), (40, 1, 1, 128)])
def test_bounds_from_the_block_table(T, E, k, B):
    from nkilib.core.moe.grouped_matmul import expert_row_offsets
    from train_helpers import table

    _, b2e, N = table(np.random.default_rng(T), T, E, k, B)
    want = [B * int((b2e < e).sum()) for e in range(E + 1)]
    assert expert_row_offsets(torch.from_numpy(b2e.astype(np.int32)).cuda(), B, E).tolist() == want
    none = torch.tensor([0, 0, 2, E + 5, -1], dtype=torch.int32, device="cuda")  # (blocks of no expert stand behind)
    got = expert_row_offsets(none, 4, 3).tolist()
    assert got == [0, 8, 8, 12]
    assert expert_row_offsets(none[:0], 4, 3).tolist() == [0, 0, 0, 0]


def test_in_a_graph_on_a_stream():
    """Recorded and replayed with other offsets, other rows; every replay is the eager result."""
    from nkilib.core.moe.grouped_matmul import expert_row_offsets, grouped_matmul, grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(7)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    x, w, d = r(96, 128), r(4, 128, 264), r(96, 264)
    b2e = torch.tensor([0, 0, 1, 2, 3, 3], dtype=torch.int32, device="cuda")

    def step():
        o = expert_row_offsets(b2e, 16, 4)
        return (grouped_matmul(x, w, o), *grouped_matmul_bwd(d, x, w, o))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i, blocks in enumerate(([0, 0, 1, 2, 3, 3], [3] * 6, [0, 1, 1, 1, 1, 2], [2, 2, 9, 9, 9, 9])):
        b2e.copy_(torch.tensor(blocks, dtype=torch.int32))
        x.copy_(r(96, 128))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_refusals():
    from nkilib.core.moe.grouped_matmul import expert_row_offsets, grouped_matmul, grouped_matmul_bwd

    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, device="cuda", dtype=dt)
    x, w, o, d = z(4, 8), z(2, 8, 6), z(3, dt=torch.int32), z(4, 6)
    bad = [
        lambda: grouped_matmul(x.float(), w.float(), o), lambda: grouped_matmul(x, w.half(), o), lambda: grouped_matmul(x, z(2, 6, 8), o),
        lambda: grouped_matmul(x, w, o.long()), lambda: grouped_matmul(x, w, o[:2]), lambda: grouped_matmul(x[0], w, o),
        lambda: grouped_matmul(x, w[0], o), lambda: grouped_matmul(x, z(1025, 8, 1), z(1026, dt=torch.int32)),
        lambda: grouped_matmul(x, z(0, 8, 6), z(1, dt=torch.int32)), lambda: grouped_matmul(z(1, 2**20 + 1), z(1, 2**20 + 1, 1), o[:2]),
        lambda: grouped_matmul_bwd(z(4, 7), x, w, o), lambda: grouped_matmul_bwd(d, z(5, 8), w, o), lambda: grouped_matmul_bwd(d, None, w, o),
        lambda: grouped_matmul_bwd(d, x.half(), w, o), lambda: grouped_matmul_bwd(d, x, w, o, weight_grad_dtype=torch.float16),
        lambda: grouped_matmul_bwd(d, x, w, o, need_x=False, need_weight=False),
        lambda: expert_row_offsets(o.long(), 4, 2), lambda: expert_row_offsets(o, 0, 2), lambda: expert_row_offsets(o, 4, 0),
        lambda: expert_row_offsets(o, 4, 1025), lambda: expert_row_offsets(o, 2**30, 2),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was not refused")


# groups whose last tile of 256 rows holds every number of 32 rows, and tiles of 128 likewise; none at all; one of several tiles
EVERY_TILE = [300, 250, 512, 190, 0, 130, 97, 60, 1, 34, 400, 225]


@pytest.mark.parametrize("N", [136, 1032, 8200, 131, 1027, 8195, 1030, 8198])
@pytest.mark.parametrize("K", [72, 256, 520, 77, 515, 58, 74, 518])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_kind_of_tile(K, N, dtype):
    """The kernel goes by the number of tiles: few columns, some and many; by whether rows are aligned (16 bytes, 4 or 2); one step and
    several, whole and cut, also inside 16 bytes."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(K + N)
    dt, S, E = getattr(torch, dtype), sum(EVERY_TILE), len(EVERY_TILE)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
    x, w, o = r(S, K), r(E, K, N), offsets_of(EVERY_TILE)
    od = torch.from_numpy(o).cuda()
    want, mag = products(x, w, o)
    assert_near(grouped_matmul(x, w, od), want, mag, K, "forward")
    # the gradient of the rows with the roles of the sizes changed, so that its columns are few, some and many as well
    wt, d = r(E, N, K), r(S, K)
    want, mag = products(d, wt.transpose(1, 2).contiguous(), o)
    assert_near(grouped_matmul_bwd(d, None, wt, od, need_weight=False)[0], want, mag, K, "d_x")


@pytest.mark.parametrize("K,N", [(136, 264), (1032, 1032), (2056, 1992), (131, 515), (1027, 1029), (2050, 1999), (1032, 1029), (1030, 1030),
                                 (2054, 1998), (1030, 1032)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_kind_of_tile_of_the_weights_gradient(K, N, dtype):
    from nkilib.core.moe.grouped_matmul import grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(K + N)
    dt, S, E = getattr(torch, dtype), sum(EVERY_TILE), len(EVERY_TILE)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
    x, d, w, o = r(S, K), r(S, N), r(E, K, N), offsets_of(EVERY_TILE)
    want, mag = outer_products(x, d, o)
    for wdt in (dt, torch.float32):
        _, dw = grouped_matmul_bwd(d, x, w, torch.from_numpy(o).cuda(), weight_grad_dtype=wdt, need_x=False)
        assert_near(dw, want, mag, max(EVERY_TILE), str(wdt))


@pytest.mark.parametrize("K,N", [(4104, 520), (4096, 264)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_both_gradients_in_one_launch(K, N, dtype):
    """Many large tiles of either: the same bits as one after the other."""
    from nkilib.core.moe.grouped_matmul import grouped_matmul_bwd

    g = torch.Generator(device="cuda").manual_seed(K + N)
    dt, S, E = getattr(torch, dtype), sum(EVERY_TILE), len(EVERY_TILE)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
    x, d, w, o = r(S, K), r(S, N), r(E, K, N), offsets_of(EVERY_TILE)
    od = torch.from_numpy(o).cuda()
    for wdt in (dt, torch.float32):
        dx, dw = grouped_matmul_bwd(d, x, w, od, weight_grad_dtype=wdt)
        want, mag = products(d, w.transpose(1, 2).contiguous(), o)
        assert_near(dx, want, mag, N, "d_x")
        want, mag = outer_products(x, d, o)
        assert_near(dw, want, mag, max(EVERY_TILE), "d_w")
        assert torch.equal(dx, grouped_matmul_bwd(d, None, w, od, need_weight=False)[0])
        assert torch.equal(dw, grouped_matmul_bwd(d, x, w, od, weight_grad_dtype=wdt, need_x=False)[1])
