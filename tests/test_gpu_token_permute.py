"""permute / combine and their gradients against the oracle in 64 bits (tolerances: ``train_helpers.bound``; a sum over k slots
takes k multiply-adds, a dot product over H a tree and a chain of fewer than H / 64 + 16)."""

import numpy as np
import pytest

from oracle import train as ot
from train_helpers import assert_within, bound, table, tensor, values

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16", "float32"]
# T, H, E, k, B: one token, one slot per block, rows of odd length (2- and 4-byte pieces, none at all), more than eight slots per
# token, more than a group of tokens per workgroup, an expert without tokens
SHAPES = [(1, 64, 4, 1, 1), (1, 7168, 256, 8, 1), (5, 3, 4, 2, 4), (33, 130, 8, 3, 16), (300, 1029, 60, 4, 32), (129, 2056, 16, 2, 128),
          (70, 515, 24, 17, 8), (40, 96, 64, 64, 1), (700, 256, 3, 3, 512), (32, 1500, 64, 64, 1), (600, 128, 3, 3, 1)]


def _case(shape, dtype, seed, skip_token=False):
    T, H, E, k, B = shape
    rng = np.random.default_rng(seed)
    tp2id, b2e, N = table(rng, T, E, k, B, skip_token)
    aff = tensor(rng.random((T + 1, E)), "bfloat16" if seed % 2 else "float32")
    y = tensor(rng.standard_normal((N * B, H)), dtype)
    return rng, tp2id, b2e, tensor(tp2id, "int32"), tensor(b2e, "int32"), aff, y


@pytest.mark.parametrize("T,E,k,B,top_k", [(1, 4, 1, 1, 1), (33, 8, 3, 16, 3), (3000, 60, 4, 32, 6), (40, 64, 64, 1, 64), (20, 8, 5, 4, 2)])
def test_token_slots(T, E, k, B, top_k):
    import torch
    from nkilib.core.moe.token_permute import build_token_slots

    tp2id, _, _ = table(np.random.default_rng(T), T, E, k, B)
    want = ot.token_slots(tp2id, T, top_k)
    got = build_token_slots(tensor(tp2id, "int32"), T, top_k).cpu().numpy()
    if top_k >= k:
        assert np.array_equal(got, want)
    else:  # a cut list: the true count, and top_k of the slots
        assert np.array_equal(got[:, 0], want[:, 0])
        with pytest.raises(AssertionError, match="more than top_k"):
            build_token_slots(tensor(tp2id, "int32"), T, top_k, check=True)
    # a table that begins anywhere (4-byte aligned only), ids far outside
    odd = torch.cat((torch.tensor([2**31 - 1, -(2**31), -1], dtype=torch.int32), torch.from_numpy(tp2id).int())).cuda()
    assert np.array_equal(build_token_slots(odd[3:], T, max(k, top_k)).cpu().numpy(), ot.token_slots(tp2id, T, max(k, top_k)))
    shifted = build_token_slots(odd, T, max(k, top_k)).cpu().numpy()
    assert np.array_equal(np.where(shifted[:, 1:] >= 0, shifted[:, 1:] - 3, -1), ot.token_slots(tp2id, T, max(k, top_k))[:, 1:])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_permute_and_gradient(shape, dtype):
    from nkilib.core.moe.token_permute import permute_tokens, permute_tokens_bwd

    T, H, E, k, B = shape
    rng, tp2id, b2e, tp, be, aff, y = _case(shape, dtype, T + H, skip_token=bool(T % 2))
    x = tensor(rng.standard_normal((T, H)), dtype)
    assert np.array_equal(values(permute_tokens(x, tp)), ot.permute(values(x), tp2id))
    want, mag = ot.combine(values(y), None, tp2id, b2e, B, T)
    assert_within(permute_tokens_bwd(y, tp, T, k), want, bound(want, mag, dtype, k + 1), f"{shape} {dtype}")


def test_permute_moves_any_bytes():
    import torch
    from nkilib.core.moe.token_permute import permute_tokens

    rng = np.random.default_rng(0)
    tp2id, _, _ = table(rng, 50, 8, 2, 16)
    for width in (1, 15, 16, 77, 1030, 1600, 4100, 8190, 8192, 20001):
        x = rng.integers(0, 256, (50, width), dtype=np.uint8)
        got = permute_tokens(torch.from_numpy(x).cuda(), tensor(tp2id, "int32"))
        assert np.array_equal(got.cpu().numpy(), ot.permute(x, tp2id)), width


@pytest.mark.parametrize("width,dtype", [(7168, "bfloat16"), (1030, "bfloat16"), (515, "float32"), (530, "bfloat16"), (100, "bfloat16"),
                                         (9001, "float32")])
def test_large_permutes(width, dtype):
    """Tables of 80 MB: tokens without slots, tokens with hundreds; rows longer than a round of a workgroup."""
    import torch
    from nkilib.core.moe.token_permute import permute_tokens

    rng = np.random.default_rng(width)
    es = 2 if dtype == "bfloat16" else 4
    S, T = (80 << 20) // (width * es), 300
    ids = rng.integers(-1, T + 2, S).astype(np.int32)
    ids[ids % 3 == 0] = -1
    ids[ids == 5] = T
    ids[rng.permutation(S)[:14]] = 5  # (14 slots; the others have hundreds, or none)
    x = tensor(rng.standard_normal((T, width)), dtype)
    tp = torch.from_numpy(ids).cuda()
    ok = (tp >= 0) & (tp < T)
    want = torch.where(ok[:, None], x[tp.long().clamp(0, T - 1)], torch.zeros((), dtype=x.dtype, device="cuda"))
    assert torch.equal(permute_tokens(x, tp), want)
    T = S // 4
    tp = torch.from_numpy(rng.permutation(np.repeat(rng.permutation(T), 4).astype(np.int32))).cuda()
    x = torch.randn((T, width), device="cuda").to(x.dtype)
    assert torch.equal(permute_tokens(x, tp), x[tp.long()])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine_and_gradient(shape, dtype):
    from nkilib.core.moe.token_permute import build_token_slots, combine_tokens, combine_tokens_bwd

    T, H, E, k, B = shape
    rng, tp2id, b2e, tp, be, aff, y = _case(shape, dtype, T + H + (dtype == "float16"), skip_token=bool(T % 2))
    a, yv = values(aff), values(y)
    want, mag = ot.combine(yv, a, tp2id, b2e, B, T)
    got = combine_tokens(y, aff, tp, be, B, T, k)
    assert_within(got, want, bound(want, mag, dtype, k + 1), f"{shape} {dtype}")
    slots = build_token_slots(tp, T, k)
    assert np.array_equal(values(combine_tokens(y, aff, tp, be, B, T, k, token_slots=slots)), values(got))  # the same bits
    d = tensor(rng.standard_normal((T, H)), dtype)
    want_y, want_a, mag_a = ot.combine_bwd(values(d), yv, a, tp2id, b2e, B)
    d_y, d_aff = combine_tokens_bwd(d, y, aff, tp, be, B, k, token_slots=slots)
    assert_within(d_y, want_y, bound(want_y, np.abs(want_y), dtype, 1), f"d_y {shape} {dtype}")
    assert str(d_aff.dtype) == "torch.float32"
    assert_within(d_aff, want_a, bound(want_a, mag_a, "float32", H / 64 + 16), f"d_aff {shape} {dtype}")


# many tokens: rows of a wave each up to 4096 bytes, of a workgroup each beyond; more than eight slots; no token in the last ones
@pytest.mark.parametrize("shape", [(3855, 65, 128, 3, 16), (2048, 3, 8, 2, 16), (2047, 1024, 16, 4, 32), (2100, 1025, 24, 9, 32),
                                   (2500, 2048, 16, 2, 64), (2048, 2049, 16, 2, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens_with_short_rows(shape, dtype):
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd

    T, H, E, k, B = shape
    rng, tp2id, b2e, tp, be, aff, y = _case(shape, dtype, T + H, skip_token=True)
    a, yv = values(aff), values(y)
    d = tensor(rng.standard_normal((T, H)), dtype)
    assert np.array_equal(values(permute_tokens(d, tp)), ot.permute(values(d), tp2id))
    want, mag = ot.combine(yv, a, tp2id, b2e, B, T)
    assert_within(combine_tokens(y, aff, tp, be, B, T, k), want, bound(want, mag, dtype, k + 1), f"{shape} {dtype}")
    want, mag = ot.combine(yv, None, tp2id, b2e, B, T)
    assert_within(permute_tokens_bwd(y, tp, T, k), want, bound(want, mag, dtype, k + 1), f"{shape} {dtype}")
    want_y, want_a, mag_a = ot.combine_bwd(values(d), yv, a, tp2id, b2e, B)
    d_y, d_aff = combine_tokens_bwd(d, y, aff, tp, be, B, k)
    assert_within(d_y, want_y, bound(want_y, np.abs(want_y), dtype, 1), f"d_y {shape} {dtype}")
    assert_within(d_aff, want_a, bound(want_a, mag_a, "float32", H / 64 + 16), f"d_aff {shape} {dtype}")
    # a token listed more often than the caller said: NaN for it, in each of the three, and for no other
    often = torch.zeros(T, dtype=torch.int32)
    ids = torch.from_numpy(tp2id).long()
    often.index_add_(0, ids[(ids >= 0) & (ids < T)], torch.ones(int(((ids >= 0) & (ids < T)).sum()), dtype=torch.int32))
    cut = (often > k - 1).numpy()
    got = values(combine_tokens(y, aff, tp, be, B, T, k - 1))
    assert np.array_equal(np.isnan(got).all(1), cut) and np.array_equal(np.isnan(got).any(1), cut)
    cut_y, cut_a = combine_tokens_bwd(d, y, aff, tp, be, B, k - 1)
    assert np.array_equal(np.isnan(values(cut_a)).all(1)[:T], cut) and not np.isnan(values(cut_a)[T:]).any()
    held = (tp2id >= 0) & (tp2id < T)
    want_nan = held & cut[np.where(held, tp2id, 0)]
    assert np.array_equal(np.isnan(values(cut_y)).all(1), want_nan) and np.array_equal(np.isnan(values(cut_y)).any(1), want_nan)


def test_padding_rows_are_not_read_and_bad_experts_count_for_nothing():
    """NaN in padding rows of y and in rows behind the tokens of the affinities; a block whose expert is -1, or E."""
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens_bwd

    T, H, E, k, B = 37, 40, 6, 2, 8
    rng, tp2id, b2e, tp, be, aff, y = _case((T, H, E, k, B), "bfloat16", 1)
    pad = torch.from_numpy((tp2id < 0) | (tp2id >= T)).cuda()
    y[pad] = float("nan")
    aff[T] = float("nan")
    b2e = b2e.copy()
    b2e[1], b2e[3] = -1, E
    be = tensor(b2e, "int32")
    a, yv = values(aff), np.where(pad.cpu().numpy()[:, None], 0, values(y))
    want, mag = ot.combine(yv, a, tp2id, b2e, B, T)
    assert_within(combine_tokens(y, aff, tp, be, B, T, k), want, bound(want, mag, "bfloat16", k + 1))
    d = tensor(rng.standard_normal((T, H)), "bfloat16")
    want_y, want_a, mag_a = ot.combine_bwd(values(d), yv, np.where(np.isnan(a), 0, a), tp2id, b2e, B)
    d_y, d_aff = combine_tokens_bwd(d, y, aff, tp, be, B, k)
    assert_within(d_y, want_y, bound(want_y, np.abs(want_y), "bfloat16", 1))
    assert_within(d_aff, want_a, bound(want_a, mag_a, "float32", 32))
    want, mag = ot.combine(yv, None, tp2id, b2e, B, T)
    assert_within(permute_tokens_bwd(y, tp, T, k), want, bound(want, mag, "bfloat16", k + 1))


def test_tokens_without_slots_and_tokens_listed_twice_for_an_expert():
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens_bwd

    rng = np.random.default_rng(5)
    T, H, E, B, k = 9, 72, 3, 4, 5
    # token 0 and 8 in no slot, token 3 twice in expert 1 and once in 0 and 2
    tp2id = np.array([1, 3, 9, -1, 3, 2, 3, 9, 4, 5, 6, 3], np.int32)
    b2e = np.array([0, 1, 2], np.int32)
    tp, be = tensor(tp2id, "int32"), tensor(b2e, "int32")
    y, aff, d = tensor(rng.standard_normal((12, H))), tensor(rng.random((T, E))), tensor(rng.standard_normal((T, H)))
    want, mag = ot.combine(values(y), values(aff), tp2id, b2e, B, T)
    out = combine_tokens(y, aff, tp, be, B, T, k)
    assert_within(out, want, bound(want, mag, "float32", k + 1))
    assert not out[0].any() and not out[8].any()
    assert not permute_tokens_bwd(y, tp, T, k)[0].any()
    want_y, want_a, mag_a = ot.combine_bwd(values(d), values(y), values(aff), tp2id, b2e, B)
    d_y, d_aff = combine_tokens_bwd(d, y, aff, tp, be, B, k)
    assert_within(d_y, want_y, bound(want_y, np.abs(want_y), "float32", 1))
    assert_within(d_aff, want_a, bound(want_a, mag_a, "float32", 40))


def test_a_token_listed_more_often_than_top_k_is_nan_and_alone():
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens_bwd

    T, H, E, k, B = 12, 24, 5, 2, 4
    rng, tp2id, b2e, tp, be, aff, y = _case((T, H, E, k, B), "float32", 2)
    tp2id = tp2id.copy()
    tp2id[np.flatnonzero(tp2id >= T)[0]] = 7  # a third slot
    tp = tensor(tp2id, "int32")
    d = tensor(rng.standard_normal((T, H)))
    out, dx = combine_tokens(y, aff, tp, be, B, T, k), permute_tokens_bwd(y, tp, T, k)
    d_y, d_aff = combine_tokens_bwd(d, y, aff, tp, be, B, k)
    others = torch.arange(T) != 7
    for t in (out, dx, d_aff[:T]):
        assert bool(t[7].isnan().all()) and not bool(t.cpu()[others].isnan().any())
    mine = torch.from_numpy(tp2id == 7)
    assert bool(d_y.cpu()[mine].isnan().all()) and not bool(d_y.cpu()[~mine].isnan().any())


def test_a_list_of_another_table_reads_nothing_outside():
    """A list that names slots behind y: those count for nothing."""
    from nkilib.core.moe.token_permute import permute_tokens_bwd

    y = tensor(np.ones((4, 8)))
    tp = tensor(np.array([0, 1, 0, 5]), "int32")
    lists = tensor(np.array([[2, 0, 2**31 - 1], [2, 1, 4]]), "int32")
    got = permute_tokens_bwd(y, tp, 2, 2, token_slots=lists)
    assert np.array_equal(values(got), np.ones((2, 8)))


def test_other_strides_streams_and_no_tokens():
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd

    T, H, E, k, B = 65, 48, 7, 3, 8
    rng, tp2id, b2e, tp, be, aff, y = _case((T, H, E, k, B), "bfloat16", 4)
    x = tensor(rng.standard_normal((H, T)), "bfloat16").t()  # columns first
    want = permute_tokens(x.contiguous(), tp)
    assert torch.equal(permute_tokens(x, tp), want)
    wide = torch.empty((y.shape[0], H + 5), dtype=y.dtype, device=y.device)
    wide[:, 3 : 3 + H] = y
    assert torch.equal(combine_tokens(wide[:, 3 : 3 + H], aff, tp, be, B, T, k), combine_tokens(y, aff, tp, be, B, T, k))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = permute_tokens(x, tp)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    # no tokens, no columns, an empty table
    none = torch.full_like(tp, -1)
    assert permute_tokens_bwd(y, none, 0, k).shape == (0, H)
    d_y, d_aff = combine_tokens_bwd(y[:0], y, aff, none, be, B, k)
    assert not d_y.any() and not d_aff.any() and d_y.shape == y.shape
    assert not permute_tokens(x[:0].contiguous(), tp).any()
    assert permute_tokens(x, tp[:0]).shape == (0, H) and not permute_tokens_bwd(y[:0], tp[:0], T, k).any()
    assert combine_tokens(y[:, :0], aff, tp, be, B, T, k).shape == (T, 0)


def test_refusals():
    import torch
    from nkilib.core.moe.token_permute import (build_token_slots, combine_tokens, combine_tokens_bwd, permute_tokens,
                                               permute_tokens_bwd)

    T, H, E, k, B = 12, 16, 4, 2, 4
    rng, tp2id, b2e, tp, be, aff, y = _case((T, H, E, k, B), "bfloat16", 3)
    d = y[:T].contiguous()
    bad = [
        lambda: permute_tokens(d, tp.long()), lambda: permute_tokens(d[0], tp), lambda: build_token_slots(tp, T, 0),
        lambda: build_token_slots(tp, T, 65), lambda: build_token_slots(tp, -1, 2),
        lambda: permute_tokens_bwd(y[:-1], tp, T, k), lambda: permute_tokens_bwd(y.to(torch.float64), tp, T, k),
        lambda: permute_tokens_bwd(y, tp, T, k, token_slots=torch.zeros((T, k), dtype=torch.int32, device="cuda")),
        lambda: combine_tokens(y, aff.half(), tp, be, B, T, k), lambda: combine_tokens(y, aff[: T - 1], tp, be, B, T, k),
        lambda: combine_tokens(y, aff.reshape(-1, 1)[:, 0], tp, be, B, T, k), lambda: combine_tokens(y, aff, tp, be, B + 1, T, k),
        lambda: combine_tokens(y, aff, tp, be.long(), B, T, k), lambda: combine_tokens(y, aff, tp, be[:-1], B, T, k),
        lambda: combine_tokens_bwd(d.float(), y, aff, tp, be, B, k), lambda: combine_tokens_bwd(d[:, :8], y, aff, tp, be, B, k),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError, match="NCC_INKI016"):
            call()
            pytest.fail(f"call {i} was not refused")


def test_rows_beyond_32_bit_offsets():
    """2.1 G elements of y: the slots of the last tokens lie past what 32 bits count."""
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens

    H, B, N = 16384, 8192, 17
    S, T, E = B * N, 64, 17
    tp = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(T, device="cuda") * 7 + (S - 64 * 7)
    tp[at] = torch.arange(T, dtype=torch.int32, device="cuda")
    be = torch.arange(N, dtype=torch.int32, device="cuda")
    assert S * H > 2**31
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn((T, H), generator=g, device="cuda").bfloat16()
    aff = torch.rand((T, E), generator=g, device="cuda")
    xs = permute_tokens(x, tp)
    assert torch.equal(xs[at], x) and float(xs.abs().sum(dtype=torch.float64)) == float(x.abs().sum(dtype=torch.float64))
    w = aff[:, N - 1 :]
    assert torch.equal(combine_tokens(xs, aff, tp, be, B, T, 1), (w * x.float()).bfloat16())
    d_y, d_aff = combine_tokens_bwd(x, xs, aff, tp, be, B, 1)
    assert torch.equal(d_y[at], (w * x.float()).bfloat16()) and not d_y[: S - 64 * 7].any()
    assert torch.allclose(d_aff[:, N - 1], (x.double() ** 2).sum(1).float(), rtol=1e-5) and not d_aff[:, : N - 1].any()
