"""Lists of long tables, launches that go round more than once, tables without slots (operators and tolerances: test_gpu_token_permute).

Long tables are looked at on the device: their oracle is torch's, in whole numbers for the lists and in 64 bits for the sums.
"""

import numpy as np
import pytest

from oracle import train as ot
from train_helpers import tensor

pytestmark = pytest.mark.gpu


def _lists(tp, T, k):
    """[T, 1 + k] of a table on the device: counts, the first k slots in ascending order, -1."""
    import torch

    ids = torch.where((tp >= 0) & (tp < T), tp.long(), T)
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=T + 1)[:T]
    first = torch.cumsum(counts, 0) - counts
    j = torch.arange(k, device=tp.device)
    at = (first[:, None] + j).clamp(max=max(tp.numel() - 1, 0))
    out = torch.where(j < counts[:, None], order[at], -1)
    return torch.cat((counts[:, None], out), 1).int()


# tokens, slots, most slots of a token: tables on either side of 2^30 entries read by the workgroups that own the tokens, tokens without
# slots in most lists, a last workgroup with few tokens
@pytest.mark.parametrize("T,S,k", [(1, 300_000, 64), (70_000, 600_000, 8), (12, 262_145, 3), (4001, 5_000_000, 64), (600_001, 5_000_002, 8),
                                   (1_000_003, 4_300_001, 1), (200_000, 4_300_003, 2), (3_000_000, 1_000_000, 5), (1_048_576, 8_600_000, 7)])
def test_lists_of_long_tables(T, S, k):
    import torch
    from nkilib.core.moe.token_permute import build_token_slots

    g = torch.Generator(device="cuda").manual_seed(T + S)
    # every token up to k times, at places in any order; the rest padding of any kind
    most = min(k * T, S - S // 10)
    tp = torch.tensor([T, -1, 2**31 - 1, -(2**31)], dtype=torch.int32, device="cuda")[torch.randint(0, 4, (S,), generator=g, device="cuda")]
    tokens = torch.arange(k * T, device="cuda", dtype=torch.int64)[torch.randperm(k * T, generator=g, device="cuda")[:most]] % T
    tp[torch.randperm(S, generator=g, device="cuda")[:most]] = tokens.int()
    want = _lists(tp, T, k)
    assert int(want[:, 0].max()) <= k
    assert torch.equal(build_token_slots(tp, T, k), want)
    odd = torch.cat((tp[:3], tp))  # a table that begins at a 4-byte address
    assert torch.equal(build_token_slots(odd[3:], T, k), want)
    if k > 1:  # lists that are cut: the true count, slots that are the token's, each once
        cut = build_token_slots(tp, T, k - 1)
        assert torch.equal(cut[:, 0], want[:, 0])
        whole = want[:, 0] < k
        assert torch.equal(cut[whole], want[whole][:, :k])
        long = cut[~whole][:, 1:]
        if long.numel():
            assert bool((tp[long.long()] == torch.nonzero(~whole).int()).all()) and bool((long[:, 1:] > long[:, :-1]).all())


def test_sums_over_a_long_table():
    """permute and combine, both ways, with lists that the calls make themselves."""
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd

    T, H, E, k, B = 1_050_000, 20, 16, 4, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.rand((T, E), generator=g, device="cuda").topk(k, dim=1).indices
    order = torch.argsort(ids.reshape(-1), stable=True)
    counts = torch.bincount(ids.reshape(-1), minlength=E)
    blocks = (counts + B - 1) // B
    first, rank = (torch.cumsum(blocks, 0) - blocks) * B, torch.arange(T * k, device="cuda") - (torch.cumsum(counts, 0) - counts)[ids.reshape(-1)[order]]
    N = int(blocks.sum())
    tp = torch.full((N * B,), T, dtype=torch.int32, device="cuda")
    at = first[ids.reshape(-1)[order]] + rank
    tp[at] = (order // k).int()
    be = torch.repeat_interleave(torch.arange(E, dtype=torch.int32, device="cuda"), blocks)
    S = N * B
    x, d = (torch.randn((T, H), generator=g, device="cuda") for _ in range(2))
    aff = torch.rand((T, E), generator=g, device="cuda")
    on = tp < T
    xs = permute_tokens(x, tp)
    assert torch.equal(xs[on], x[tp[on].long()]) and not xs[~on].any()
    e = be.long().repeat_interleave(B)[on]
    t = tp[on].long()
    w = aff.double()[t, e]
    want = torch.zeros((T, H), dtype=torch.float64, device="cuda").index_add_(0, t, xs[on].double())
    mag = torch.zeros_like(want).index_add_(0, t, xs[on].double().abs())
    near = lambda got, want, mag, steps: bool(((got.double() - want).abs() <= 2.0**-24 * (want.abs() + steps * mag)).all())
    assert near(permute_tokens_bwd(xs, tp, T, k), want, mag, k + 1)
    want = torch.zeros_like(want).index_add_(0, t, xs[on].double() * w[:, None])
    assert near(combine_tokens(xs, aff, tp, be, B, T, k), want, torch.zeros_like(want).index_add_(0, t, (xs[on].double() * w[:, None]).abs()), k + 2)
    d_y, d_aff = combine_tokens_bwd(d, xs, aff, tp, be, B, k)
    assert near(d_y[on], d.double()[t] * w[:, None], torch.zeros((), device="cuda"), 0) and not d_y[~on].any()
    terms = d.double()[t] * xs[on].double()
    want = torch.zeros((T, E), dtype=torch.float64, device="cuda").index_put_((t, e), terms.sum(1))
    mag = torch.zeros_like(want).index_put_((t, e), terms.abs().sum(1))
    assert near(d_aff, want, mag, H / 64 + 16)


def test_a_long_tables_lists_in_a_graph_and_on_two_streams():
    import torch
    from nkilib.core.moe.token_permute import build_token_slots

    T, S, k = 400_000, 4_500_000, 40  # (no token lies in 40 slots)
    tables = [torch.randint(-1, T + 2, (S,), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").int() for i in range(4)]
    want = [_lists(t, T, k) for t in tables]
    assert max(int(w[:, 0].max()) for w in want) <= k
    buf = tables[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        build_token_slots(buf, T, k)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = build_token_slots(buf, T, k)
    for i in (1, 2, 3, 1):
        buf.copy_(tables[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        assert torch.equal(build_token_slots(tables[0], T, k), want[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got.append(build_token_slots(tables[i], T, k))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_slots_and_no_table():
    """Without slots there is no table to hand over, and every sum is zero whatever the scratch memory holds."""
    import torch
    from nkilib import _native as nv

    L = nv.lib()
    y = torch.ones((1, 16), device="cuda")
    aff, be = torch.ones((4, 3), device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for T in (1, 4, 600):
        for fill in (0, 2, 10**6, -1):
            slots = torch.full((T, 3), fill, dtype=torch.int32, device="cuda")
            out = torch.full((T, 16), 7.0, device="cuda")
            rc = L.moe_combine_tokens(y.data_ptr(), nv.DT_FP32, None, 0, 0, 0, None, None, 0, 0, slots.data_ptr(), 2, 1, 0, T, 16,
                                      out.data_ptr(), nv.stream_ptr(y.device))
            assert rc == 0 and not out.any(), (T, fill)
            if T <= 4:
                out.fill_(7.0)
                rc = L.moe_combine_tokens(y.data_ptr(), nv.DT_FP32, aff.data_ptr(), nv.DT_FP32, 4, 3, None, be.data_ptr(), 4, 0,
                                          slots.data_ptr(), 2, 1, 0, T, 16, out.data_ptr(), nv.stream_ptr(y.device))
                assert rc == 0 and not out.any(), (T, fill)


# A launch holds at most 2^20 workgroups, which take their next job 2^20 further on: rows of more than 4 KB are a workgroup's job,
# shorter ones a wave's, four to a workgroup.
@pytest.mark.parametrize("T,H,dtype", [((1 << 20) + 77, 2051, "bfloat16"), ((1 << 22) + 77, 9, "float16"), ((1 << 22) + 77, 3, "float32")])
def test_more_rows_than_a_launch_has_workgroups(T, H, dtype):
    import torch
    from nkilib.core.moe.token_permute import build_token_slots, combine_tokens, combine_tokens_bwd, permute_tokens

    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(H)
    B, E = 64, 3
    N = (T + 5 + B - 1) // B
    S = N * B
    tp = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    at = torch.randperm(S, generator=g, device="cuda")[:T]
    tp[at] = torch.arange(T, dtype=torch.int32, device="cuda")
    be = torch.randint(0, E, (N,), generator=g, device="cuda").int()
    # values of few bits: every product is exact in fp32, so that the results are known to the bit
    x = torch.randint(-8, 9, (T, H), generator=g, device="cuda", dtype=torch.int8).to(dt)
    aff = torch.randint(1, 9, (T + 2, E), generator=g, device="cuda").float() / 8
    xs = permute_tokens(x, tp)
    parts = [slice(i, min(i + (1 << 18), T)) for i in range(0, T, 1 << 18)]
    for p in parts:
        assert torch.equal(xs[at[p]], x[p])
    pad = torch.nonzero(tp < 0)[:, 0]
    assert not xs[pad].any()
    slots = build_token_slots(tp, T, 1)
    assert torch.equal(slots[:, 1], at.int()) and bool((slots[:, 0] == 1).all())
    w = aff[torch.arange(T, device="cuda"), be.long()[at // B]]
    out = combine_tokens(xs, aff, tp, be, B, T, 1, token_slots=slots)
    for p in parts:
        assert torch.equal(out[p], (w[p, None] * x[p].float()).to(dt))
    del out
    d_y, d_aff = combine_tokens_bwd(x, xs, aff, tp, be, B, 1, token_slots=slots)
    assert not d_y[pad].any()
    total = 0.0
    for p in parts:
        assert torch.equal(d_y[at[p]], (w[p, None] * x[p].float()).to(dt))
        sums = (x[p].float() ** 2).sum(1)
        assert torch.equal(d_aff[p].gather(1, be.long()[at[p] // B][:, None])[:, 0], sums)
        total += float(sums.double().sum())
    assert float(d_aff.double().sum()) == total


def test_more_rows_of_a_record_than_a_launch_has_threads():
    """Rows of one value: four pieces each, 2^32 of them past 2^30 rows."""
    import torch
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd

    R, far = (1 << 30) + 300, 1 << 30
    x = torch.ones((R, 2, 1), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    x[-1000:] = torch.randn((1000, 2, 1), generator=g, device="cuda").bfloat16()
    h, c, s = glu_checkpoint(x)
    h1, c1, s1 = glu_checkpoint(x[-1000:].contiguous())
    assert torch.equal(h[-1000:], h1) and torch.equal(c[-1000:], c1) and torch.equal(s[-1000:], s1)
    assert bool((h[: far - 1000 : 4099] == h[0]).all()) and bool((c[: far - 1000 : 4099] == c[0]).all())
    del x
    v = dequantize_checkpoint(c, s)
    assert torch.equal(v[-1000:], dequantize_checkpoint(c1, s1)) and bool((v[: far - 1000 : 4099] == 1).all())
    del v
    d_gu, h2 = glu_checkpoint_bwd(c, s, h)
    d1, h3 = glu_checkpoint_bwd(c1, s1, h1)
    assert torch.equal(d_gu[-1000:], d1) and torch.equal(h2[-1000:], h3) and bool((d_gu[: far - 1000 : 4099] == d_gu[0]).all())


def test_more_blocks_of_a_checkpoint_than_a_launch_takes():
    import torch
    from nkilib.core.moe.glu_checkpoint import pack_gate_up_checkpoint

    N = (1 << 23) + 300  # (two tiles a block, fewer than 2^24 a launch)
    x = torch.ones((N, 2, 1, 1), dtype=torch.bfloat16, device="cuda")
    x[-1000:] = torch.randn((1000, 2, 1, 1), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").bfloat16()
    c, s = pack_gate_up_checkpoint(x)
    c1, s1 = pack_gate_up_checkpoint(x[-1000:].contiguous())
    assert torch.equal(c[-1000:], c1) and torch.equal(s[-1000:], s1)
    assert bool((c[:-1000] == c[0]).all()) and bool((s[:-1000] == s[0]).all())
    assert np.array_equal(c1.cpu().numpy(), ot.record(x[-1000:, :, :, 0].float().cpu().numpy())[0])


@pytest.mark.parametrize("H,dtype", [(2047, "bfloat16"), (2048, "float16"), (2559, "bfloat16"), (2560, "bfloat16"), (1279, "float32"), (1281, "float32")])
def test_a_row_is_summed_alike_by_a_wave_and_by_a_workgroup(H, dtype):
    """Few tokens (a workgroup each) and the same among many (a wave each, up to the rule's length): the same bits."""
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, permute_tokens_bwd

    g = torch.Generator(device="cuda").manual_seed(H)
    E, k, B = 8, 3, 16
    for T in (2047, 2048):
        ids = torch.arange(T * k, device="cuda", dtype=torch.int32) // k
        N = (T * k + B - 1) // B
        tp = torch.full((N * B,), T, dtype=torch.int32, device="cuda")
        tp[: T * k] = ids[torch.randperm(T * k, generator=g, device="cuda")]
        tp[: T * k][tp[: T * k] == T - 1] = T  # (the last token has no slot)
        if T == 2047:
            be = torch.randint(0, E, (N,), generator=g, device="cuda").int()
            y = torch.randn((N * B, H), generator=g, device="cuda").to(getattr(torch, dtype))
            aff = torch.rand((T, E), generator=g, device="cuda")
            first = (tp, be, y, aff)
            want = combine_tokens(y, aff, tp, be, B, T, k), permute_tokens_bwd(y, tp, T, k)
        else:
            tp, be, y, aff = first
            aff = torch.cat((aff, aff[:1]))
            tp = torch.where(tp == 2047, -1, tp)
            got = combine_tokens(y, aff, tp, be, B, T, k), permute_tokens_bwd(y, tp, T, k)
            for a, b in zip(got, want):
                assert torch.equal(a[:2047], b) and not a[2047].any()
