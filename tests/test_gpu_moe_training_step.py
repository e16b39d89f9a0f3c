"""A routed layer's forward and backward pass from its operators, as a training step runs them.

1. A program that multiplies the experts itself: route -> block build -> permute -> gate/up product -> activation with the 8-bit
   record -> down product -> combine, and back.  The expert products are torch's, in fp32; everything else is the package's.
   Compared with the same layer in 64 bits whose activation's inputs are replaced, for the gradients, by the recorded values.
2. The backward pass of a layer that ``moe_cte`` ran with its checkpoints.

Tolerances: every value of the chain is a sum of products of bf16 values whose roundings are known; the bound used is the largest
of them, half a step of bf16 (2^-8) per rounded tensor on the way (counted per gradient), relative to the largest value of
the gradient, times the number of independent roundings.
"""

import numpy as np
import pytest

from oracle import train as ot
from train_helpers import tensor, values

pytestmark = pytest.mark.gpu


def _layer(seed, T=70, H=256, I=96, E=8, k=3, B=16):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).bfloat16()
    x = torch.cat((r(T, H), torch.zeros((1, H), device="cuda").bfloat16()))
    return dict(T=T, H=H, I=I, E=E, k=k, B=B, x=x, wr=r(H, E, std=H**-0.5), br=r(E).float(), wgu=r(E, H, 2, I, std=H**-0.5),
                wd=r(E, I, H, std=I**-0.5), d_out=r(T, H))


def _slots_by_expert(tp2id, b2e, B, T, E):
    e = np.repeat(b2e, B)
    on = (tp2id >= 0) & (tp2id < T)
    return [np.flatnonzero(on & (e == i)) for i in range(E)]


def _near(got, want, roundings, what):
    got = values(got)
    assert got.shape == want.shape
    err = np.abs(got - want).max()
    limit = roundings * 2.0**-8 * np.abs(want).max()
    assert err <= limit, f"{what}: off by {err:.3e}, at most {limit:.3e}"


def test_step_of_a_program_that_multiplies_the_experts():
    import torch
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd
    from nkilib.core.moe.moe_cte import build_token_blocks
    from nkilib.core.moe.token_permute import build_token_slots, combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd
    from nkilib.core.router_topk import route_for_moe, router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    L = _layer(1)
    T, H, I, E, k, B = (L[n] for n in "THIEkB")
    x, wgu, wd, d_out = L["x"], L["wgu"], L["wd"], L["d_out"]
    ids, aff, logits = route_for_moe(x, L["wr"], L["br"], k, RouterActFnType.SIGMOID, True, return_router_logits=True)
    tp, be, _ = build_token_blocks(ids, E, B, check=True)
    slots = build_token_slots(tp, T, k, check=True)
    lists = _slots_by_expert(tp.cpu().numpy(), be.cpu().numpy(), B, T, E)
    at = [torch.from_numpy(l).cuda() for l in lists]
    S = tp.numel()

    def products(rows, weight, out_cols):  # rows [S, K] x weight [E, K, out]: torch, fp32, rounded to bf16
        out = torch.zeros((S, out_cols), device="cuda")
        for e in range(E):
            out[at[e]] = rows[at[e]].float() @ weight[e].float()
        return out.bfloat16()

    xs = permute_tokens(x[:T], tp)
    gu = products(xs, wgu.reshape(E, H, 2 * I), 2 * I).view(S, 2, I)
    h, codes, scales = glu_checkpoint(gu, token_position_to_id=tp, n_tokens=T)
    ys = products(h, wd, H)
    out = combine_tokens(ys, aff, tp, be, B, T, k, token_slots=slots)
    # backward
    d_ys, d_aff = combine_tokens_bwd(d_out, ys, aff, tp, be, B, k, token_slots=slots)
    d_h = products(d_ys, wd.transpose(1, 2).contiguous(), I)
    d_gu, h2 = glu_checkpoint_bwd(codes, scales, d_h, token_position_to_id=tp, n_tokens=T)
    d_xs = products(d_gu.view(S, 2 * I), wgu.reshape(E, H, 2 * I).transpose(1, 2).contiguous(), H)
    d_x = permute_tokens_bwd(d_xs, tp, T, k, token_slots=slots)
    d_xr, d_wr, d_br = router_topk_bwd(d_aff, x[:T], L["wr"], L["br"], logits, ids, RouterActFnType.SIGMOID, norm_topk_prob=True)
    d_wd = [h2[a].float().t() @ d_ys[a].float() for a in at]

    # the same in 64 bits
    xv, wv, dv, dov, lv = values(x[:T]), values(wgu).reshape(E, H, 2 * I), values(wd), values(d_out), values(logits)
    idn = ids.cpu().numpy()
    assert np.array_equal(np.sort(idn, 1), np.sort(np.argsort(-lv, 1, kind="stable")[:, :k], 1))
    a = ot.router_affinities(lv, idn, False, True, True)
    _near(aff[:T], a, 1, "affinities")
    rec = values(dequantize_checkpoint(codes, scales))
    wout, wdx, wda = np.zeros((T, H)), np.zeros((T, H)), np.zeros((T, E))
    tpn = tp.cpu().numpy()
    for e in range(E):
        t = tpn[lists[e]]
        g64 = (xv[t] @ wv[e]).reshape(-1, 2, I)
        y64 = (ot.act(g64[:, 0], "silu")[0] * g64[:, 1]) @ dv[e]
        wout[t] += a[t, e : e + 1] * y64
        dy = a[t, e : e + 1] * dov[t]
        wda[t, e] = (dov[t] * y64).sum(1)
        dg, du, h64 = ot.glu_bwd(rec[lists[e], 0], rec[lists[e], 1], dy @ dv[e].T, "silu")
        wdx[t] += np.concatenate((dg, du), 1) @ wv[e].T
        _near(d_wd[e], h64.T @ dy, 4, f"down weights of expert {e}")  # h, dy, its affinity, their product's factors
        assert np.abs(rec[lists[e]] - g64).max() <= (2.0**-4 + 2.0**-8) * np.abs(g64).max()
    _near(out, wout, 6, "output")            # gate/up, h, y, affinity, the sum
    _near(d_aff[:T], wda, 6, "affinities' gradient")
    assert not d_aff[T].any()
    _near(d_x, wdx, 8, "tokens' gradient")    # affinity, dy, dh, dg, du, dxs, the sum
    want = ot.router_d_logits(values(d_aff[:T]), lv, idn, False, True, True)
    _near(d_xr, want @ values(L["wr"]).T, 2, "router's tokens")
    _near(d_wr, xv.T @ want, 2, "router's weights")
    _near(d_br, want.sum(0), 1, "router's bias")


def test_backward_of_a_layer_with_checkpoints():
    """moe_cte leaves gate_up_activations_T and down_activations; packed to 8 bits and combined backwards."""
    import torch
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint, glu_checkpoint_bwd, pack_gate_up_checkpoint
    from nkilib.core.moe.moe_cte import MoECTEImplementation, MoECTESpec, ShardOnIConfig, build_token_blocks, moe_cte
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd
    from nkilib.core.router_topk import route_for_moe
    from nkilib.core.utils.common_types import RouterActFnType

    L = _layer(2, T=150, H=256, I=128, E=4, k=2, B=152)  # (the layer with both checkpoints has a block per expert)
    T, H, I, E, k, B = (L[n] for n in "THIEkB")
    ids, aff = route_for_moe(L["x"], L["wr"], None, k, RouterActFnType.SOFTMAX, True)
    tp, be, cond = build_token_blocks(ids, E, B, E)
    spec = MoECTESpec(MoECTEImplementation.shard_on_i_dropping, shard_on_I=ShardOnIConfig(checkpoint_activation=True))
    out, gate_up_T, down = moe_cte(L["x"], aff.reshape(-1, 1), L["wgu"], L["wd"], tp, be, B, spec)
    N = be.numel()
    ys = down.view(N * B, H)
    # the layer's own sum adds in bf16 (one rounding per slot), this one in fp32
    mine = combine_tokens(ys, aff, tp, be, B, T, k)
    layer = out.reshape(-1, H)[:T] if out.dim() == 2 else out[0][:T]
    _near(mine, values(layer), k + 1, "combine of the checkpoint")
    codes, scales = pack_gate_up_checkpoint(gate_up_T, tp, T)
    rows = values(gate_up_T).transpose(0, 3, 1, 2).reshape(N * B, 2, I)
    on = (tp.cpu().numpy() >= 0) & (tp.cpu().numpy() < T)
    c, s = ot.record(rows)
    assert np.array_equal(codes.cpu().numpy(), c * on[:, None, None]) and np.array_equal(scales.cpu().numpy(), s * on[:, None, None])
    d_ys, d_aff = combine_tokens_bwd(L["d_out"], ys, aff, tp, be, B, k)
    want_y, want_a, _ = ot.combine_bwd(values(L["d_out"]), values(ys), values(aff), tp.cpu().numpy(), be.cpu().numpy(), B)
    _near(d_ys, want_y, 1, "d_ys")
    _near(d_aff, want_a, 1, "d_aff")
    d_h = torch.randn((N * B, I), device="cuda").bfloat16()
    d_gu, h = glu_checkpoint_bwd(codes, scales, d_h, token_position_to_id=tp, n_tokens=T)
    v = values(dequantize_checkpoint(codes, scales))
    dg, du, h64 = ot.glu_bwd(v[:, 0], v[:, 1], values(d_h), "silu")
    _near(h, h64 * on[:, None], 1, "h")
    _near(d_gu, np.stack((dg, du), 1) * on[:, None, None], 1, "d_gu")


def test_a_step_replays_from_a_graph():
    """Forward and backward recorded once; replayed with eager work of the same operators between the replays and with new inputs in
    the recorded buffers, every replay equals the eager result bit for bit."""
    import torch
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd
    from nkilib.core.moe.moe_cte import build_token_blocks
    from nkilib.core.router_topk import route_for_moe, router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    L = _layer(3, T=300, H=384, I=192, E=12, k=4, B=16)
    T, E, k, B, I = L["T"], L["E"], L["k"], L["B"], L["I"]

    def step(x, d_out):
        ids, aff, logits = route_for_moe(x, L["wr"], L["br"], k, RouterActFnType.SOFTMAX, True, return_router_logits=True)
        tp, be, _ = build_token_blocks(ids, E, B)
        xs = permute_tokens(x[:T], tp)
        gu = xs[:, : 2 * I].reshape(-1, 2, I)  # (stands for the products)
        h, codes, scales = glu_checkpoint(gu, token_position_to_id=tp, n_tokens=T)
        out = combine_tokens(h, aff, tp, be, B, T, k)
        d_h, d_aff = combine_tokens_bwd(d_out[:, :I].contiguous(), h, aff, tp, be, B, k)
        d_gu, _ = glu_checkpoint_bwd(codes, scales, d_h, token_position_to_id=tp, n_tokens=T)
        d_x = permute_tokens_bwd(d_gu.view(-1, 2 * I), tp, T, k)
        return (out, d_x, d_aff, codes, *router_topk_bwd(d_aff, x[:T], L["wr"], L["br"], logits, ids, RouterActFnType.SOFTMAX,
                                                        norm_topk_prob=True))

    x, d = L["x"].clone(), L["d_out"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, d)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, d)
    for replay in range(4):
        M = _layer(10 + replay, T=300, H=384, I=192, E=12, k=4, B=16)
        want = [t.clone() for t in step(M["x"], M["d_out"])]
        x.copy_(M["x"])
        d.copy_(M["d_out"])
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got, w), f"replay {replay}"
        step(x, d)  # eager work between the replays
        torch.cuda.synchronize()


def test_two_streams_at_once():
    """The same operators on two streams with different inputs share no memory."""
    import torch
    from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd, permute_tokens_bwd
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType
    from train_helpers import table

    rng = np.random.default_rng(0)
    T, H, E, k, B = 500, 512, 16, 4, 16
    cases = []
    for i in range(2):
        tp2id, b2e, N = table(rng, T, E, k, B)
        l = rng.standard_normal((T, E)).astype(np.float32)
        cases.append((tensor(tp2id, "int32"), tensor(b2e, "int32"), tensor(rng.standard_normal((N * B, H)), "bfloat16"),
                      tensor(rng.random((T + 1, E))), tensor(rng.standard_normal((T, H)), "bfloat16"), tensor(l),
                      tensor(np.argsort(-l, 1)[:, :k].copy(), "int32"), tensor(rng.standard_normal((H, E)), "bfloat16")))

    def work(c):
        tp, be, y, aff, d, l, ids, w = c
        d_y, d_aff = combine_tokens_bwd(d, y, aff, tp, be, B, k)
        return (combine_tokens(y, aff, tp, be, B, T, k), d_y, d_aff, permute_tokens_bwd(y, tp, T, k),
                *router_topk_bwd(d_aff, d, w, None, l, ids, RouterActFnType.SIGMOID)[:2])

    want = [work(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(work(c))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
