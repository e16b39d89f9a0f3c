"""The products and norms together, as a program runs a layer with them.

1. A training step: route -> block build in compact order -> permute -> gate/up product -> gated activation -> down product -> combine,
   and back, every product the package's; against the same step in 64 bits.
2. A serving step in 8-bit integers: norm with the residual -> permute of codes and scales -> gate/up -> activation -> rows to 8
   bits -> down -> combine; every stage against its formula on what the stage before gave.
3. Both from a recorded graph.

Tolerances as in test_gpu_moe_training_step.py: half a step of bf16 (2^-8) per rounded tensor on the way, relative to the largest value.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _near(got, want, roundings, what):
    got = got.double()
    assert got.shape == want.shape, what
    err, limit = (got - want).abs().max().item(), roundings * 2.0**-8 * want.abs().max().item()
    assert err <= limit, f"{what}: off by {err:.3e}, at most {limit:.3e}"


def _layer(seed, T=70, H=256, I=96, E=8, k=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).bfloat16()
    x = torch.cat((r(T, H), torch.zeros((1, H), device="cuda").bfloat16()))
    return dict(T=T, H=H, I=I, E=E, k=k, x=x, wr=r(H, E, std=H**-0.5), wgu=r(E, H, 2 * I, std=H**-0.5), wd=r(E, I, H, std=I**-0.5),
                gamma=(1 + 0.1 * torch.randn(H, generator=g, device="cuda")).bfloat16(), res=r(T, H), d_out=r(T, H))


def _train(L, ids, aff, B):
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint, glu_checkpoint_bwd
    from nkilib.core.moe.grouped_matmul import expert_row_offsets, grouped_matmul, grouped_matmul_bwd
    from nkilib.core.moe.moe_cte import build_token_blocks
    from nkilib.core.moe.token_permute import build_token_slots, combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd

    T, H, I, E, k = (L[n] for n in "THIEk")
    x = L["x"][:T]
    tp, be, _ = build_token_blocks(ids, E, B)
    o = expert_row_offsets(be, B, E)
    slots = build_token_slots(tp, T, k)
    xs = permute_tokens(x, tp)
    gu = grouped_matmul(xs, L["wgu"], o)
    h, codes, scales = glu_checkpoint(gu.view(-1, 2, I), token_position_to_id=tp, n_tokens=T)
    ys = grouped_matmul(h, L["wd"], o)
    out = combine_tokens(ys, aff, tp, be, B, T, k, token_slots=slots)
    d_ys, d_aff = combine_tokens_bwd(L["d_out"], ys, aff, tp, be, B, k, token_slots=slots)
    d_h, _ = grouped_matmul_bwd(d_ys, None, L["wd"], o, need_weight=False)
    d_gu, h2 = glu_checkpoint_bwd(codes, scales, d_h, token_position_to_id=tp, n_tokens=T)
    _, d_wd = grouped_matmul_bwd(d_ys, h2, L["wd"], o, need_x=False)
    d_xs, d_wgu = grouped_matmul_bwd(d_gu.view(-1, 2 * I), xs, L["wgu"], o, weight_grad_dtype=torch.float32)
    d_x = permute_tokens_bwd(d_xs, tp, T, k, token_slots=slots)
    return dict(out=out, d_x=d_x, d_wd=d_wd, d_wgu=d_wgu, d_aff=d_aff, codes=codes, scales=scales, tp=tp, be=be, o=o)


@pytest.mark.parametrize("B", [1, 16])
def test_training_step(B):
    from nkilib.core.moe.glu_checkpoint import dequantize_checkpoint
    from nkilib.core.router_topk import route_for_moe
    from nkilib.core.utils.common_types import RouterActFnType

    L = _layer(1)
    T, H, I, E, k = (L[n] for n in "THIEk")
    ids, aff = route_for_moe(L["x"], L["wr"], None, k, RouterActFnType.SIGMOID, True)
    got = _train(L, ids, aff, B)
    x, wgu, wd, d_out, a = L["x"][:T].double(), L["wgu"].double(), L["wd"].double(), L["d_out"].double(), aff[:T].double()
    rec = dequantize_checkpoint(got["codes"], got["scales"]).double()
    tp, row_e = got["tp"].long(), got["be"].repeat_interleave(B)
    out, d_x, d_wd, d_wgu = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(wd), torch.zeros_like(wgu)
    assert got["o"].tolist() == [B * int((got["be"] < e).sum()) for e in range(E + 1)]
    for e in range(E):
        at = ((row_e == e) & (tp >= 0) & (tp < T)).nonzero()[:, 0]
        t = tp[at]
        assert torch.equal(t.sort().values, (ids == e).any(1).nonzero()[:, 0])
        g64 = (x[t] @ wgu[e]).view(-1, 2, I)
        y = (torch.nn.functional.silu(g64[:, 0]) * g64[:, 1]) @ wd[e]
        out[t] += a[t, e : e + 1] * y
        dy = a[t, e : e + 1] * d_out[t]
        # (the activation's gradient is that at the values which its 8-bit record holds)
        r64 = rec[at].clone().requires_grad_()
        h64 = torch.nn.functional.silu(r64[:, 0]) * r64[:, 1]
        (dg,) = torch.autograd.grad(h64, r64, dy @ wd[e].t().contiguous())
        dg = dg.view(-1, 2 * I)
        d_x[t] += dg @ wgu[e].t().contiguous()
        d_wd[e] = h64.detach().t().contiguous() @ dy
        d_wgu[e] = x[t].t().contiguous() @ dg
    _near(got["out"], out, 6, "output")                    # gate/up, h, y, affinity, the sum
    _near(got["d_x"], d_x, 8, "tokens' gradient")          # affinity, dy, dh, dg, dxs, the sum
    _near(got["d_wd"], d_wd, 4, "down weights")            # h, affinity, dy, the sum
    _near(got["d_wgu"], d_wgu, 5, "gate/up weights")       # affinity, dy, dh, dg
    assert got["d_wgu"].dtype == torch.float32


def _serve(L, ids, aff, w):
    from nkilib.core.int8_matmul import grouped_int8_matmul
    from nkilib.core.moe.glu_checkpoint import glu_checkpoint
    from nkilib.core.moe.grouped_matmul import expert_row_offsets
    from nkilib.core.moe.moe_cte import build_token_blocks
    from nkilib.core.moe.token_permute import combine_tokens, permute_tokens
    from nkilib.core.rmsnorm import rmsnorm_quant_rows

    T, I, E, k = (L[n] for n in "TIEk")
    tp, be, _ = build_token_blocks(ids, E, 1)
    o = expert_row_offsets(be, 1, E)
    codes, scales, stream = rmsnorm_quant_rows(L["x"][:T], L["gamma"], residual=L["res"])
    xs, ss = permute_tokens(codes, tp), permute_tokens(scales[:, None], tp)
    gu = grouped_int8_matmul(xs, ss, w["gu"], w["gu_s"], o)
    h, _, _ = glu_checkpoint(gu.view(-1, 2, I), token_position_to_id=tp, n_tokens=T)
    hq, hs = rmsnorm_quant_rows(h, None, do_norm=False)
    ys = grouped_int8_matmul(hq, hs, w["d"], w["d_s"], o)
    out = combine_tokens(ys, aff, tp, be, 1, T, k)
    return dict(codes=codes, scales=scales, stream=stream, gu=gu, h=h, hq=hq, hs=hs, ys=ys, out=out, tp=tp, be=be)


def _weights(L):
    from nkilib.core.rmsnorm import rmsnorm_quant_rows

    gu, gu_s = rmsnorm_quant_rows(L["wgu"].transpose(1, 2).contiguous(), None, do_norm=False)
    d, d_s = rmsnorm_quant_rows(L["wd"].transpose(1, 2).contiguous(), None, do_norm=False)
    return dict(gu=gu, gu_s=gu_s, d=d, d_s=d_s)


@pytest.mark.parametrize("T", [1, 70])
def test_serving_step_in_8_bit_integers(T):
    from nkilib.core.rmsnorm import dequantize_rows
    from nkilib.core.router_topk import route_for_moe
    from nkilib.core.utils.common_types import RouterActFnType

    L = _layer(2, T=T)
    I, E, k = L["I"], L["E"], L["k"]
    w = _weights(L)
    wg, wd = dequantize_rows(w["gu"], w["gu_s"], torch.float32).double(), dequantize_rows(w["d"], w["d_s"], torch.float32).double()
    # a weight is off by at most half a step of its channel's scale
    assert bool(((wg - L["wgu"].double().transpose(1, 2)).abs() <= w["gu_s"].double()[..., None] * (0.5 + 2.0**-16)).all())
    ids, aff = route_for_moe(L["x"], L["wr"], None, k, RouterActFnType.SIGMOID, True)
    got = _serve(L, ids, aff, w)
    s = (L["x"][:T].float() + L["res"].float()).bfloat16()
    assert torch.equal(got["stream"], s)
    y = s.double() / torch.sqrt((s.double() ** 2).mean(1, keepdim=True) + 1e-6) * L["gamma"].double()
    xq = got["codes"].double() * got["scales"].double()[:, None]
    assert bool(((xq - y).abs() <= got["scales"].double()[:, None] * (0.5 + 2.0**-16)).all())
    tp, be, a = got["tp"].long(), got["be"].long(), aff[:T].double()
    out = torch.zeros_like(y)
    hq = got["hq"].double() * got["hs"].double()[:, None]
    for e in range(E):
        at = ((be == e) & (tp >= 0) & (tp < T)).nonzero()[:, 0]
        if at.numel() == 0:
            continue
        t = tp[at]
        gu = xq[t] @ wg[e].t().contiguous()
        _near(got["gu"][at], gu, 1.01, f"gate/up of expert {e}")
        g64 = got["gu"][at].double().view(-1, 2, I)
        _near(got["h"][at], torch.nn.functional.silu(g64[:, 0]) * g64[:, 1], 1.01, f"activation of expert {e}")
        ys = hq[at] @ wd[e].t().contiguous()
        _near(got["ys"][at], ys, 1.01, f"down of expert {e}")
        out[t] += a[t, e : e + 1] * ys
    assert bool(((hq - got["h"].double()).abs() <= got["hs"].double()[:, None] * (0.5 + 2.0**-16)).all())
    _near(got["out"], out, 3, "output")


def test_both_steps_from_a_graph():
    from nkilib.core.router_topk import route_for_moe
    from nkilib.core.utils.common_types import RouterActFnType

    L = _layer(3)
    w = _weights(L)
    ids, aff = route_for_moe(L["x"], L["wr"], None, L["k"], RouterActFnType.SIGMOID, True)
    step = lambda: list(_train(L, ids, aff, 1).values()) + list(_serve(L, ids, aff, w).values())
    step(), step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        L["x"][: L["T"]] = torch.randn_like(L["x"][: L["T"]])
        new_ids, new_aff = route_for_moe(L["x"], L["wr"], None, L["k"], RouterActFnType.SIGMOID, True)
        ids.copy_(new_ids)
        aff.copy_(new_aff)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_launches_are_made_on_the_tensors_device(monkeypatch):
    """As in test_gpu_other_device.py: the stream is asked for inside the tensors' device."""
    import contextlib

    from nkilib import _native as nv
    from nkilib.core.int8_matmul import grouped_int8_matmul, int8_matmul
    from nkilib.core.moe.grouped_matmul import expert_row_offsets, grouped_matmul, grouped_matmul_bwd
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

    inside, asked = [], []
    real = nv.stream_ptr

    @contextlib.contextmanager
    def on_device(device):
        inside.append(device)
        yield
        inside.pop()

    monkeypatch.setattr(nv, "on_device", on_device)
    monkeypatch.setattr(nv, "stream_ptr", lambda device: (asked.append(inside[-1:] == [device]), real(device))[1])
    x, w = torch.randn(8, 16, device="cuda").bfloat16(), torch.randn(2, 16, 24, device="cuda").bfloat16()
    o = torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda")
    c, s = rmsnorm_quant_rows(x, None)
    wc, ws = rmsnorm_quant_rows(w.transpose(1, 2).contiguous(), None, do_norm=False)
    calls = [lambda: grouped_matmul(x, w, o), lambda: grouped_matmul_bwd(grouped_matmul(x, w, o), x, w, o),
             lambda: expert_row_offsets(o, 1, 9),
             lambda: int8_matmul(c, s, wc[0], ws[0]), lambda: grouped_int8_matmul(c, s, wc, ws, o), lambda: rmsnorm_quant_rows(x, None),
             lambda: rmsnorm_quant_rows_bwd(x, x, None), lambda: dequantize_rows(c, s)]
    for i, call in enumerate(calls):
        asked.clear()
        call()
        assert asked and all(asked), i
