"""The router's gradient against the oracle in 64 bits.

Tolerances.  dl, in fp32, is off by a few units of 2^-24 of the magnitudes that make it (32 of them: exponentials, a sum over up to
512 experts in a tree, two divisions) and, in the products, by 2^-17 more of its own (two bf16).  An entry of dx adds up E products,
one of dw T of them, in fp32: at most that many steps of 2^-24 of the terms' magnitudes; then half a step of bf16.
"""

import numpy as np
import pytest

from oracle import train as ot
from train_helpers import assert_within, bound, tensor, values

pytestmark = pytest.mark.gpu

# softmax, router_pre_norm, norm_topk_prob, mask_to_topk
MODES = [(True, True, True, True), (True, True, False, True), (True, False, False, True), (False, True, True, True),
         (False, True, False, True), (False, False, False, True), (True, True, False, False), (False, True, False, False)]
# T, H, E, k: one token; every K of the kernels and odd numbers of experts at either side of their borders; the token axis cut
SHAPES = [(1, 128, 4, 1), (31, 256, 60, 4), (33, 128, 64, 8), (200, 384, 65, 8), (129, 256, 128, 2), (100, 640, 160, 6), (77, 128, 256, 8),
          (50, 256, 257, 8), (64, 128, 512, 3), (1500, 128, 33, 5)]


def _case(T, H, E, k, seed):
    rng = np.random.default_rng(seed)
    l = (rng.standard_normal((T, E)) * 2).astype(np.float32)
    ids = np.argsort(-l, 1, kind="stable")[:, :k].astype(np.int32)
    g = rng.standard_normal((T + 1, E)).astype(np.float32)
    return rng, l, ids, g, tensor(rng.standard_normal((T, H)), "bfloat16"), tensor(rng.standard_normal((H, E)) / 8, "bfloat16")


def _dl_limits(g, l, ids, mode):
    """dl in 64 bits and the error of the one in the products."""
    dl = ot.router_d_logits(g, l, ids, *mode)
    on = np.zeros(l.shape, bool)
    np.put_along_axis(on, ids, True, 1)
    # magnitudes: the terms whose difference dl is, with the largest affinity that stands before them
    p = np.abs(ot.router_affinities(l, ids, *mode[:3]))
    used = np.where(on | (not mode[3] and mode[1] and not mode[2]), np.abs(g), 0.0)
    if mode[0]:
        full = mode[1] and not mode[2]
        m = l if full else np.where(on, l, -np.inf)
        q = np.exp(m.astype(np.float64) - m.max(1, keepdims=True))
        q /= q.sum(1, keepdims=True)
        mag = q * (used + (used * q).sum(1, keepdims=True))
    else:
        s = 1 / (1 + np.exp(-l.astype(np.float64)))
        if mode[1] and mode[2]:
            total = np.where(on, s, 0).sum(1, keepdims=True)
            mag = np.where(on, (used + (used * s).sum(1, keepdims=True) / total) / total * s * (1 - s), 0.0)
        else:
            mag = used * s * (1 - s)
    del p
    return dl, 32 * 2.0**-24 * mag + 2.0**-17 * np.abs(dl)


def _check(got, want_dl, err, x, w, what, bias):
    d_x, d_w, d_b = got
    T, E = want_dl.shape
    a = np.abs(want_dl)
    want = want_dl @ w.T
    assert_within(d_x, want, bound(want, a @ np.abs(w.T), "bfloat16", E + 2) + err @ np.abs(w.T), "dx " + what)
    want = x.T @ want_dl
    assert_within(d_w, want, bound(want, np.abs(x.T) @ a, "bfloat16", T + 2) + np.abs(x.T) @ err, "dw " + what)
    if bias is None:
        assert d_b is None
    else:
        want = want_dl.sum(0)
        assert str(d_b.dtype) == "torch." + bias and d_b.shape == (E,)
        assert_within(d_b, want, bound(want, a.sum(0), bias, T + 2) + err.sum(0), "db " + what)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("mode", MODES)
def test_gradients(shape, mode):
    import torch
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    T, H, E, k = shape
    rng, l, ids, g, x, w = _case(T, H, E, k, T + E)
    bias = [None, "float32", "bfloat16"][(T + E + MODES.index(mode)) % 3]
    if (T + MODES.index(mode)) % 2:
        g = values(tensor(g, "bfloat16")).astype(np.float32)
    gd, ld = "bfloat16" if (T + MODES.index(mode)) % 2 else "float32", "bfloat16" if T % 3 == 1 else "float32"
    lt = tensor(l, ld)
    g[T] = np.nan  # the padding token's row is not read
    g_t = tensor(g, gd)
    if mode[3] or not mode[1] or mode[2]:  # gradients of experts that were not chosen are not read either
        on = np.zeros((T + 1, E), bool)
        np.put_along_axis(on[:T], ids, True, 1)
        g_t[~torch.from_numpy(on).cuda()] = float("nan")
    act = RouterActFnType.SOFTMAX if mode[0] else RouterActFnType.SIGMOID
    b = None if bias is None else torch.zeros(E, dtype=getattr(torch, bias), device="cuda")
    got = router_topk_bwd(g_t, x, w, b, lt, tensor(ids, "int32"), act, router_pre_norm=mode[1], norm_topk_prob=mode[2],
                          mask_to_topk=mode[3])
    want, err = _dl_limits(g[:T].astype(np.float64), values(lt), ids, mode)
    _check(got, want, err, values(x), values(w), f"{shape} {mode}", bias)


@pytest.mark.parametrize("T,H,E,k,softmax", [(8192, 7168, 256, 8, False), (4096, 2048, 128, 8, False), (1999, 4096, 60, 4, False),
                                             (3000, 1024, 300, 8, False), (17001, 1024, 300, 3, False), (16500, 1152, 70, 1, False),
                                             (8200, 2176, 512, 2, False), (9000, 2048, 200, 4, True)])
def test_large_shapes_on_the_device(T, H, E, k, softmax):
    """The token axis in many parts, dw and dx in one launch and in two, against products in 64 bits on the GPU."""
    import torch
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    rng, l, ids, g, x, w = _case(T, H, E, k, 9)
    mode = (softmax, True, not softmax, True)
    want, err = _dl_limits(g[:T].astype(np.float64), l, ids, mode)
    bias = torch.zeros(E, device="cuda")
    d_x, d_w, d_b = router_topk_bwd(tensor(g), x, w, bias, tensor(l), tensor(ids, "int32"),
                                    RouterActFnType.SOFTMAX if softmax else RouterActFnType.SIGMOID, norm_topk_prob=not softmax)
    dl, er = torch.from_numpy(want).cuda(), torch.from_numpy(err).cuda()
    xd, wd = x.double(), w.double()

    def near(got, val, mag, steps, e):
        limit = 2.0**-8 * val.abs() * (1 + 2.0**-7) + steps * 2.0**-24 * mag + e + 2.0**-134
        assert bool(((got.double() - val).abs() <= limit).all())

    wt, xt = wd.t().contiguous(), xd.t().contiguous()
    near(d_x, dl @ wt, dl.abs() @ wt.abs(), E + 2, er @ wt.abs())
    near(d_w, xt @ dl, xt.abs() @ dl.abs(), T + 2, xt.abs() @ er)
    assert_within(d_b, want.sum(0), bound(want.sum(0), np.abs(want).sum(0), "float32", T + 2) + err.sum(0))


def test_what_cancels_over_the_experts_does():
    """w with a large part that all experts share: a softmax's dl sum to zero, so that it leaves nothing in dx."""
    import torch
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    T, H, E, k = 40, 128, 64, 8
    rng, l, ids, g, x, w = _case(T, H, E, k, 1)
    small = (rng.integers(-8, 9, (H, E)) / 64).astype(np.float32)
    w = tensor(16.0 + small)  # 16 and steps of 1/64: not a bf16
    w = w.to(torch.bfloat16)
    want, err = _dl_limits(g[:T].astype(np.float64), l, ids, MODES[0])
    got = router_topk_bwd(tensor(g), x, w, None, tensor(l), tensor(ids, "int32"), RouterActFnType.SOFTMAX, norm_topk_prob=True)
    _check(got, want, err, values(x), values(w), "cancels", None)


def test_wrong_indices_and_repeats():
    """An index outside of the experts counts for nothing, one named twice counts once."""
    import torch
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    T, H, E = 3, 128, 10
    rng, l, _, g, x, w = _case(T, H, E, 3, 2)
    ids = np.array([[4, 2, 4], [-1, 10, 7], [-5, 2**31 - 1, -1]], np.int32)
    for mode in MODES[:6]:
        act = RouterActFnType.SOFTMAX if mode[0] else RouterActFnType.SIGMOID
        got = router_topk_bwd(tensor(g), x, w, None, tensor(l), tensor(ids, "int32"), act, router_pre_norm=mode[1], norm_topk_prob=mode[2])
        want, err = np.zeros((T, E)), np.zeros((T, E))
        for t, mine in enumerate(([4, 2], [7], [])):
            if mine:
                want[t : t + 1], err[t : t + 1] = _dl_limits(g[t : t + 1].astype(np.float64), l[t : t + 1], np.array([mine]), mode)
        _check(got, want, err, values(x), values(w), str(mode), None)


def test_extreme_logits():
    """Logits far out and infinite: gradients of saturated scores are zero, not NaN; the rest of the batch is as without them."""
    import torch
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    T, H, E, k = 5, 128, 12, 3
    rng, l, ids, g, x, w = _case(T, H, E, k, 3)
    l[1], l[2, ids[2, 0]], l[3, ids[3, 1:]] = l[1] * 1e4, np.inf, -np.inf
    for mode in ((False, True, False, True), (True, True, True, True)):
        if mode[0]:
            l[2, ids[2, 0]] = 300.0  # (a softmax of an infinity has no value)
        act = RouterActFnType.SOFTMAX if mode[0] else RouterActFnType.SIGMOID
        d_x, d_w, _ = router_topk_bwd(tensor(g), x, w, None, tensor(l), tensor(ids, "int32"), act, norm_topk_prob=mode[2])
        with np.errstate(all="ignore"):
            want, err = _dl_limits(g[:T].astype(np.float64), l, ids, mode)
        _check((d_x, d_w, None), want, err, values(x), values(w), str(mode), None)


def test_scores_near_zero_divided_by_their_sum():
    """Sigmoid scores of 1e-37 divided by their sum are ordinary affinities with ordinary gradients."""
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    T, H, E, k = 20, 128, 12, 4
    rng, l, ids, g, x, w = _case(T, H, E, k, 6)
    l = (l / 4 - 85).astype(np.float32)
    g *= 100
    mode = (False, True, True, True)
    got = router_topk_bwd(tensor(g), x, w, None, tensor(l), tensor(ids, "int32"), RouterActFnType.SIGMOID, norm_topk_prob=True)
    want, err = _dl_limits(g[:T].astype(np.float64), l, ids, mode)
    _check(got, want, err, values(x), values(w), str(mode), None)


def test_route_for_moe_hands_out_the_logits():
    import torch
    from nkilib.core.router_topk import route_for_moe
    from nkilib.core.utils.common_types import RouterActFnType

    rng = np.random.default_rng(4)
    T, H, E, k = 50, 256, 24, 4
    x, w = tensor(rng.standard_normal((T + 1, H)), "bfloat16"), tensor(rng.standard_normal((H, E)) / 16, "bfloat16")
    b = tensor(rng.standard_normal(E))
    idx, aff = route_for_moe(x, w, b, k, RouterActFnType.SIGMOID, True)
    idx2, aff2, logits = route_for_moe(x, w, b, k, RouterActFnType.SIGMOID, True, return_router_logits=True)
    assert torch.equal(idx, idx2) and torch.equal(aff, aff2) and logits.dtype == torch.float32
    want = values(x)[:T] @ values(w) + values(b)
    assert_within(logits, want, (H + 4) * 2.0**-24 * (np.abs(values(x)[:T]) @ np.abs(values(w)) + np.abs(values(b))))


def test_refusals():
    import torch
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    T, H, E, k = 6, 128, 8, 2
    rng, l, ids, g, x, w = _case(T, H, E, k, 5)
    a = dict(d_expert_affinities=tensor(g), x=x, w=w, w_bias=None, router_logits=tensor(l), expert_index=tensor(ids, "int32"),
             act_fn=RouterActFnType.SOFTMAX)
    bad = [dict(x=x.float()), dict(x=x[:, :64]), dict(w=w[:64]), dict(x=x[:, :96], w=w[:96]), dict(expert_index=a["expert_index"].long()),
           dict(expert_index=a["expert_index"][:3]), dict(router_logits=a["router_logits"][:, :4]), dict(router_logits=a["router_logits"].half()),
           dict(d_expert_affinities=tensor(g)[:3]), dict(d_expert_affinities=tensor(g).double()), dict(w_bias=torch.zeros(3, device="cuda")),
           dict(expert_index=torch.zeros((T, 9), dtype=torch.int32, device="cuda"))]
    for kw in bad:
        with pytest.raises(AssertionError, match="NCC_INKI016"):
            router_topk_bwd(**{**a, **kw})
            pytest.fail(f"{list(kw)} was not refused")
    d_x, d_w, d_b = router_topk_bwd(tensor(g)[:0], x[:0], w, torch.zeros(E, device="cuda"), tensor(l)[:0], a["expert_index"][:0], 1)
    assert d_x.shape == (0, H) and not d_w.any() and not d_b.any()
