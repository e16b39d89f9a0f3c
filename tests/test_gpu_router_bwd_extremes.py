"""The router's gradient where logits, gradients and repeats are at their worst (tolerances: test_gpu_router_topk_bwd)."""

import numpy as np
import pytest

import test_gpu_router_topk_bwd as base
from test_gpu_router_topk_bwd import MODES, _case, _check, _dl_limits
from train_helpers import tensor, values

pytestmark = pytest.mark.gpu


def _call(g, x, w, l, ids, mode, bias=None):
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    return router_topk_bwd(tensor(g), x, w, bias, tensor(l), tensor(ids, "int32"), RouterActFnType.SOFTMAX if mode[0] else RouterActFnType.SIGMOID,
                           router_pre_norm=mode[1], norm_topk_prob=mode[2], mask_to_topk=mode[3])


@pytest.mark.parametrize("mode", [m for m in MODES if m[0]])
@pytest.mark.parametrize("shift", [-90.0, -150.0, -1e4, 90.0, 1e4])
@pytest.mark.parametrize("k", [1, 3, 5, 8])
def test_softmax_of_shifted_logits(mode, shift, k):
    """A softmax does not change when every logit is shifted; its gradient neither."""
    import torch

    T, H, E = 37, 128, 12
    rng, l, ids, g, x, w = _case(T, H, E, k, int(abs(shift)) + k)
    l = (l + np.float32(shift)).astype(np.float32)
    ids = np.argsort(-l, 1, kind="stable")[:, :k].astype(np.int32)
    want, err = _dl_limits(g[:T].astype(np.float64), l, ids, mode)
    got = _call(g, x, w, l, ids, mode, torch.zeros(E, device="cuda"))
    _check(got, want, err, values(x), values(w), f"{mode} {shift} {k}", "float32")


@pytest.mark.parametrize("mode", [m for m in MODES if m[0] and (m[2] or not m[1])])
@pytest.mark.parametrize("shift", [-90.0, -150.0])
def test_repeats_and_wrong_indices_beside_small_logits(mode, shift):
    """Lanes of repeated and wrong indices have no part in a token's maximum."""
    T, H, E = 3, 128, 10
    rng, l, _, g, x, w = _case(T, H, E, 3, 2)
    l = (l + np.float32(shift)).astype(np.float32)
    ids = np.array([[4, 2, 4], [-1, 10, 7], [9, 9, 9]], np.int32)
    want, err = np.zeros((T, E)), np.zeros((T, E))
    for t, mine in enumerate(([4, 2], [7], [9])):
        want[t : t + 1], err[t : t + 1] = _dl_limits(g[t : t + 1].astype(np.float64), l[t : t + 1], np.array([mine]), mode)
    _check(_call(g, x, w, l, ids, mode), want, err, values(x), values(w), str(mode), None)


@pytest.mark.parametrize("T,E,k", [(5, 12, 3), (33, 60, 8), (70, 300, 2), (600, 64, 4)])
@pytest.mark.parametrize("mode", [(False, True, False, True), (False, False, False, True), (False, True, False, False)])
def test_infinite_gradients_stay_infinite(T, E, k, mode):
    """An affinity's gradient that is infinite: dx of its token and dw of its expert are infinite with the sign of their factors, as a
    sum in fp32 has them, and the rest is as without it, another one of the largest magnitude included."""
    import torch

    H = 128
    rng, l, ids, g, x, w = _case(T, H, E, k, T + E)
    e, t, e2, t2 = int(ids[1, 0]), 1, int(ids[T - 1, k - 1]), T - 1
    if e2 == e:
        e2 = int(ids[T - 1, 0])
    assert e2 != e
    l[t2, e2] = 0.0  # (the slope's largest value, 1/4)
    g[t, e], g[t2, e2] = np.inf, -3.4e38
    xv, wv = values(x), values(w)
    assert (xv[t] != 0).all() and (wv[:, e] != 0).all()
    clean = g.copy()
    clean[t, e] = 0
    want, err = _dl_limits(clean[:T].astype(np.float64), l, ids, mode)
    d_x, d_w, d_b = _call(g, x, w, l, ids, mode, torch.zeros(E, device="cuda"))
    got_x, got_w, got_b = values(d_x), values(d_w), values(d_b)
    assert np.array_equal(got_x[t], np.sign(wv[:, e]) * np.inf) and np.array_equal(got_w[:, e], np.sign(xv[t]) * np.inf)
    assert np.isposinf(got_b[e])
    rows, cols = np.arange(T) != t, np.arange(E) != e
    fits = lambda a: np.where(np.abs(a) < 3.3e38, a, np.nan)
    wx, ww = want @ wv.T, xv.T @ want
    mx = 2.0**-8 * np.abs(wx) * (1 + 2.0**-7) + (E + 2) * 2.0**-24 * (np.abs(want) @ np.abs(wv.T)) + err @ np.abs(wv.T) + 2.0**-134
    mw = 2.0**-8 * np.abs(ww) * (1 + 2.0**-7) + (T + 2) * 2.0**-24 * (np.abs(xv.T) @ np.abs(want)) + np.abs(xv.T) @ err + 2.0**-134
    okx, okw = np.isfinite(fits(wx))[rows], np.isfinite(fits(ww))[:, cols]
    assert (np.abs(got_x - wx)[rows] <= mx[rows])[okx].all()
    assert (np.abs(got_w - ww)[:, cols] <= mw[:, cols])[okw].all()


@pytest.mark.parametrize("E,k", [(64, 8), (256, 8), (300, 5)])
def test_what_cancels_over_all_experts_does(E, k):
    """The softmax over all experts, whose dx is a product on the matrix cores: a part of w that all experts share leaves nothing."""
    import torch

    T, H = 40, 128
    mode = (True, True, False, False)
    rng, l, ids, g, x, w = _case(T, H, E, k, 1)
    small = (rng.integers(-8, 9, (H, E)) / 8).astype(np.float32)
    w = tensor(16.0 + small, "bfloat16")
    for m in (mode, (True, True, False, True)):
        want, err = _dl_limits(g[:T].astype(np.float64), l, ids, m)
        assert np.abs(want.sum(1)).max() < 1e-12
        _check(_call(g, x, w, l, ids, m), want, err, values(x), values(w), "cancels", None)


def test_the_same_call_gives_the_same_bits():
    import torch

    for T, H, E, k, mode in ((1999, 512, 60, 4, MODES[3]), (8192, 2176, 256, 8, MODES[3]), (3000, 256, 300, 3, MODES[1])):
        rng, l, ids, g, x, w = _case(T, H, E, k, 5)
        first = _call(g, x, w, l, ids, mode, torch.zeros(E, device="cuda"))
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, _call(g, x, w, l, ids, mode, torch.zeros(E, device="cuda"))))


# dw and dx in two launches from 16 M values of x on for up to 64 experts, from 6 M on beyond: every instance of either side
@pytest.mark.parametrize("T,H,E,k,softmax", [(8200, 2176, 8, 2, False), (8200, 2176, 60, 3, True), (8200, 2176, 64, 7, False), (7600, 2176, 64, 8, True),
                                             (3100, 2176, 65, 1, True), (3100, 2176, 128, 4, False), (3100, 2176, 128, 8, False), (2800, 2176, 128, 8, False),
                                             (3100, 2176, 200, 2, True), (3100, 2176, 256, 5, False), (3100, 2176, 257, 4, True), (3100, 2176, 512, 8, False)])
def test_one_launch_and_two(T, H, E, k, softmax):
    base.test_large_shapes_on_the_device(T, H, E, k, softmax)
