"""The oracle of the training operators: gradients against central differences, the 8-bit record against a search."""

import numpy as np
import pytest

from oracle import blocks as ob
from oracle import train as ot
from oracle.numerics import E4M3FN_TABLE


def _case(seed, T=7, E=5, k=3, B=4, H=6):
    rng = np.random.default_rng(seed)
    mask = np.zeros((T, E))
    for t in range(T):
        mask[t, rng.permutation(E)[:k]] = 1
    N = ob.get_n_blocks(T, k, E, B)
    tp2id, b2e, _ = ob.build_token_blocks(mask, B, N)
    return rng, tp2id, b2e, B, rng.standard_normal((N * B, H)), rng.random((T + 1, E)), T


def _difference(f, x, h=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + h
        up = f()
        x[i] = keep - h
        g[i] = (up - f()) / (2 * h)
        x[i] = keep
    return g


def test_permute_and_combine_gradients_against_differences():
    rng, tp2id, b2e, B, y, aff, T = _case(1)
    r = rng.standard_normal((T, y.shape[1]))
    loss = lambda: (ot.combine(y, aff, tp2id, b2e, B, T)[0] * r).sum()
    d_y, d_aff, _ = ot.combine_bwd(r, y, aff, tp2id, b2e, B)
    assert np.allclose(d_y, _difference(loss, y), atol=1e-7) and np.allclose(d_aff, _difference(loss, aff), atol=1e-7)
    x = rng.standard_normal((T, y.shape[1]))
    r = rng.standard_normal(y.shape)
    got = ot.combine(r, None, tp2id, b2e, B, T)[0]
    assert np.allclose(got, _difference(lambda: (ot.permute(x, tp2id) * r).sum(), x), atol=1e-7)


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "swish"])
def test_glu_gradient_against_differences(kind):
    rng = np.random.default_rng(2)
    g, u, d = rng.standard_normal((3, 5, 9)) * 2
    clamps = (1.5, None, 1.0, -1.0)
    f = lambda: (d * np.prod([ot.act(ot.clamp_glu(g, u, clamps)[0], kind)[0], ot.clamp_glu(g, u, clamps)[1]], 0)).sum()
    dg, du, _ = ot.glu_bwd(g, u, d, kind, clamps)
    assert np.allclose(dg, _difference(f, g), atol=1e-6) and np.allclose(du, _difference(f, u), atol=1e-6)


def test_record_takes_the_smallest_scale_and_the_nearest_value():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((40, 70)) * np.exp2(rng.integers(-130, 120, (40, 1)))).astype(np.float32)
    x[0] = 0
    x[1, :32] = 448.0  # a border: 448 itself needs no larger scale
    x[2, :32] = np.nextafter(np.float32(448.0), np.float32(500))
    x[3, 5], x[3, 40], x[3, 50] = np.inf, np.nan, -np.inf
    codes, scales = ot.record(x)
    assert scales[1, 0] == 127 and scales[2, 0] == 128 and scales[0].max() == 0 and codes[0].max() == 0
    assert codes[3, 5] == 0x7F and codes[3, 50] == 0xFF
    v = ot.record_values(codes, scales)
    finite = E4M3FN_TABLE[np.isfinite(E4M3FN_TABLE)].astype(np.float64)
    for r in range(40):
        for c in range(70):
            if not np.isfinite(x[r, c]):
                assert np.isnan(v[r, c])
                continue
            group = x[r, c // 32 * 32 : c // 32 * 32 + 32]
            amax = np.abs(group[np.isfinite(group)]).max().astype(np.float64)
            s = np.exp2(float(scales[r, c // 32]) - 127)
            assert amax <= 448 * s and (scales[r, c // 32] == 0 or amax > 224 * s)
            assert abs(v[r, c] - x[r, c]) == np.abs(finite * s - x[r, c]).min()


@pytest.mark.parametrize("limit", [7.0, 7.2, 10.5, 20.6, 6.2, 1.1, 0.9, -0.7, 7.2503, 0.0, 1e-3, 500.0])
@pytest.mark.parametrize("bf16", [False, True])
def test_clamped_values_are_clamped_in_the_record(limit, bf16):
    """Values clamped at the limit (kept as bf16 between, or not) lie at their clamp in the record, those far inside do not."""
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((50, 160)) * np.exp2(rng.integers(-4, 9, (50, 1)))).astype(np.float32)
    for upper in (True, False):
        v = np.minimum(x, np.float32(limit)) if upper else np.maximum(x, np.float32(limit))
        if bf16:
            v = np.vectorize(ot.bf16_value, otypes=[np.float32])(v)
        codes, scales = ot.record(v)
        rec = ot.record_values(codes, scales)
        got = ot.reaches(rec, float(np.float32(limit)), upper, scales)
        out = x >= np.float32(limit) if upper else x <= np.float32(limit)
        assert got[out].all()
        far = abs(limit) / 8 + np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, axis=1)[:, : x.shape[1]] / 512
        inside = x < limit - far if upper else x > limit + far
        assert inside.any() and not got[inside].any()


@pytest.mark.parametrize("softmax", [True, False])
@pytest.mark.parametrize("pre_norm,norm", [(True, True), (True, False), (False, False)])
def test_router_gradient_against_differences(softmax, pre_norm, norm):
    rng = np.random.default_rng(4)
    l, r = rng.standard_normal((2, 6, 9))
    ids = np.argsort(-l, 1)[:, :4]
    f = lambda: (ot.router_affinities(l, ids, softmax, pre_norm, norm) * r).sum()
    assert np.allclose(ot.router_d_logits(r, l, ids, softmax, pre_norm, norm), _difference(f, l), atol=1e-7)


def test_router_gradient_of_the_full_table_against_differences():
    rng = np.random.default_rng(5)
    l, r = rng.standard_normal((2, 6, 9))
    ids = np.argsort(-l, 1)[:, :4]
    soft = lambda: (np.exp(l) / np.exp(l).sum(1, keepdims=True) * r).sum()
    assert np.allclose(ot.router_d_logits(r, l, ids, True, True, False, masked=False), _difference(soft, l), atol=1e-7)
    sig = lambda: (r / (1 + np.exp(-l))).sum()
    assert np.allclose(ot.router_d_logits(r, l, ids, False, True, False, masked=False), _difference(sig, l), atol=1e-7)
