"""What the tests of the training operators share: tables, types and the bounds that their results keep to.

``bound``: a value computed in 32 bits from ``terms`` magnitudes and rounded once to a type differs from the value in 64 bits by
at most half a step of the type relative to the value, the steps of the sum (2^-24 of the magnitudes each), and half of the
type's smallest subnormal.
"""

import numpy as np

from oracle import blocks as ob

HALF = {"bfloat16": 2.0**-8, "float16": 2.0**-11, "float32": 2.0**-24}
TINY = {"bfloat16": 2.0**-134, "float16": 2.0**-25, "float32": 2.0**-150}


def table(rng, T, E, k, B, skip_token=False, N=None):
    mask = np.zeros((T, E))
    for t in range(T):
        mask[t, rng.permutation(E)[:k]] = 1
    N = N or ob.get_n_blocks(T, k, E, B)
    tp2id, b2e, _ = ob.build_token_blocks(mask, B, N, skip_token=skip_token)
    return tp2id, b2e, N


def tensor(a, dtype="float32", dev="cuda:0"):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).to(dev).to(getattr(torch, dtype))


def values(t):
    """A tensor's own (rounded) values in 64 bits."""
    return t.detach().double().cpu().numpy()


def bound(want, magnitude, dtype, steps):
    return HALF[dtype] * np.abs(want) * (1 + 2.0**-7) + steps * 2.0**-24 * magnitude + TINY[dtype]


def assert_within(got, want, limit, what=""):
    got = values(got) if not isinstance(got, np.ndarray) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    err = np.abs(got - want)
    bad = ~((err <= limit) | np.isnan(want) | (got == want))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}"
