"""What the tests of the products by expert share: groups of rows, and the products of whole groups in 64 bits."""

import numpy as np
import torch

from train_helpers import HALF, TINY


def offsets_of(counts, ahead=0):
    return np.concatenate(([ahead], ahead + np.cumsum(counts))).astype(np.int32)


def taken(offsets, S):
    """Offsets as the operators take them: into [0, S], never falling."""
    return np.maximum.accumulate(np.clip(np.asarray(offsets, dtype=np.int64), 0, S))


def groups(offsets, S):
    o = taken(offsets, S)
    return [(e, int(o[e]), int(o[e + 1])) for e in range(len(o) - 1)]


def products(x, w, offsets):
    """x [S, K], w [E, K, N] (any type) -> sums in 64 bits and the sums of their terms' magnitudes."""
    out = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    for e, a, b in groups(offsets, x.shape[0]):
        if b > a:
            xe, we = x[a:b].double(), w[e].double()
            out[a:b] = xe @ we
            mag[a:b] = xe.abs() @ we.abs()
    return out, mag


def outer_products(x, d, offsets):
    """x [S, K], d [S, N] -> every group's sums of x[s, k] d[s, n], and of their magnitudes."""
    E = len(offsets) - 1
    out = torch.zeros((E, x.shape[1], d.shape[1]), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    for e, a, b in groups(offsets, x.shape[0]):
        if b > a:
            xe, de = x[a:b].double().t().contiguous(), d[a:b].double()
            out[e] = xe @ de
            mag[e] = xe.abs() @ de.abs()
    return out, mag


def assert_near(got, want, mag, steps, what=""):
    """A sum of terms that are exact products, taken in 32 bits (at most a rounding of 2^-24 of the magnitudes per step) and rounded
    once to got's type."""
    name = str(got.dtype).split(".")[1]
    g = got.double()
    limit = HALF[name] * want.abs() * (1 + 2.0**-7) + steps * 2.0**-24 * mag * (1 + 2.0**-7) + TINY[name]
    bad = ~((g - want).abs() <= limit)
    bad &= ~(torch.isnan(g) & torch.isnan(want)) & ~(g == want)
    assert got.shape == want.shape, what
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                                 f"{g[bad][0].item()} for {want[bad][0].item()} within {limit[bad][0].item()}")
