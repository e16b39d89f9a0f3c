"""The operators of a routed layer's training in 64 bits: tokens into block order and back, the gated activation with its
inputs kept in 8 bits, the gradient of the router.  Oracle: test infrastructure only.

The reference has no counterpart of these; each function is the operator's formula, written for clarity.  Their gradients
are pinned by central differences (``tests/test_oracle_train.py``).
"""

import math

import numpy as np

from .numerics import E4M3FN_TABLE, e4m3fn_encode


def slots_of(tp2id, T):
    """List of ascending slots per token."""
    out = [[] for _ in range(T)]
    for s, t in enumerate(np.asarray(tp2id).tolist()):
        if 0 <= t < T:
            out[t].append(s)
    return out


def token_slots(tp2id, T, k):
    """[T, 1 + k]: count, ascending slots, -1."""
    out = np.full((T, 1 + k), -1, np.int32)
    for t, l in enumerate(slots_of(tp2id, T)):
        out[t, 0] = len(l)
        out[t, 1 : 1 + min(k, len(l))] = l[:k]
    return out


def permute(x, tp2id):
    T = x.shape[0]
    out = np.zeros((len(tp2id), x.shape[1]), x.dtype)
    for s, t in enumerate(np.asarray(tp2id).tolist()):
        if 0 <= t < T:
            out[s] = x[t]
    return out


def combine(y, aff, tp2id, b2e, B, T):
    """(sum, sum of the magnitudes of its terms) [T, H]; aff None: weights of one."""
    out = np.zeros((T, y.shape[1]))
    mag = np.zeros_like(out)
    for t, l in enumerate(slots_of(tp2id, T)):
        for s in l:
            w = 1.0
            if aff is not None:
                e = int(b2e[s // B])
                if not 0 <= e < aff.shape[1]:
                    continue
                w = float(aff[t, e])
            out[t] += w * y[s].astype(np.float64)
            mag[t] += np.abs(w * y[s].astype(np.float64))
    return out, mag


def combine_bwd(d_out, y, aff, tp2id, b2e, B):
    """d_y, d_aff, sum of the magnitudes of d_aff's terms."""
    T = d_out.shape[0]
    d_y = np.zeros(y.shape)
    d_aff = np.zeros(aff.shape)
    mag = np.zeros(aff.shape)
    for t, l in enumerate(slots_of(tp2id, T)):
        for s in l:
            e = int(b2e[s // B])
            if not 0 <= e < aff.shape[1]:
                continue
            d_y[s] = float(aff[t, e]) * d_out[t].astype(np.float64)
            terms = d_out[t].astype(np.float64) * y[s].astype(np.float64)
            d_aff[t, e] += terms.sum()
            mag[t, e] += np.abs(terms).sum()
    return d_y, d_aff, mag


def record(x):
    """float32 rows [..., I] -> (codes uint8 [..., I], scales uint8 [..., ceil(I/32)])."""
    x = np.ascontiguousarray(x, np.float32)
    I = x.shape[-1]
    codes = np.zeros(x.shape, np.uint8)
    scales = np.zeros((*x.shape[:-1], -(-I // 32)), np.uint8)
    for g in range(scales.shape[-1]):
        part = x[..., 32 * g : 32 * g + 32].astype(np.float64)
        finite = np.where(np.isfinite(part), np.abs(part), 0.0)
        amax = finite.max(-1)
        m, ex = np.frexp(amax)  # amax = m 2^ex, m in [0.5, 1)
        s = ex - 9 + (m > 0.875)  # the smallest s with amax <= 448 * 2^s (448 = 0.875 * 2^9)
        s = np.where(amax == 0, -127, np.maximum(s, -127))
        scales[..., g] = s + 127
        v = part * np.exp2(-s.astype(np.float64))[..., None]
        c = e4m3fn_encode(np.where(np.isfinite(v), v, 0.0).astype(np.float32))
        bad = ~np.isfinite(part)
        codes[..., 32 * g : 32 * g + 32] = np.where(bad, np.where(np.signbit(part), 0xFF, 0x7F), c)
    return codes, scales


def record_values(codes, scales):
    s = np.exp2(np.repeat(scales.astype(np.float64) - 127, 32, axis=-1)[..., : codes.shape[-1]])
    return E4M3FN_TABLE[codes].astype(np.float64) * s


def act(x, kind):
    """(act(x), act'(x)) in 64 bits; kind: silu, gelu, gelu_tanh, swish."""
    x = np.asarray(x, np.float64)
    if kind == "gelu":
        phi = 0.5 * np.vectorize(math.erfc, otypes=[float])(-x / math.sqrt(2))
        return x * phi, phi + x * np.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        z = c * (x + 0.044715 * x**3)
        s = 1 / (1 + np.exp(-2 * z))  # 0.5 (1 + tanh z), which loses everything of a large negative z
        return x * s, s + 2 * x * s * (1 - s) * c * (1 + 3 * 0.044715 * x * x)
    a = 1.702 if kind == "swish" else 1.0
    s = 1 / (1 + np.exp(-a * x))
    return x * s, s * (1 + a * x * (1 - s))


def clamp_glu(gate, up, clamps):
    """clamps: (gate upper, gate lower, up upper, up lower), None where there is none."""
    gh, gl, uh, ul = clamps
    gate = gate if gh is None else np.where(gate > gh, gh, gate)
    gate = gate if gl is None else np.where(gate < gl, gl, gate)
    up = up if uh is None else np.where(up > uh, uh, up)
    up = up if ul is None else np.where(up < ul, ul, up)
    return gate, up


def recorded_limit(limit, scales, I):
    """What the record of a clamped value holds, per value of rows [..., I] with `scales` [..., ceil(I/32)]: the limit as one of its
    group's e4m3 values; the limit itself where it lies beyond all of them (no value of the group met it)."""
    s = np.exp2(np.repeat(scales.astype(np.float64) - 127, 32, axis=-1)[..., :I])
    v = limit / s
    code = e4m3fn_encode(np.clip(v, -448, 448).astype(np.float32))
    return np.where(np.abs(v) <= 448, E4M3FN_TABLE[code].astype(np.float64) * s, limit)


def bf16_value(x):
    u = np.asarray(x, np.float32).reshape(1).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> np.uint64(16)) & np.uint64(1))) & np.uint64(0xFFFF0000)
    return float(u.astype(np.uint32).view(np.float32)[0])


def reaches(v, limit, upper, scales=None):
    """Where recorded values are at their clamp or beyond.  With `scales`, at what the record holds of it: of the limit or of its
    bf16 (the layer's checkpoint), whichever lies further inside.  Without, limits that every group holds."""
    if limit is None:
        return np.zeros(v.shape, bool)
    at = [limit] if scales is None else [recorded_limit(l, scales, v.shape[-1]) for l in (limit, bf16_value(limit))]
    return v >= np.minimum.reduce(at) if upper else v <= np.maximum.reduce(at)


def glu_bwd(gate, up, d, kind, clamps=(None,) * 4, scales=None):
    """(d_gate, d_up, h) at the recorded values; zero at and beyond a clamp.  scales: the record's, [..., 2, ceil(I/32)]."""
    g, u = clamp_glu(gate, up, clamps)
    gh, gl, uh, ul = clamps
    sg, su = (None, None) if scales is None else (scales[..., 0, :], scales[..., 1, :])
    in_g = ~(reaches(gate, gh, True, sg) | reaches(gate, gl, False, sg))
    in_u = ~(reaches(up, uh, True, su) | reaches(up, ul, False, su))
    a, da = act(g, kind)
    return np.where(in_g, d * u * da, 0.0), np.where(in_u, d * a, 0.0), a * u


def router_affinities(logits, ids, softmax, pre_norm, norm_topk):
    """What the router makes of logits [T, E] and its choice [T, k], zero outside the choice."""
    T, E = logits.shape
    l = logits.astype(np.float64)
    on = np.zeros((T, E), bool)
    np.put_along_axis(on, ids, True, 1)
    if softmax:
        m = l if pre_norm else np.where(on, l, -np.inf)
        p = np.exp(m - m.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 1 / (1 + np.exp(-l))
    p = np.where(on, p, 0.0)
    return p / p.sum(1, keepdims=True) if pre_norm and norm_topk else p


def router_d_logits(d_aff, logits, ids, softmax, pre_norm, norm_topk, masked=True):
    """Gradient of the logits from that of the affinities.  masked False: affinities of the experts outside the choice were
    handed out too (the router's full table, without pre_norm's division)."""
    l = logits.astype(np.float64)
    on = np.zeros(l.shape, bool)
    np.put_along_axis(on, ids, True, 1)
    everyone = pre_norm and not norm_topk
    part = on if (masked or not everyone) else np.ones_like(on)
    g = np.where(part, d_aff, 0.0)
    if softmax:
        m = l if everyone else np.where(on, l, -np.inf)
        p = np.exp(m - m.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        return p * (g - (g * p).sum(1, keepdims=True))
    s = 1 / (1 + np.exp(-l))
    if pre_norm and norm_topk:
        total = np.where(on, s, 0.0).sum(1, keepdims=True)
        g = np.where(on, (g - (g * s).sum(1, keepdims=True) / total) / total, 0.0)
    return g * s * (1 - s)
