"""The products and norms that stand around a layer's routing, as they are timed.

A case is one pass through one operator: products of the rows of every expert with its weights (``grouped``, forward and
backward), products in 8-bit integers with a scale per token and per channel, dense or by expert (``int8``), the root-mean-square
norm with the residual's addition and an output in 8 bits with a scale per row (``norm``, forward and backward).  ``listed()``
are sizes of the repository's configurations and tests, ``draw()`` gives further cases of the same ranges.

Keys of a case: ``op``; ``direction`` (``forward`` | ``backward``); ``dtype`` of the rows (int8: of the result); T tokens, E
experts (0: a dense product), k experts per token, B rows that an expert's rows are filled up to a multiple of (1: none);
K length of a row and N columns of the product (norm: K alone); ``bias`` (dense int8); ``codes`` (norm: ``int8`` | ``e4m3``),
``residual`` (norm).

``run`` computes the plain form in 32 bits where ``own`` is false and calls the package where it is true.
"""

import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_DEFAULTS = dict(direction="forward", dtype="bf16", E=0, k=1, B=1, N=0, bias=False, codes="int8", residual=True)
_EPS = 1e-6
_SMALLEST = 2.0**-100  # the least magnitude that a row's largest value counts as


def _case(name, **kw):
    return dict(_DEFAULTS, name=name, **kw)


def listed():
    return [
        # gate/up of a decode batch of 8 tokens over Qwen3-MoE-shaped experts: the weights of the experts hit, read once
        _case("grouped_decode_8", op="grouped", T=8, E=128, k=8, K=2048, N=1536),
        # the same layer's gate/up of a prompt, experts popular and unpopular
        _case("grouped_8192", op="grouped", T=8192, E=128, k=8, K=2048, N=1536),
        # gate/up over the few large experts of the Mixtral shape, fp16
        _case("grouped_fp16_4096", op="grouped", dtype="fp16", T=4096, E=8, k=2, K=4096, N=28672),
        # the backward pass of the down product of the bf16 layer of few large experts
        _case("grouped_bwd_4096", op="grouped", direction="backward", T=4096, E=8, k=2, K=4096, N=2048),
        # a backward pass at sizes that fit no tile, experts filled up to blocks of 32 rows
        _case("grouped_bwd_fp16_1999", op="grouped", direction="backward", dtype="fp16", T=1999, E=60, k=4, B=32, K=1030, N=515),
        # one token through a projection as wide as the DeepSeek-V3-shaped expert's gate/up
        _case("int8_decode_1", op="int8", T=1, K=7168, N=4096),
        # a prompt of odd length at odd sizes, with a bias, fp16 results
        _case("int8_fp16_1999", op="int8", dtype="fp16", T=1999, K=1030, N=515, bias=True),
        # gate/up of the benchmark's prompt over DeepSeek-V3-shaped experts in 8-bit integers
        _case("int8_grouped_8192", op="int8", T=8192, E=256, k=8, K=7168, N=4096),
        # a decode batch ahead of such a layer
        _case("norm_decode_8", op="norm", T=8, K=7168),
        # the benchmark's prompt ahead of such a layer
        _case("norm_8192", op="norm", T=8192, K=7168),
        # an odd number of tokens at an odd size, fp32, into 8-bit floating point
        _case("norm_fp32_1999", op="norm", dtype="fp32", T=1999, K=1030, codes="e4m3"),
        # a training step's gradient of the norm over the Mixtral-shaped prompt
        _case("norm_bwd_4096", op="norm", direction="backward", T=4096, K=4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _length(rng, lo, hi, step):
    """A row's length: a multiple of ``step``, or in a fifth of the cases any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.2 else max(step, n // step * step)


def draw(rng):
    """From one token to 8192, sizes over the range of the listed ones, any number of experts; no case moves more bytes or
    computes more than the listed ones of its operator."""
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = max(b, w["bytes"]), max(f, w["flops"])
    while True:
        op = rng.choice(("grouped", "grouped", "int8", "int8", "norm"))
        c = dict(_DEFAULTS, op=op, T=_log_int(rng, 1, 8192), K=_length(rng, 64, 7168, 64))
        if op == "norm":
            c["direction"] = rng.choice(("forward", "forward", "backward"))
            c["dtype"] = rng.choice(("bf16", "bf16", "fp16", "fp32"))
            c["codes"] = rng.choice(("int8", "int8", "e4m3"))
            c["residual"] = rng.random() < 0.7
        else:
            c["N"] = _length(rng, 64, 28672, 64)
            if op == "grouped":
                c["direction"] = rng.choice(("forward", "backward"))
                c["dtype"] = rng.choice(("bf16", "fp16"))
            else:
                c["dtype"] = rng.choice(("bf16", "bf16", "fp16", "fp32"))
            if op == "grouped" or rng.random() < 0.5:
                c["E"] = rng.choice((1, 4, 8, 16, 32, 60, 64, 128, 160, 256))
                c["k"] = rng.randint(1, min(8, c["E"]))
                c["B"] = rng.choice((1, 1, 1, 16, 32, 128))
            else:
                c["bias"] = rng.random() < 0.5
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1]:
            return c


def _rows(c):
    """Rows of a case: one per routed pair, and what the worst routing fills up."""
    if not c["E"]:
        return c["T"]
    return (math.ceil((c["T"] * c["k"] - (c["E"] - 1)) / c["B"]) + c["E"] - 1) * c["B"]


# ---- inputs ---------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    c = dict(case)
    if own:
        pkg = os.path.abspath("nki-library_amd")  # (run from the repository's root)
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from nkilib import _native

        _native.lib()
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = _DT[c["dtype"]]
    T, E, K, N = (c[n] for n in ("T", "E", "K", "N"))

    def randn(*shape, std=1.0, dtype=dt):
        out = torch.empty(shape, dtype=dtype, device=dev)
        flat, part = out.view(-1), 1 << 28
        for i in range(0, flat.numel(), part):
            n = min(part, flat.numel() - i)
            flat[i : i + n] = torch.randn(n, generator=g, device=dev).mul_(std)
        return out

    def codes(*shape):
        """Integers as rows of normal values become whose largest is 127."""
        out = torch.empty(shape, dtype=torch.int8, device=dev)
        flat, part = out.view(-1), 1 << 28
        for i in range(0, flat.numel(), part):
            n = min(part, flat.numel() - i)
            flat[i : i + n] = torch.randn(n, generator=g, device=dev).mul_(32.0).round_().clamp_(-127, 127)
        return out

    st = {"case": c}
    S = _rows(c)
    if E:
        # popular and unpopular experts, as a router has them; rows of an expert beside each other, experts ascending
        logits = torch.randn((T, E), generator=g, device=dev) + 0.5 * torch.randn((E,), generator=g, device=dev)
        counts = torch.bincount(logits.topk(c["k"], dim=1).indices.reshape(-1), minlength=E)
        filled = (counts + c["B"] - 1) // c["B"] * c["B"]
        st["offsets"] = torch.cat((filled.new_zeros(1), filled.cumsum(0))).to(torch.int32)
        st["offsets_host"] = st["offsets"].tolist()
        # zeros in the rows that an expert is filled up with, and behind the last expert's
        row = torch.arange(S, device=dev)
        e = torch.searchsorted(st["offsets"][1:].long(), row, right=True).clamp_(max=E - 1)
        routed = row - st["offsets"][e].long() < counts[e]
    if c["op"] == "grouped":
        st["x"] = randn(S, K).mul_(routed[:, None])
        st["w"] = randn(E, K, N, std=K**-0.5)
        if c["direction"] == "backward":
            st["d_out"] = randn(S, N).mul_(routed[:, None])
    elif c["op"] == "int8":
        st["x"] = codes(S, K)
        st["x_scale"] = torch.rand(S, generator=g, device=dev) * 0.02 + 0.02
        st["w"] = codes(*((E,) if E else ()), N, K)
        st["w_scale"] = (torch.rand((*((E,) if E else ()), N), generator=g, device=dev) + 1.0) * (0.03 * K**-0.5)
        if E:
            st["x"].mul_(routed[:, None])
        st["bias"] = randn(N) if c["bias"] else None
    else:
        # a few channels are far larger than the others, as in a model's residual stream
        wide = 1.0 + 20.0 * (torch.rand(K, generator=g, device=dev) < 0.004)
        st["x"] = (randn(T, K, dtype=torch.float32) * wide).to(dt)
        st["gamma"] = (1.0 + 0.2 * randn(K, dtype=torch.float32)).to(dt)
        if c["direction"] == "backward":
            st["d_y"] = randn(T, K)
            st["d_res"] = randn(T, K) if c["residual"] else None
        else:
            st["res"] = (randn(T, K, dtype=torch.float32) * wide).to(dt) if c["residual"] else None
    return st


# ---- plain forms ----------------------------------------------------------------------------------------------------


def _groups(st):
    o = st["offsets_host"]
    return [(e, o[e], o[e + 1]) for e in range(len(o) - 1)]


def _plain_grouped(st):
    x, w = st["x"], st["w"]
    if st["case"]["direction"] == "forward":
        out = x.new_zeros((x.shape[0], w.shape[2]))
        for e, a, b in _groups(st):
            if b > a:
                out[a:b] = (x[a:b].float() @ w[e].float()).to(x.dtype)
        return out
    d = st["d_out"]
    d_x, d_w = torch.zeros_like(x), torch.zeros_like(w)
    for e, a, b in _groups(st):
        if b > a:
            df = d[a:b].float()
            d_x[a:b] = (df @ w[e].float().t()).to(x.dtype)
            d_w[e] = (x[a:b].float().t() @ df).to(w.dtype)
    return d_x, d_w


def _int8_sums(x, w):
    """Products of codes: sums of 1024 of them at a time are whole numbers below 2^24, which 32 bits hold exactly."""
    total = None
    for i in range(0, x.shape[1], 1024):
        part = x[:, i : i + 1024].float() @ w[:, i : i + 1024].float().t()
        total = part.double() if total is None else total.add_(part)
    return total.float()


def _plain_int8(st):
    dt = _DT[st["case"]["dtype"]]
    x, w, xs, ws = st["x"], st["w"], st["x_scale"], st["w_scale"]
    if st["case"]["E"]:
        out = torch.zeros((x.shape[0], w.shape[1]), dtype=dt, device=x.device)
        for e, a, b in _groups(st):
            if b > a:
                out[a:b] = (_int8_sums(x[a:b], w[e]) * xs[a:b, None] * ws[e]).to(dt)
        return out
    out = _int8_sums(x, w) * xs[:, None] * ws
    if st["bias"] is not None:
        out = out + st["bias"].float()
    return out.to(dt)


def _inverse_rms(x):
    """1 / sqrt(mean of squares + eps) of rows in 32 bits; the sum in 64."""
    return torch.rsqrt(x.double().square().mean(1, keepdim=True) + _EPS).float()


def _plain_norm(st):
    c, dt = st["case"], st["x"].dtype
    x = st["x"].float()
    if c["direction"] == "backward":
        n = x * _inverse_rms(x)
        dy = st["d_y"].float()
        dn = dy * st["gamma"].float()
        d_x = (dn - n * (dn * n).mean(1, keepdim=True)) * _inverse_rms(x)
        if st["d_res"] is not None:
            d_x = d_x + st["d_res"].float()
        return d_x.to(dt), (dy * n).sum(0, dtype=torch.float64).to(dt)
    if st["res"] is not None:
        x = (x + st["res"].float()).to(dt).float()
    y = x * _inverse_rms(x) * st["gamma"].float()
    most = 127.0 if c["codes"] == "int8" else 448.0
    largest = y.abs().amax(1, keepdim=True).clamp(min=_SMALLEST)
    m = torch.full_like(largest, most)  # (a division by a number would be a product with its rounded inverse)
    q = y * (m / largest)
    q = torch.round(q) if c["codes"] == "int8" else q.clamp(-most, most).to(torch.float8_e4m3fn).float()
    values = (q * (largest / m)).to(torch.bfloat16)
    return (values, x.to(dt)) if st["res"] is not None else values


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    if not own:
        return {"grouped": _plain_grouped, "int8": _plain_int8, "norm": _plain_norm}[c["op"]](state)
    if c["op"] == "grouped":
        from nkilib.core.moe.grouped_matmul import grouped_matmul, grouped_matmul_bwd

        if c["direction"] == "backward":
            return grouped_matmul_bwd(state["d_out"], state["x"], state["w"], state["offsets"])
        return grouped_matmul(state["x"], state["w"], state["offsets"])
    if c["op"] == "int8":
        from nkilib.core.int8_matmul import grouped_int8_matmul, int8_matmul

        args = (state["x"], state["x_scale"], state["w"], state["w_scale"])
        if c["E"]:
            return grouped_int8_matmul(*args, state["offsets"], out_dtype=_DT[c["dtype"]])
        return int8_matmul(*args, bias=state["bias"], out_dtype=_DT[c["dtype"]])
    from nkilib.core.rmsnorm import dequantize_rows, rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

    if c["direction"] == "backward":
        return rmsnorm_quant_rows_bwd(state["d_y"], state["x"], state["gamma"], eps=_EPS, d_residual=state["d_res"])
    out = rmsnorm_quant_rows(state["x"], state["gamma"], eps=_EPS, residual=state["res"],
                             code_dtype=torch.int8 if c["codes"] == "int8" else torch.float8_e4m3fn)
    values = dequantize_rows(out[0], out[1], torch.bfloat16)
    return (values, out[2]) if state["res"] is not None else values


# ---- the least work ---------------------------------------------------------------------------------------------------


def work(case):
    c = case
    T, E, k, K, N = (c[n] for n in ("T", "E", "k", "K", "N"))
    es, back = _SIZE[c["dtype"]], c["direction"] == "backward"
    if c["op"] == "norm":
        if back:
            return {"bytes": es * T * K * (4 if c["residual"] else 3) + 2 * es * K, "flops": 12 * T * K}
        return {"bytes": es * (T * K * (3 if c["residual"] else 1) + K) + 2 * T * K, "flops": 7 * T * K}
    S, routed = _rows(c), T * k if E else T
    # weights of the experts that tokens choose (all of them alike)
    hit = E * (1.0 - (1.0 - k / E) ** T) if E else 1.0
    if c["op"] == "int8":
        return {"bytes": int(routed * (K + 4) + hit * N * (K + 4) + S * N * es + (es * N if c["bias"] else 0)), "flops": 2 * routed * K * N}
    if back:
        return {"bytes": int(es * (routed * (K + N) + S * K + (hit + E) * K * N)), "flops": 4 * routed * K * N}
    return {"bytes": int(es * (routed * K + S * N + hit * K * N)), "flops": 2 * routed * K * N}


# ---- in 64 bits -------------------------------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["op"] == "norm":
        return _exact_norm(st)
    x, w = st["x"], st["w"]
    bounds = [0, x.shape[0]] if not c["E"] else st["offsets_host"]
    w = w if c["E"] else w[None]
    # (the weights' columns by parts: an expert in 64 bits takes four times its bytes)
    if c["op"] == "int8":
        ws = st["w_scale"] if c["E"] else st["w_scale"][None]
        out = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device=x.device)
        for e in range(w.shape[0]):
            r = slice(bounds[e], bounds[e + 1])
            if r.stop > r.start:
                scaled = x[r].double() * st["x_scale"][r].double()[:, None]
                out[r] = torch.mm(scaled, (w[e].double() * ws[e].double()[:, None]).t().contiguous())
        return out + st["bias"].double() if st["bias"] is not None else out
    if c["direction"] == "forward":
        out = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64, device=x.device)
        for e in range(w.shape[0]):
            r = slice(bounds[e], bounds[e + 1])
            if r.stop > r.start:
                out[r] = torch.mm(x[r].double(), w[e].double())
        return out
    d_x = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    d_w = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for e in range(w.shape[0]):
        r = slice(bounds[e], bounds[e + 1])
        if r.stop > r.start:
            d = st["d_out"][r].double()
            d_x[r] = torch.mm(d, w[e].double().t().contiguous())
            d_w[e] = torch.mm(x[r].double().t().contiguous(), d)
    return d_x, d_w


def _exact_norm(st):
    c, K = st["case"], st["case"]["K"]
    x, gamma = st["x"].double(), st["gamma"].double()
    if c["direction"] == "backward":
        x.requires_grad_()
        gamma.requires_grad_()
        y = x / torch.sqrt((x * x).sum(1, keepdim=True) / K + _EPS) * gamma
        d_x, d_gamma = torch.autograd.grad(y, (x, gamma), st["d_y"].double())
        return d_x + (st["d_res"].double() if st["d_res"] is not None else 0), d_gamma
    if st["res"] is not None:
        x = (x + st["res"].double()).to(st["x"].dtype).double()  # (the stream is kept in its type, and that is what is normalised)
    y = x / torch.sqrt((x * x).sum(1, keepdim=True) / K + _EPS) * gamma
    most = 127 if c["codes"] == "int8" else 448
    scale = torch.clamp(y.abs().max(1, keepdim=True).values, min=_SMALLEST) / most
    v = y / scale
    if c["codes"] == "int8":
        q = torch.floor(v + 0.5)
    else:  # to the nearest of 8 values per power of two, ties to the even one; 2^-9 apart below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3)
        q = torch.round(v / step) * step
    return (q * scale, x) if st["res"] is not None else q * scale
