"""The operators of a routed layer's training and of experts that a program multiplies itself, as they are timed.

A case is one pass through one operator: tokens put into the order of the block table (``permute``) and back with the
routing weights applied (``combine``), the gated activation with its inputs kept in 8 bits for the backward pass
(``glu``), the gradient of the router (``router``).  ``listed()`` are sizes of the repository's configurations and
tests, ``draw()`` gives further cases of the same ranges.

Keys of a case: ``op``; ``direction`` (``forward`` | ``backward``, for ``glu`` also ``pack``: the 8-bit record made of the
checkpoint that ``moe_cte`` returns); ``dtype`` of the activations; T tokens, H hidden size, I intermediate size, E
experts, k experts per token, B block size; ``act``, ``clamps`` (glu); ``mode`` (router: how affinities come of logits).

``run`` computes the plain form in 32 bits where ``own`` is false and calls the package where it is true.
"""

import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_DEFAULTS = dict(direction="forward", dtype="bf16", H=0, I=0, B=128, act="silu", clamps=False, mode="", bias=False)
# gate <= 7, -7 <= up <= 7: the clamp triple of the models that clamp
_CLAMP = 7.0
_MODES = ("softmax_norm", "softmax", "sigmoid_norm", "sigmoid", "chosen_softmax", "chosen_sigmoid")


def _case(name, **kw):
    return dict(_DEFAULTS, name=name, **kw)


def listed():
    return [
        # a decode batch of 8 tokens sorted for experts of a model served in bf16: compact order (blocks of one slot), all latency
        _case("permute_decode_8", op="permute", T=8, H=7168, E=256, k=8, B=1),
        # the DeepSeek-V3-shaped prompt of the benchmark, sorted into blocks of 128
        _case("permute_8192", op="permute", T=8192, H=7168, E=256, k=8),
        # gradient of a training step's tokens from the gradients of their slots, Qwen3-MoE shape
        _case("permute_bwd_8192", op="permute", direction="backward", T=8192, H=2048, E=128, k=8),
        # the same decode batch of 8 tokens brought back, weights applied
        _case("combine_decode_8", op="combine", T=8, H=7168, E=256, k=8, B=1),
        # an odd number of tokens at a hidden size that is no multiple of a vector, fp32, top-4 of 60
        _case("combine_fp32_1999", op="combine", dtype="fp32", T=1999, H=1030, E=60, k=4, B=32),
        # the backward pass of the benchmark's prompt: gradients of the slots and of the routing weights
        _case("combine_bwd_8192", op="combine", direction="backward", T=8192, H=7168, E=256, k=8),
        # forward of a training step over Mixtral-shaped experts, fp16, the activations kept in 8 bits
        _case("glu_fp16_4096", op="glu", dtype="fp16", T=4096, I=14336, E=8, k=2),
        # what moe_cte returned for the smallest prefill, packed
        _case("glu_pack_256", op="glu", direction="pack", T=256, I=1024, E=8, k=2),
        # the backward pass over DeepSeek-V3-shaped experts, from the 8-bit record
        _case("glu_bwd_8192", op="glu", direction="backward", T=8192, I=2048, E=256, k=8),
        # a short sequence through the router of the Qwen3-MoE shape
        _case("router_128", op="router", direction="backward", T=128, H=2048, E=128, k=8, mode="softmax_norm"),
        # an odd batch, sigmoid scores with a bias
        _case("router_1999", op="router", direction="backward", T=1999, H=4096, E=60, k=4, mode="sigmoid_norm", bias=True),
        # the router of the DeepSeek-V3-shaped layer
        _case("router_8192", op="router", direction="backward", T=8192, H=7168, E=256, k=8, mode="sigmoid_norm"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Token counts from one to 8192, hidden and intermediate sizes over the range of the listed ones (a fifth of them odd),
    any number of experts a table takes, blocks of one slot and of many; no case moves more than its operator's largest."""
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], 0), w["bytes"])
    while True:
        op = rng.choice(("permute", "combine", "glu", "router"))
        c = dict(_DEFAULTS, op=op, T=_log_int(rng, 1, 8192), E=rng.choice((4, 8, 16, 32, 60, 64, 128, 160, 256)))
        c["k"] = rng.randint(1, min(8, c["E"]))
        if op == "router":
            c.update(direction="backward", H=128 * _log_int(rng, 2, 56), mode=rng.choice(_MODES), bias=rng.random() < 0.3)
        else:
            c["dtype"] = rng.choice(("bf16", "bf16", "fp16", "fp32"))
            c["B"] = rng.choice((1, 16, 32, 128, 128, 256, 512))
            if op == "glu":
                c["direction"] = rng.choice(("forward", "backward", "pack"))
                c["I"] = _log_int(rng, 33, 14336) if rng.random() < 0.2 else 32 * _log_int(rng, 6, 448)
                c["act"] = rng.choice(("silu", "silu", "swish", "gelu", "gelu_tanh"))
                c["clamps"] = c["act"] == "swish" and c["direction"] != "pack"
                if c["direction"] == "pack":
                    c["dtype"] = "bf16"  # (moe_cte's checkpoints)
            else:
                c["direction"] = rng.choice(("forward", "backward"))
                c["H"] = _log_int(rng, 64, 7168) if rng.random() < 0.2 else 128 * _log_int(rng, 2, 56)
        if work(c)["bytes"] <= most[op]:
            return c


# ---- the block table ----------------------------------------------------------------------------------------------


def _blocks(c):
    """Blocks that the worst routing of T tokens needs."""
    return math.ceil((c["T"] * c["k"] - (c["E"] - 1)) / c["B"]) + c["E"] - 1


def _table(ids, E, B, N):
    """Token of every slot (T in padding slots) and expert of every block, from the chosen experts ``[T, k]``: expert
    after expert, tokens ascending, each expert's last block filled up with padding, spare blocks at the end."""
    T, k = ids.shape
    dev = ids.device
    counts = torch.bincount(ids.reshape(-1).long(), minlength=E)
    blocks = (counts + B - 1) // B
    blocks[E - 1] += N - blocks.sum()
    order = torch.argsort(ids.reshape(-1).long(), stable=True)  # by expert, then by token
    expert = ids.reshape(-1).long()[order]
    first = (torch.cumsum(blocks, 0) - blocks) * B
    rank = torch.arange(T * k, device=dev) - (torch.cumsum(counts, 0) - counts)[expert]
    table = torch.full((N * B,), T, dtype=torch.int32, device=dev)
    table[first[expert] + rank] = (order // k).to(torch.int32)
    return table, torch.repeat_interleave(torch.arange(E, dtype=torch.int32, device=dev), blocks)


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

    def randn(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)

    T, H, I, E, k, B = (c[n] for n in ("T", "H", "I", "E", "k", "B"))
    st = {"case": c}
    # popular and unpopular experts, as a router has them
    logits = torch.randn((T, E), generator=g, device=dev) + 0.5 * torch.randn((E,), generator=g, device=dev)
    if c["op"] == "router":
        st["x"] = randn(T, H)
        st["w"] = randn(H, E, std=H ** -0.5)
        st["bias"] = randn(E, std=0.5, dtype=torch.float32) if c["bias"] else None
        st["logits"] = logits
        st["ids"] = logits.topk(k, dim=1).indices.to(torch.int32)
        # what the combine's backward pass hands over: zero where a token was not routed, a row for the padding token
        st["d_aff"] = torch.zeros((T + 1, E), device=dev)
        st["d_aff"][:T].scatter_(1, st["ids"].long(), randn(T, k, dtype=torch.float32))
        return st
    N = _blocks(c)
    st["n_tokens"], st["block_size"], st["top_k"] = T, B, k
    ids = logits.topk(k, dim=1).indices
    st["table"], st["experts"] = _table(ids, E, B, N)
    if c["op"] == "permute":
        st["x"] = randn(T, H) if c["direction"] == "forward" else randn(N * B, H)
        return st
    if c["op"] == "combine":
        probs = torch.softmax(logits, 1)
        aff = torch.zeros((T + 1, E), device=dev)
        aff[:T].scatter_(1, ids, probs.gather(1, ids))
        st["aff"] = aff.to(torch.bfloat16)
        st["y"] = randn(N * B, H)
        if c["direction"] == "backward":
            st["d_out"] = randn(T, H)
        return st
    if c["direction"] == "pack":
        st["gate_up_T"] = randn(N, 2, I, B, std=2.0)
        return st
    gate_up = randn(N * B, 2, I, std=2.0 if not c["clamps"] else 4.0)
    if c["direction"] == "forward":
        st["gate_up"] = gate_up
        return st
    st["codes"], st["scales"] = _quantise(gate_up.float(), _routed(st))
    st["d_h"] = randn(N * B, I)
    return st


# ---- plain forms ----------------------------------------------------------------------------------------------------


def _routed(st):
    return (st["table"] >= 0) & (st["table"] < st["n_tokens"])


def _quantise(x, routed):
    """Rows ``[R, 2, I]`` -> e4m3 codes and one E8M0 scale per 32 neighbours of I: the smallest power of two that brings
    the largest of them to 448 or less.  Rows of padding slots are zero."""
    R, _, I = x.shape
    pad = -I % 32
    xg = torch.nn.functional.pad(x, (0, pad)).view(R, 2, -1, 32)
    xg = torch.where(routed.view(-1, 1, 1, 1), xg, torch.zeros_like(xg))
    amax = xg.abs().amax(-1)
    bits = amax.view(torch.int32)
    s = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp_(min=0)  # (448 = 1.75 * 2^8)
    inv = ((254 - s) << 23).view(torch.float32)
    codes = (xg * inv.unsqueeze(-1)).to(torch.float8_e4m3fn).view(R, 2, -1)[..., :I].contiguous()
    return codes.view(torch.uint8), s.to(torch.uint8)


def _dequantise(codes, scales):
    v = codes.view(torch.float8_e4m3fn).float()
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return v * s.repeat_interleave(32, dim=-1)[..., : v.shape[-1]]


def _act(x, act):
    """Value and derivative."""
    if act == "gelu":
        phi = 0.5 * torch.erfc(x * -0.7071067811865476)
        return x * phi, phi + x * torch.exp(-0.5 * x * x) * 0.3989422804014327
    if act == "gelu_tanh":
        s = torch.sigmoid(1.5957691216057308 * (x + 0.044715 * x * x * x))
        return x * s, s * (1 + x * (1 - s) * 1.5957691216057308 * (1 + 3 * 0.044715 * x * x))
    a = 1.702 if act == "swish" else 1.0
    s = torch.sigmoid(a * x)
    return x * s, s * (1 + a * x * (1 - s))


def _plain_permute(st):
    T = st["n_tokens"]
    x = st["x"].float()
    if st["case"]["direction"] == "forward":
        ids = st["table"].long().clamp(0, T - 1)
        return torch.where(_routed(st)[:, None], x[ids], torch.zeros((), device=x.device)).to(st["x"].dtype)
    ids = torch.where(_routed(st), st["table"].long(), T)
    out = torch.zeros((T + 1, x.shape[1]), device=x.device).index_add_(0, ids, x)
    return out[:T].to(st["x"].dtype)


def _plain_combine(st):
    T, B = st["n_tokens"], st["block_size"]
    routed = _routed(st)
    ids = torch.where(routed, st["table"].long(), T)
    e = st["experts"].long().repeat_interleave(B)
    w = st["aff"].float()[ids, e]
    y = st["y"].float()
    if st["case"]["direction"] == "forward":
        out = torch.zeros((T + 1, y.shape[1]), device=y.device).index_add_(0, ids, y * w[:, None])
        return out[:T].to(st["y"].dtype)
    rows = torch.where(routed[:, None], st["d_out"].float()[ids.clamp(max=T - 1)], torch.zeros((), device=y.device))
    d_aff = torch.zeros_like(st["aff"], dtype=torch.float32)
    d_aff.index_put_((ids, e), (rows * y).sum(1), accumulate=True)
    return (rows * w[:, None]).to(st["y"].dtype), d_aff


def _plain_glu(st):
    c = st["case"]
    if c["direction"] == "pack":
        x = st["gate_up_T"].float().permute(0, 3, 1, 2).reshape(-1, 2, c["I"])
        return _dequantise(*_quantise(x, _routed(st))).to(torch.bfloat16)
    routed = _routed(st)[:, None]
    zero = torch.zeros((), device=routed.device)
    if c["direction"] == "forward":
        x = st["gate_up"].float()
        if c["clamps"]:
            x = torch.stack((x[:, 0].clamp(max=_CLAMP), x[:, 1].clamp(-_CLAMP, _CLAMP)), 1)
        h = torch.where(routed, _act(x[:, 0], c["act"])[0] * x[:, 1], zero)
        return h.to(st["gate_up"].dtype), _dequantise(*_quantise(x, _routed(st))).to(torch.bfloat16)
    v = _dequantise(st["codes"], st["scales"])
    gate, up = v[:, 0], v[:, 1]
    keep_g = keep_u = None
    if c["clamps"]:
        keep_g, keep_u = gate < _CLAMP, up.abs() < _CLAMP
        gate, up = gate.clamp(max=_CLAMP), up.clamp(-_CLAMP, _CLAMP)
    a, d = _act(gate, c["act"])
    dh = st["d_h"].float()
    dg, du = dh * up * d, dh * a
    if c["clamps"]:
        dg, du = torch.where(keep_g, dg, zero), torch.where(keep_u, du, zero)
    d_gate_up = torch.where(routed[:, None], torch.stack((dg, du), 1), zero)
    return d_gate_up.to(st["d_h"].dtype), torch.where(routed, a * up, zero).to(st["d_h"].dtype)


def _plain_router(st):
    mode = st["case"]["mode"]
    l, ids, T = st["logits"], st["ids"].long(), st["case"]["T"]
    ga = st["d_aff"][:T].gather(1, ids)
    if mode in ("softmax_norm", "chosen_softmax"):  # dividing a softmax by the sum of a part is the softmax of that part
        a = torch.softmax(l.gather(1, ids), 1)
        dl = torch.zeros_like(l).scatter_(1, ids, a * (ga - (ga * a).sum(1, keepdim=True)))
    elif mode == "softmax":
        p = torch.softmax(l, 1)
        g = torch.zeros_like(l).scatter_(1, ids, ga)
        dl = p * (g - (g * p).sum(1, keepdim=True))
    else:
        s = torch.sigmoid(l.gather(1, ids))
        if mode == "sigmoid_norm":
            total = s.sum(1, keepdim=True)
            ga = (ga - (ga * s).sum(1, keepdim=True) / total) / total
        dl = torch.zeros_like(l).scatter_(1, ids, ga * s * (1 - s))
    out = [(dl @ st["w"].float().t()).to(st["x"].dtype), (st["x"].float().t() @ dl).to(st["w"].dtype)]
    return out + ([dl.sum(0)] if st["bias"] is not None else [])


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    if not own:
        return {"permute": _plain_permute, "combine": _plain_combine, "glu": _plain_glu, "router": _plain_router}[c["op"]](state)
    back = c["direction"] == "backward"
    if c["op"] == "permute":
        from nkilib.core.moe.token_permute import permute_tokens, permute_tokens_bwd

        if back:
            return permute_tokens_bwd(state["x"], state["table"], state["n_tokens"], state["top_k"])
        return permute_tokens(state["x"], state["table"])
    if c["op"] == "combine":
        from nkilib.core.moe.token_permute import combine_tokens, combine_tokens_bwd

        args = (state["y"], state["aff"], state["table"], state["experts"], state["block_size"])
        if back:
            return combine_tokens_bwd(state["d_out"], *args, state["top_k"])
        return combine_tokens(*args, state["n_tokens"], state["top_k"])
    if c["op"] == "glu":
        from nkilib.core.moe.glu_checkpoint import (dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd,
                                                    pack_gate_up_checkpoint)
        from nkilib.core.utils.common_types import ActFnType

        table = dict(token_position_to_id=state["table"], n_tokens=state["n_tokens"])
        if c["direction"] == "pack":
            return dequantize_checkpoint(*pack_gate_up_checkpoint(state["gate_up_T"], **table))
        opts = dict(table, activation_function={"silu": ActFnType.SiLU, "swish": ActFnType.Swish, "gelu": ActFnType.GELU,
                                                "gelu_tanh": ActFnType.GELU_Tanh_Approx}[c["act"]])
        if c["clamps"]:
            opts.update(gate_clamp_upper_limit=_CLAMP, up_clamp_upper_limit=_CLAMP, up_clamp_lower_limit=-_CLAMP)
        if back:
            return glu_checkpoint_bwd(state["codes"], state["scales"], state["d_h"], **opts)
        h, codes, scales = glu_checkpoint(state["gate_up"], **opts)
        return h, dequantize_checkpoint(codes, scales)
    from nkilib.core.router_topk import router_topk_bwd
    from nkilib.core.utils.common_types import RouterActFnType

    mode = c["mode"]
    out = router_topk_bwd(state["d_aff"], state["x"], state["w"], state["bias"], state["logits"], state["ids"],
                          RouterActFnType.SOFTMAX if "softmax" in mode else RouterActFnType.SIGMOID,
                          router_pre_norm=not mode.startswith("chosen"), norm_topk_prob=mode.endswith("_norm"))
    return out if state["bias"] is not None else out[:2]


# ---- the least work ---------------------------------------------------------------------------------------------------


def work(case):
    c = case
    T, H, I, E, k = (c[n] for n in ("T", "H", "I", "E", "k"))
    es, back = _SIZE[c["dtype"]], c["direction"] == "backward"
    if c["op"] == "router":
        # tokens, weights, logits, gradients of the chosen affinities and their indices in; gradients out
        return {"bytes": 2 * 2 * (T * H + H * E) + T * E * 4 + 8 * T * k, "flops": 4 * T * H * E}
    S, routed = _blocks(c) * c["B"], T * k
    if c["op"] == "permute":
        return {"bytes": 4 * S + es * H * ((routed + T) if back else (T + S)), "flops": routed * H if back else 0}
    if c["op"] == "combine":
        if back:
            return {"bytes": 4 * S + 2 * routed + es * H * (T + routed + S) + 4 * (T + 1) * E, "flops": 3 * routed * H}
        return {"bytes": 4 * S + 2 * routed + es * H * (routed + T), "flops": 2 * routed * H}
    # (records are returned as the values that they stand for, which bf16 holds exactly)
    scales = 2 * math.ceil(I / 32)
    if c["direction"] == "pack":
        return {"bytes": 4 * S + routed * 2 * I * es + S * 2 * I * 2, "flops": routed * 2 * I}
    if back:
        return {"bytes": 4 * S + routed * (2 * I + scales + I * es) + S * 3 * I * es, "flops": 10 * routed * I}
    return {"bytes": 4 * S + routed * 2 * I * es + S * I * (es + 2 * 2), "flops": 8 * routed * I}


# ---- in 64 bits -------------------------------------------------------------------------------------------------------


def _slot_lists(st):
    """``[T, k]`` slots of every token, ascending."""
    order = torch.argsort(torch.where(_routed(st), st["table"].long(), st["n_tokens"]), stable=True)
    return order[: st["n_tokens"] * st["top_k"]].view(st["n_tokens"], st["top_k"])


def _e4m3_values(x):
    """Groups of 32 along the last axis (any length) in 64 bits -> the values their 8-bit record stands for."""
    n = x.shape[-1]
    x = torch.cat((x, x.new_zeros(*x.shape[:-1], -n % 32)), -1)
    x = x.reshape(*x.shape[:-1], -1, 32)
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448).clamp(min=-127.0)))
    v = x / scale
    # (log2 of a quotient beside a power of two may fall on either side)
    scale = torch.where(amax > 448 * scale, 2 * scale, torch.where(amax <= 224 * scale, 0.5 * scale, scale)).clamp(min=2.0 ** -127)
    v = x / scale
    exponent = ((v.view(torch.int64) >> 52) & 0x7FF) - 1023
    step = torch.exp2(exponent.double().clamp(min=-6.0) - 3)
    return (torch.round(v / step) * step * scale).reshape(*x.shape[:-2], -1)[..., :n]


def _act64(x, act):
    if act == "gelu":
        return torch.nn.functional.gelu(x)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(x, approximate="tanh")
    return x / (1 + torch.exp(-(1.702 if act == "swish" else 1.0) * x))


def exact(case, seed):
    st = prepare(case, seed)
    c, T = st["case"], case["T"]
    if c["op"] == "router":
        return _exact_router(st)
    S, parts = st["table"].numel(), 8192
    if c["op"] == "permute":
        x = st["x"].double()
        if c["direction"] == "backward":
            lists = _slot_lists(st)
            return sum(x[lists[:, j]] for j in range(c["k"]))
        return torch.cat((x, x.new_zeros(1, x.shape[1])))[st["table"].long()]
    if c["op"] == "combine":
        lists = _slot_lists(st)
        e = st["experts"].long()[lists // c["B"]]
        w = st["aff"][:T].double().gather(1, e)
        if c["direction"] == "forward":
            return sum(w[:, j : j + 1] * st["y"][lists[:, j]].double() for j in range(c["k"]))
        d_out = st["d_out"].double()
        d_y = d_out.new_zeros(S, d_out.shape[1])
        d_aff = d_out.new_zeros(T + 1, c["E"])
        for j in range(c["k"]):
            d_y[lists[:, j]] = w[:, j : j + 1] * d_out
            d_aff[:T].scatter_(1, e[:, j : j + 1], (d_out * st["y"][lists[:, j]].double()).sum(1, keepdim=True))
        return d_y, d_aff
    routed = _routed(st)
    outs = []
    for r0 in range(0, S, parts):  # (rows by parts: every intermediate is 64 bits wide)
        r = slice(r0, min(r0 + parts, S))
        on = routed[r].double().view(-1, 1)
        if c["direction"] == "pack":
            rows = torch.arange(r.start, r.stop, device=routed.device)
            x = st["gate_up_T"][rows // c["B"], :, :, rows % c["B"]].double()
            outs.append((_e4m3_values(x * on[:, None]),))
            continue
        if c["direction"] == "forward":
            x = st["gate_up"][r].double()
            gate, up = x[:, 0], x[:, 1]
            if c["clamps"]:
                gate, up = torch.minimum(gate, gate.new_tensor(_CLAMP)), up.clamp(-_CLAMP, _CLAMP)
            outs.append((_act64(gate, c["act"]) * up * on, _e4m3_values(torch.stack((gate, up), 1) * on[:, None])))
            continue
        scale = torch.exp2(st["scales"][r].double() - 127).repeat_interleave(32, dim=-1)[..., : c["I"]]
        v = st["codes"][r].view(torch.float8_e4m3fn).double() * scale
        gate, up = v[:, 0].clone().requires_grad_(), v[:, 1].clone().requires_grad_()
        g, u = gate, up
        if c["clamps"]:  # (a value at its limit counts as clamped)
            g = torch.where(gate < _CLAMP, gate, torch.full_like(gate, _CLAMP))
            u = torch.where(up < _CLAMP, torch.where(up > -_CLAMP, up, torch.full_like(up, -_CLAMP)), torch.full_like(up, _CLAMP))
        h = _act64(g, c["act"]) * u
        dg, du = torch.autograd.grad(h, (gate, up), st["d_h"][r].double())
        outs.append((torch.stack((dg, du), 1) * on[:, None], (h * on).detach()))
    outs = tuple(torch.cat(o) for o in zip(*outs))
    return outs if len(outs) > 1 else outs[0]


def _exact_router(st):
    mode, T = st["case"]["mode"], st["case"]["T"]
    l = st["logits"].double().requires_grad_()
    chosen = torch.zeros_like(l, dtype=torch.bool).scatter_(1, st["ids"].long(), True)
    if mode.startswith("chosen"):
        a = torch.softmax(l.masked_fill(~chosen, -math.inf), 1) if mode.endswith("softmax") else torch.sigmoid(l) * chosen
    else:
        a = (torch.softmax(l, 1) if "softmax" in mode else torch.sigmoid(l)) * chosen
        if mode.endswith("_norm"):
            a = a / a.sum(1, keepdim=True)
    (dl,) = torch.autograd.grad(a, l, st["d_aff"][:T].double())
    out = [torch.matmul(dl, st["w"].double().t().contiguous()), torch.matmul(st["x"].double().t().contiguous(), dl)]
    return out + ([dl.sum(0)] if st["bias"] is not None else [])
