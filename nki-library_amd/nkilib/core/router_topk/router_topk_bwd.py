"""The gradient of ``router_topk`` over ``moe_router_topk_bwd`` of the C ABI.

The reference has the forward pass only (src/nkilib_src/nkilib/core/router_topk/router_topk.py:55-75); the formulas are those of
its semantics (router_topk_torch.py:23-135), differentiated.  A plain call, outside of torch's autograd: it returns no graph.
"""

import torch

from ... import _native as nv
from ..utils.common_types import RouterActFnType
from ..utils.kernel_assert import kernel_assert


def router_topk_bwd(d_expert_affinities, x, w, w_bias, router_logits, expert_index, act_fn, router_pre_norm=True,
                    norm_topk_prob=False, mask_to_topk=True):
    """By default the gradient of ``route_for_moe``, whose affinities are zero outside of the choice.  That of ``router_topk``'s full table
    (its default, ``norm_topk_prob=False``: every expert has an affinity, and a loss over all of them a gradient) needs
    ``mask_to_topk=False``; with ``True`` gradients of experts that were not chosen are ignored.

    ``d_expert_affinities`` ``[T or more, E]`` float32 or bfloat16 (``combine_tokens_bwd`` returns it) -> gradients
    ``[d_x [T, H], d_w [H, E], d_bias]`` in the types of ``x``, ``w`` (bfloat16) and ``w_bias`` (``None`` without one).

    ``x`` ``[T, H]`` (``x_hbm_layout=1``), ``w`` ``[H, E]``, ``w_bias`` and the options are those of the forward call;
    ``router_logits`` ``[T, E]`` (float32, or bfloat16 at that precision) and ``expert_index`` ``[T, k]`` are what it returned.
    (``norm_topk_prob`` or ``router_pre_norm=False`` leave the selected experts alone an affinity, and ``mask_to_topk`` no choice.)
    The gradient of the logits is fp32; into ``d_w``, and into the ``d_x`` of a softmax over all experts or of the full table, it enters
    as the sum of two bf16 (2^-17 of it)."""
    x = nv.require_device_tensor(x, "x")
    w = nv.require_device_tensor(w, "w")
    g = nv.require_device_tensor(d_expert_affinities, "d_expert_affinities")
    logits = nv.require_device_tensor(router_logits, "router_logits")
    ids = nv.require_device_tensor(expert_index, "expert_index")
    if x.dim() != 2 or w.dim() != 2 or x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or x.shape[1] != w.shape[0]:
        kernel_assert(False, f"x and w must be bfloat16 [T, H] and [H, E] but are {x.dtype} {tuple(x.shape)} and {w.dtype} "
                             f"{tuple(w.shape)}")
    if x.data_ptr() % 16:  # (rows are read in pieces of 16 bytes)
        x = x.clone()
    (T, H), E = x.shape, w.shape[1]
    if not 1 <= E <= 512:
        kernel_assert(False, f"E must be in [1, 512] but got {E}")
    if H < 1 or H % 128 != 0 or H > 2**20:
        kernel_assert(False, f"H must be a multiple of 128 up to 2^20 but got {H}")
    if ids.dim() != 2 or ids.dtype not in (torch.int32, torch.uint32) or ids.shape[0] != T or not 1 <= ids.shape[1] <= min(8, E):
        kernel_assert(False, f"expert_index must be a 32-bit integer [T, k] with k in [1, min(8, E)] but is {ids.dtype} {tuple(ids.shape)}")
    for t, what, rows in ((g, "d_expert_affinities", "T or more"), (logits, "router_logits", "T")):
        if t.dtype not in (torch.bfloat16, torch.float32) or t.dim() != 2 or t.shape[1] != E or t.shape[0] < T or \
                (rows == "T" and t.shape[0] != T):
            kernel_assert(False, f"{what} must be bfloat16 or float32 [{rows}, {E}] with T = {T} but is {t.dtype} {tuple(t.shape)}")
    dev = x.device
    bias = d_bias = None
    if w_bias is not None:
        bias = nv.require_device_tensor(w_bias, "w_bias")
        if bias.numel() != E or bias.dtype not in (torch.bfloat16, torch.float32):
            kernel_assert(False, f"w_bias must hold E = {E} bfloat16 or float32 values but is {bias.dtype} {tuple(bias.shape)}")
        d_bias = torch.empty_like(bias)
    for t in (w, g, logits, ids, bias):
        if t is not None and t.device != dev:
            kernel_assert(False, f"all tensors must be on {dev} but one is on {t.device}")
    act = act_fn if isinstance(act_fn, RouterActFnType) else RouterActFnType(act_fn)
    d_x, d_w = torch.empty_like(x), torch.empty_like(w)
    if T == 0:
        return [d_x, d_w.zero_(), None if d_bias is None else d_bias.zero_()]
    L = nv.lib()
    ws = torch.empty(L.moe_router_topk_bwd_workspace_bytes(T, H, E), dtype=torch.uint8, device=dev)
    with nv.on_device(dev):
        rc = L.moe_router_topk_bwd(g.data_ptr(), nv.dtype_code(g, "d_expert_affinities"), x.data_ptr(), w.data_ptr(), logits.data_ptr(),
                                   nv.dtype_code(logits, "router_logits"), ids.data_ptr(), T, H, E, ids.shape[1], act.value,
                                   int(bool(router_pre_norm)), int(bool(norm_topk_prob)), int(bool(mask_to_topk)), d_x.data_ptr(),
                                   d_w.data_ptr(), nv.ptr(d_bias), nv.DT_FP32 if bias is None else nv.dtype_code(bias, "w_bias"),
                                   nv.ptr(ws), ws.numel(), nv.stream_ptr(dev))
    nv.check(rc, "router_topk_bwd")
    return [d_x, d_w, d_bias]
