"""Tokens into the order of the block table and back, with routing weights, and their gradients.

``moe_cte`` gathers its tokens and adds up its contributions inside the layer, as the reference does
(src/nkilib_src/nkilib/core/moe/moe_cte/bwmm_shard_on_block.py:972-1038).  A program that multiplies the experts itself, or
runs the backward pass of a layer, does it through these operators, on the tables that ``build_token_blocks`` builds:

    xs      = permute_tokens(x[:T], tp2id)                                       # [N*B, H]
    out     = combine_tokens(ys, aff, tp2id, b2e, B, T, k)                       # [T, H]
    d_ys, d_aff = combine_tokens_bwd(d_out, ys, aff, tp2id, b2e, B, k)
    d_x     = permute_tokens_bwd(d_xs, tp2id, T, k)

Slot s holds token ``token_position_to_id[s]``; ids outside ``[0, T)`` (T, or -1 with ``skip_token``) are padding, whose rows
are zero on the way out and never read on the way in.  Sums are taken over a token's slots in ascending order in fp32 and
rounded once.  Rows are bfloat16, float16 or float32.

Plain calls, outside of torch's autograd: what they return has no graph, also where an input requires a gradient.
"""

from typing import Optional

import torch

from .... import _native as nv
from ...utils.kernel_assert import kernel_assert


def _table(token_position_to_id):
    t = nv.require_device_tensor(token_position_to_id, "token_position_to_id")
    if t.dim() != 1:
        t = t.reshape(-1)
    if t.dtype != torch.int32:
        kernel_assert(False, f"token_position_to_id must be int32 but got {t.dtype}")
    return t


def _rows(t, what, n=None):
    t = nv.require_device_tensor(t, what)
    if t.dim() != 2 or (n is not None and t.shape[0] != n):
        kernel_assert(False, f"{what} must be a matrix of {'tokens' if n is None else n} rows but got {tuple(t.shape)}")
    return t


def _same_device(*tensors):
    dev = tensors[0].device
    for t in tensors:
        if t.device != dev:
            kernel_assert(False, f"tensors must be on one device but are on {[str(t.device) for t in tensors]}")
    return dev


def _slots(tp2id, n_tokens, top_k, token_slots):
    """The list to go by, and whether the call has yet to make it."""
    if not 1 <= top_k <= 64:
        kernel_assert(False, f"top_k must be in [1, 64] but got {top_k}")
    if n_tokens < 0:
        kernel_assert(False, f"n_tokens must not be negative but got {n_tokens}")
    if token_slots is None:
        return tp2id.new_empty((n_tokens, 1 + top_k)), 1
    token_slots = nv.require_device_tensor(token_slots, "token_slots")
    if token_slots.dtype != torch.int32 or token_slots.shape != (n_tokens, 1 + top_k):
        kernel_assert(False, f"token_slots must be int32 [{n_tokens}, {1 + top_k}] but got {token_slots.dtype} "
                             f"{tuple(token_slots.shape)}")
    return token_slots, 0


def _routing(expert_affinities_masked, block_to_expert, block_size, tp2id, n_tokens):
    """Checked affinities ``[T1, E]``, experts of the blocks, block size, number of blocks."""
    aff = nv.require_device_tensor(expert_affinities_masked, "expert_affinities_masked")
    if aff.dtype not in (torch.bfloat16, torch.float32):
        kernel_assert(False, f"expert_affinities_masked must be bfloat16 or float32 but got {aff.dtype}")
    if aff.dim() != 2 or aff.shape[0] < n_tokens or aff.shape[1] < 1:
        kernel_assert(False, f"expert_affinities_masked must be [{n_tokens} or more, E] but got {tuple(aff.shape)}")
    b2e = nv.require_device_tensor(block_to_expert, "block_to_expert")
    if b2e.dim() != 1:
        b2e = b2e.reshape(-1)
    if b2e.dtype != torch.int32:
        kernel_assert(False, f"block_to_expert must be int32 but got {b2e.dtype}")
    B = int(block_size)
    if B < 1 or b2e.numel() * B != tp2id.numel():
        kernel_assert(False, f"token_position_to_id must hold N*B = {b2e.numel()}*{B} slots but holds {tp2id.numel()}")
    return aff, b2e, B


def build_token_slots(token_position_to_id: torch.Tensor, n_tokens: int, top_k: int, check: bool = False):
    """The block table's inverse, int32 ``[n_tokens, 1 + top_k]``: how many slots a token has, its slots in ascending order,
    -1 behind them.  The operators below make it for each call that is not given one (``token_slots``); a step that calls
    several makes it once.  It belongs to the table that it was made of.  A token that the table lists more than ``top_k``
    times (at most 64) comes out as NaN wherever it is summed; ``check=True`` synchronises and raises instead."""
    t = _table(token_position_to_id)
    n_tokens, top_k = int(n_tokens), int(top_k)
    dev = t.device
    out, _ = _slots(t, n_tokens, top_k, None)
    if n_tokens == 0:
        return out
    with nv.on_device(dev):
        rc = nv.lib().moe_token_slots(t.data_ptr(), t.numel(), n_tokens, top_k, out.data_ptr(), nv.stream_ptr(dev))
    nv.check(rc, "build_token_slots")
    if check:
        most = int(out[:, 0].max().item())
        kernel_assert(most <= top_k, f"a token has {most} slots, more than top_k = {top_k}")
    return out


def permute_tokens(hidden_states: torch.Tensor, token_position_to_id: torch.Tensor):
    """Rows ``[T, H]`` -> ``[N*B, H]``: slot s gets the row of its token, zeros where it holds padding.  Rows of any type:
    records and codes of a quantising front end too."""
    x = _rows(hidden_states, "hidden_states")
    t = _table(token_position_to_id)
    dev = _same_device(x, t)
    out = x.new_empty((t.numel(), x.shape[1]))
    if out.numel() == 0:
        return out
    if x.shape[0] == 0:
        return out.zero_()
    with nv.on_device(dev):
        rc = nv.lib().moe_permute_tokens(x.data_ptr(), t.data_ptr(), t.numel(), x.shape[0], x.shape[1] * x.element_size(),
                                         out.data_ptr(), nv.stream_ptr(dev))
    nv.check(rc, "permute_tokens")
    return out


def permute_tokens_bwd(d_permuted: torch.Tensor, token_position_to_id: torch.Tensor, n_tokens: int, top_k: int,
                       token_slots: Optional[torch.Tensor] = None):
    """Gradient of ``permute_tokens``: ``[N*B, H]`` -> ``[n_tokens, H]``, the sum over each token's slots (zero for a token
    without any)."""
    t = _table(token_position_to_id)
    d = _rows(d_permuted, "d_permuted", t.numel())
    n_tokens, top_k = int(n_tokens), int(top_k)
    dev = _same_device(d, t)
    dt = nv.dtype_code(d, "d_permuted")
    slots, build = _slots(t, n_tokens, top_k, token_slots)
    _same_device(d, slots)
    out = d.new_empty((n_tokens, d.shape[1]))
    if out.numel() == 0 or t.numel() == 0:
        return out.zero_()
    with nv.on_device(dev):
        rc = nv.lib().moe_combine_tokens(d.data_ptr(), dt, None, 0, 0, 0, t.data_ptr(), None, 0, 0, slots.data_ptr(), top_k, build,
                                         t.numel(), n_tokens, d.shape[1], out.data_ptr(), nv.stream_ptr(dev))
    nv.check(rc, "permute_tokens_bwd")
    return out


def combine_tokens(permuted: torch.Tensor, expert_affinities_masked: torch.Tensor, token_position_to_id: torch.Tensor,
                   block_to_expert: torch.Tensor, block_size: int, n_tokens: int, top_k: int,
                   token_slots: Optional[torch.Tensor] = None):
    """``[N*B, H]`` -> ``[n_tokens, H]``: each token's slots, weighted with its affinity for the slot's expert and added.
    ``expert_affinities_masked`` ``[n_tokens or more, E]`` bfloat16 or float32, as ``route_for_moe`` returns it (rows behind
    the tokens are not read).  Slots of blocks whose expert is outside ``[0, E)`` count for nothing."""
    t = _table(token_position_to_id)
    y = _rows(permuted, "permuted", t.numel())
    n_tokens, top_k = int(n_tokens), int(top_k)
    aff, b2e, B = _routing(expert_affinities_masked, block_to_expert, block_size, t, n_tokens)
    dev = _same_device(y, t, aff, b2e)
    dt = nv.dtype_code(y, "permuted")
    slots, build = _slots(t, n_tokens, top_k, token_slots)
    _same_device(y, slots)
    out = y.new_empty((n_tokens, y.shape[1]))
    if out.numel() == 0 or t.numel() == 0:
        return out.zero_()
    with nv.on_device(dev):
        rc = nv.lib().moe_combine_tokens(y.data_ptr(), dt, aff.data_ptr(), nv.dtype_code(aff, "expert_affinities_masked"),
                                         aff.shape[0], aff.shape[1], t.data_ptr(), b2e.data_ptr(), B, b2e.numel(), slots.data_ptr(),
                                         top_k, build, t.numel(), n_tokens, y.shape[1], out.data_ptr(), nv.stream_ptr(dev))
    nv.check(rc, "combine_tokens")
    return out


def combine_tokens_bwd(d_output: torch.Tensor, permuted: torch.Tensor, expert_affinities_masked: torch.Tensor,
                       token_position_to_id: torch.Tensor, block_to_expert: torch.Tensor, block_size: int, top_k: int,
                       token_slots: Optional[torch.Tensor] = None):
    """Gradients of ``combine_tokens`` from that of its output, ``[T, H]``: of ``permuted`` (its shape and type; zero rows in
    padding slots) and of ``expert_affinities_masked`` (its shape, float32; zero where a token has no slot of the expert)."""
    t = _table(token_position_to_id)
    y = _rows(permuted, "permuted", t.numel())
    d = _rows(d_output, "d_output")
    n_tokens, top_k = d.shape[0], int(top_k)
    if d.dtype != y.dtype or d.shape[1] != y.shape[1]:
        kernel_assert(False, f"d_output and permuted must agree in type and row length but are {d.dtype} {tuple(d.shape)} and "
                             f"{y.dtype} {tuple(y.shape)}")
    aff, b2e, B = _routing(expert_affinities_masked, block_to_expert, block_size, t, n_tokens)
    dev = _same_device(y, t, d, aff, b2e)
    dt = nv.dtype_code(y, "permuted")
    slots, build = _slots(t, n_tokens, top_k, token_slots)
    _same_device(y, slots)
    d_y = torch.empty_like(y)
    d_aff = torch.empty(aff.shape, dtype=torch.float32, device=dev)
    if n_tokens == 0 or y.numel() == 0:  # (a table of padding only, rows of no elements)
        return d_y.zero_(), d_aff.zero_()
    with nv.on_device(dev):
        rc = nv.lib().moe_combine_tokens_bwd(d.data_ptr(), y.data_ptr(), dt, aff.data_ptr(),
                                             nv.dtype_code(aff, "expert_affinities_masked"), aff.shape[0], aff.shape[1], t.data_ptr(),
                                             b2e.data_ptr(), B, b2e.numel(), slots.data_ptr(), top_k, build, n_tokens, y.shape[1],
                                             d_y.data_ptr(), d_aff.data_ptr(), nv.stream_ptr(dev))
    nv.check(rc, "combine_tokens_bwd")
    return d_y, d_aff
