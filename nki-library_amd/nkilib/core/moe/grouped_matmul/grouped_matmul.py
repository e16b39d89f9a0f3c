"""Products of the rows of every expert with its weights, for experts of any number of rows, and their gradients.

``moe_cte`` multiplies its experts inside the layer, as the reference does
(src/nkilib_src/nkilib/core/moe/moe_cte/bwmm_shard_on_block.py:972-1038).  A program that runs a layer from its parts
multiplies the rows that ``permute_tokens`` put into the order of the experts through these operators:

    offsets = expert_row_offsets(b2e, B, E)                       # int32 [E+1], on the device
    gu      = grouped_matmul(xs, w_gate_up.view(E, H, 2 * I), offsets)
    d_xs, d_w = grouped_matmul_bwd(d_gu, xs, w_gate_up.view(E, H, 2 * I), offsets)

Rows ``[row_offsets[e], row_offsets[e + 1])`` are expert e's.  Offsets are read on the device and nothing waits for them: whatever they
are, they are taken into ``[0, S]`` and as never falling; rows of no expert are zero in a result.  Everything is bfloat16 or
float16; sums are taken in fp32 and rounded once.  What is not contiguous is copied in every call, weights ``[E, N, K]`` handed over as
their transposed view among it.

Plain calls, outside of torch's autograd: what they return has no graph, also where an input requires a gradient.
"""

from typing import Optional

import torch

from .... import _native as nv
from ...utils.kernel_assert import kernel_assert

MAX_EXPERTS = 1024
MAX_COLUMNS = 1 << 20


def expert_row_offsets(block_to_expert: torch.Tensor, block_size: int, num_experts: int):
    """Bounds of every expert's rows, int32 ``[num_experts + 1]``, from the experts of the blocks as ``build_token_blocks`` returns
    them (ascending; blocks of no expert in ``[0, num_experts)`` behind the others) and the rows of a block."""
    b2e = nv.require_device_tensor(block_to_expert, "block_to_expert").reshape(-1)
    if b2e.dtype != torch.int32:
        kernel_assert(False, f"block_to_expert must be int32 but got {b2e.dtype}")
    B, E, N = int(block_size), int(num_experts), b2e.numel()
    if not 1 <= E <= MAX_EXPERTS:
        kernel_assert(False, f"num_experts must be in [1, {MAX_EXPERTS}] but got {E}")
    if B < 1 or N * B >= 1 << 31:
        kernel_assert(False, f"block_size must be positive and {N} blocks hold fewer than 2^31 rows but got {B}")
    dev = b2e.device
    out = torch.empty(E + 1, dtype=torch.int32, device=dev)
    with nv.on_device(dev):
        rc = nv.lib().moe_expert_row_offsets(b2e.data_ptr(), N, B, E, out.data_ptr(), nv.stream_ptr(dev))
    nv.check(rc, "expert_row_offsets")
    return out


def check_offsets(row_offsets, E, dev):
    o = nv.require_device_tensor(row_offsets, "row_offsets")
    if o.dtype != torch.int32 or o.shape != (E + 1,):
        kernel_assert(False, f"row_offsets must be int32 [{E + 1}] but got {o.dtype} {tuple(o.shape)}")
    if o.device != dev:
        kernel_assert(False, f"tensors must be on one device but are on {dev} and {o.device}")
    return o


def check_sizes(S, K, N, E):
    if not 1 <= E <= MAX_EXPERTS:
        kernel_assert(False, f"there must be 1 to {MAX_EXPERTS} experts but got {E}")
    if K > MAX_COLUMNS or N > MAX_COLUMNS or S >= (1 << 31) - 1024:
        kernel_assert(False, f"rows of at most {MAX_COLUMNS} values and fewer than 2^31 - 1024 of them but got {S} x {K} and {N} columns")


def _operand(t, what, dims, like=None):
    t = nv.require_device_tensor(t, what)
    if t.dtype not in (torch.bfloat16, torch.float16):
        kernel_assert(False, f"{what} must be bfloat16 or float16 but got {t.dtype}")
    if t.dim() != dims:
        kernel_assert(False, f"{what} must have {dims} dimensions but got {tuple(t.shape)}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        kernel_assert(False, f"{what} must agree with the other tensors in type and device but is {t.dtype} on {t.device}, "
                             f"not {like.dtype} on {like.device}")
    return t


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, row_offsets: torch.Tensor):
    """Rows ``[S, K]`` times the weights ``[E, K, N]`` of their experts -> ``[S, N]``."""
    x = _operand(x, "x", 2)
    w = _operand(weight, "weight", 3, x)
    (S, K), (E, Kw, N) = x.shape, w.shape
    if K != Kw:
        kernel_assert(False, f"weight must be [E, {K}, N] but got {tuple(w.shape)}")
    check_sizes(S, K, N, E)
    dev = x.device
    o = check_offsets(row_offsets, E, dev)
    out = x.new_empty((S, N))
    if K == 0 or out.numel() == 0:
        return out.zero_()
    with nv.on_device(dev):
        rc = nv.lib().moe_grouped_matmul(x.data_ptr(), w.data_ptr(), nv.dtype_code(x, "x"), o.data_ptr(), S, K, N, E, out.data_ptr(),
                                         nv.stream_ptr(dev))
    nv.check(rc, "grouped_matmul")
    return out


def grouped_matmul_bwd(d_output: torch.Tensor, x: Optional[torch.Tensor], weight: torch.Tensor, row_offsets: torch.Tensor,
                       weight_grad_dtype: Optional[torch.dtype] = None, need_x: bool = True, need_weight: bool = True):
    """Gradients of ``grouped_matmul`` from that of its result, ``[S, N]``: of ``x`` (its shape and type; zero in rows of no expert) and
    of ``weight`` (its shape; its type or ``torch.float32``; zero for an expert without rows).  What is not needed is not computed and
    comes back as None; ``x`` may be None without the weights' gradient."""
    d = _operand(d_output, "d_output", 2)
    w = _operand(weight, "weight", 3, d)
    (S, N), (E, K, Nw) = d.shape, w.shape
    if N != Nw:
        kernel_assert(False, f"weight must be [E, K, {N}] but got {tuple(w.shape)}")
    kernel_assert(need_x or need_weight, "at least one gradient must be needed")
    check_sizes(S, K, N, E)
    dev = d.device
    o = check_offsets(row_offsets, E, dev)
    dt = nv.dtype_code(d, "d_output")
    d_x = d_w = None
    if need_weight:
        kernel_assert(x is not None, "x must be given for the weights' gradient")
        x = _operand(x, "x", 2, d)
        if x.shape != (S, K):
            kernel_assert(False, f"x must be [{S}, {K}] but got {tuple(x.shape)}")
        wdt = w.dtype if weight_grad_dtype is None else weight_grad_dtype
        if wdt not in (w.dtype, torch.float32):
            kernel_assert(False, f"weight_grad_dtype must be {w.dtype} or torch.float32 but got {wdt}")
        d_w = torch.empty(w.shape, dtype=wdt, device=dev)
    if need_x:
        d_x = d.new_empty((S, K))
    if S == 0 or K == 0 or N == 0:
        return d_x.zero_() if need_x else None, d_w.zero_() if need_weight else None
    with nv.on_device(dev):
        rc = nv.lib().moe_grouped_matmul_bwd(d.data_ptr(), x.data_ptr() if need_weight else None, w.data_ptr(), dt, o.data_ptr(), S, K, N, E,
                                             nv.ptr(d_x), nv.ptr(d_w), nv.dtype_code(d_w, "d_weight") if need_weight else dt,
                                             nv.stream_ptr(dev))
    nv.check(rc, "grouped_matmul_bwd")
    return d_x, d_w
