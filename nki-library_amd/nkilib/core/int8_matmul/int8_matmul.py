"""Products in 8-bit integers with a scale per token and per channel, of one matrix or of the rows of every expert.

The rows' codes and scales are what ``rmsnorm_quant_rows`` makes of a residual stream, the weights' what it makes of their rows
without a norm (codes ``[N, K]``, one scale per row of them).  ``permute_tokens`` moves codes and scales into the order of the
experts.  Sums are whole numbers and exact; each is multiplied with its two scales in fp32 and rounded once to the result's type.

    codes, scales, residual = rmsnorm_quant_rows(hidden, gamma, residual=residual)
    out = int8_matmul(codes, scales, w_codes, w_scales, bias)                       # [T, N]
    out = grouped_int8_matmul(permute_tokens(codes, tp2id), permute_tokens(scales[:, None], tp2id), w_codes, w_scales, offsets)

Plain calls, outside of torch's autograd.
"""

from typing import Optional

import torch

from ... import _native as nv
from ..moe.grouped_matmul.grouped_matmul import check_offsets, check_sizes
from ..utils.kernel_assert import kernel_assert

MAX_TERMS = (1 << 17) - 1  # (products of at most 2^14: their sums stay inside 32 bits)


def _codes(t, what, dims=None):
    t = nv.require_device_tensor(t, what)
    if t.dtype != torch.int8:
        kernel_assert(False, f"{what} must be int8 but got {t.dtype}")
    if dims is None and t.dim() < 1 or dims is not None and t.dim() != dims:
        kernel_assert(False, f"{what} must have {dims or '1 or more'} dimensions but got {tuple(t.shape)}")
    return t


def _scales(t, what, shape, dev):
    t = nv.require_device_tensor(t, what)
    if t.dtype != torch.float32:
        kernel_assert(False, f"{what} must be float32 but got {t.dtype}")
    if t.shape != shape and t.shape != (*shape, 1):
        kernel_assert(False, f"{what} must be {list(shape)} but got {tuple(t.shape)}")
    if t.device != dev:
        kernel_assert(False, f"tensors must be on one device but are on {dev} and {t.device}")
    return t


def _run(x, x_scales, weight, weight_scales, bias, row_offsets, S, K, N, E, shape, out_dtype, what):
    if out_dtype not in (torch.bfloat16, torch.float16, torch.float32):
        kernel_assert(False, f"out_dtype must be bfloat16, float16 or float32 but got {out_dtype}")
    dev = x.device
    if weight.device != dev:
        kernel_assert(False, f"tensors must be on one device but are on {dev} and {weight.device}")
    check_sizes(S, K, N, E)
    if K > MAX_TERMS:
        kernel_assert(False, f"rows must have at most {MAX_TERMS} codes but have {K}")
    if bias is not None:
        bias = nv.require_device_tensor(bias, "bias")
        if bias.dtype != out_dtype or bias.shape != (N,) or bias.device != dev:
            kernel_assert(False, f"bias must be {out_dtype} [{N}] on {dev} but got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    out = x.new_empty(shape, dtype=out_dtype)
    if K == 0 and out.numel():  # (sums of nothing)
        return out.zero_() if bias is None else out.copy_(bias.detach().expand(shape))
    if out.numel() == 0:
        return out
    with nv.on_device(dev):
        rc = nv.lib().moe_int8_matmul(x.data_ptr(), x_scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(), nv.ptr(bias),
                                      nv.ptr(row_offsets), S, K, N, E, out.data_ptr(), nv.dtype_code(out, "out_dtype"),
                                      nv.stream_ptr(dev))
    nv.check(rc, what)
    return out


def int8_matmul(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16):
    """Codes ``[..., K]`` with scales ``[...]`` (or ``[..., 1]``) times codes ``[N, K]`` with scales ``[N]`` -> ``[..., N]``, bfloat16,
    float16 or float32; ``bias`` ``[N]`` of that type is added ahead of the rounding."""
    x = _codes(x, "x")
    w = _codes(weight, "weight", 2)
    (N, Kw), lead, dev = w.shape, x.shape[:-1], x.device
    K = x.shape[-1]
    if Kw != K:
        kernel_assert(False, f"weight must be [N, {K}] but got {tuple(w.shape)}")
    S = lead.numel()
    xs = _scales(x_scales, "x_scales", lead, dev)
    ws = _scales(weight_scales, "weight_scales", (N,), dev)
    return _run(x, xs, w, ws, bias, None, S, K, N, 1, (*lead, N), out_dtype, "int8_matmul")


def grouped_int8_matmul(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor,
                        row_offsets: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16):
    """Codes ``[S, K]`` with scales ``[S]`` (or ``[S, 1]``) times the codes ``[E, N, K]`` with scales ``[E, N]`` of their experts ->
    ``[S, N]``.  Rows ``[row_offsets[e], row_offsets[e + 1])`` are expert e's, as for ``grouped_matmul``; rows of no expert are zero."""
    x = _codes(x, "x", 2)
    w = _codes(weight, "weight", 3)
    (S, K), (E, N, Kw) = x.shape, w.shape
    if K != Kw:
        kernel_assert(False, f"weight must be [E, N, {K}] but got {tuple(w.shape)}")
    xs = _scales(x_scales, "x_scales", (S,), x.device)
    ws = _scales(weight_scales, "weight_scales", (E, N), x.device)
    o = check_offsets(row_offsets, E, x.device)
    return _run(x, xs, w, ws, None, o, S, K, N, E, (S, N), out_dtype, "grouped_int8_matmul")
