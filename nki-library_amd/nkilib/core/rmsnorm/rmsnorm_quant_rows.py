"""RMSNorm with the residual's addition and an output in 8 bits with one scale per row, its gradient, and such rows as values.

The reference quantises rows without a residual (``rmsnorm_quant_kernel``, src/nkilib_src/nkilib/core/rmsnorm/rmsnorm_quant.py:86-92)
and adds a residual ahead of an MX output (``rmsnorm_mx_quantize_tkg``,
src/nkilib_src/nkilib/core/subkernels/rmsnorm_mx_quantize_tkg.py:29-40); this is the front end of the products in 8-bit
integers (``nkilib.core.int8_matmul``), codes and scales apart:

    codes, scales, stream = rmsnorm_quant_rows(hidden, gamma, residual=stream)    # [..., H] int8, [...] fp32, [..., H]
    w_codes, w_scales = rmsnorm_quant_rows(w, None, do_norm=False)                # weights [N, K], a scale per channel
    d_hidden, d_gamma = rmsnorm_quant_rows_bwd(d_y, stream, gamma, d_residual=d_stream)

Rows are bfloat16, float16 or float32 of up to 16384 values.  Plain calls, outside of torch's autograd.
"""

from typing import Optional

import torch

from ... import _native as nv
from ..utils.kernel_assert import kernel_assert
from .rmsnorm_quant import MAX_H

_CODES = {torch.int8: nv.DT_INT8, torch.float8_e4m3fn: nv.DT_FP8}


def _rows(t, what, like=None):
    t = nv.require_device_tensor(t, what)
    nv.dtype_code(t, what)
    if t.dim() < 1 or not 1 <= t.shape[-1] <= MAX_H:
        kernel_assert(False, f"{what} must have rows of 1 to {MAX_H} values but got {tuple(t.shape)}")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        kernel_assert(False, f"{what} must be {like.dtype} {tuple(like.shape)} on {like.device} but got {t.dtype} {tuple(t.shape)} "
                             f"on {t.device}")
    return t


def _gamma(gamma, H, dev):
    g = nv.require_device_tensor(gamma, "gamma")
    nv.dtype_code(g, "gamma")
    if g.numel() != H or g.shape[-1] != H or g.device != dev:
        kernel_assert(False, f"gamma must hold {H} values on {dev} but got {tuple(g.shape)} on {g.device}")
    return g


def _eps(eps):
    eps = float(eps)
    kernel_assert(eps >= 0, f"Epsilon must be positive but got {eps}")
    return eps


def rmsnorm_quant_rows(hidden: torch.Tensor, gamma: Optional[torch.Tensor] = None, eps: float = 1e-6, do_norm: bool = True,
                       residual: Optional[torch.Tensor] = None, code_dtype: torch.dtype = torch.int8):
    """``hidden`` ``[..., H]`` -> codes ``[..., H]`` (``torch.int8`` or ``torch.float8_e4m3fn``) and scales ``[...]`` (fp32), and with
    ``residual`` (hidden's shape and type) ``hidden + residual`` rounded to that type, which is what is normalised.

    y = s / sqrt(mean(s^2) + eps) * gamma (``gamma`` None: ones; ``do_norm=False``: y = s, and no gamma);
    scale = max(max|y|, 2^-100) / M, code = y * (M / max(max|y|, 2^-100)) to nearest, M = 127 or 448.  A row of zeros has codes 0; a row
    whose y is not finite has the scale NaN and codes 0."""
    x = _rows(hidden, "hidden")
    if code_dtype not in _CODES:
        kernel_assert(False, f"code_dtype must be int8 or float8_e4m3fn but got {code_dtype}")
    eps = _eps(eps)
    H, dev = x.shape[-1], x.device
    kernel_assert(do_norm or gamma is None, "gamma must be None without the norm")
    g = _gamma(gamma, H, dev) if gamma is not None else None
    r = out_r = None
    if residual is not None:
        r = _rows(residual, "residual", x)
        out_r = torch.empty_like(x)
    codes = torch.empty(x.shape, dtype=code_dtype, device=dev)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    rows = scales.numel()
    if rows:
        with nv.on_device(dev):
            rc = nv.lib().moe_rmsnorm_quant_rows(x.data_ptr(), nv.dtype_code(x, "hidden"), nv.ptr(r), nv.ptr(g),
                                                 nv.dtype_code(g, "gamma") if g is not None else nv.DT_BF16, 1 if do_norm else 0, eps,
                                                 rows, H, _CODES[code_dtype], codes.data_ptr(), scales.data_ptr(), nv.ptr(out_r),
                                                 nv.stream_ptr(dev))
        nv.check(rc, "rmsnorm_quant_rows")
    return (codes, scales) if residual is None else (codes, scales, out_r)


def rmsnorm_quant_rows_bwd(d_normed: torch.Tensor, hidden: torch.Tensor, gamma: Optional[torch.Tensor], eps: float = 1e-6,
                           d_residual: Optional[torch.Tensor] = None):
    """Gradient of the norm from that of its values, ``d_normed`` ``[..., H]``; ``hidden`` is what was normalised (with a residual: the sum
    that came back), of the same type.  The rounding to codes passes gradients on as they are.  ``d_residual``: gradient of the sum
    from its other uses, added.  Returns the gradient of the sum, which is ``hidden``'s and ``residual``'s alike, and that of ``gamma``
    (its shape and type; None without one)."""
    x = _rows(hidden, "hidden")
    d = _rows(d_normed, "d_normed", x)
    r = _rows(d_residual, "d_residual", x) if d_residual is not None else None
    eps = _eps(eps)
    H, dev = x.shape[-1], x.device
    rows = x.numel() // H
    g = _gamma(gamma, H, dev) if gamma is not None else None
    d_x = torch.empty_like(x)
    d_g = torch.empty_like(g) if g is not None else None
    if rows == 0:
        return d_x, d_g.zero_() if d_g is not None else None
    L = nv.lib()
    nbytes = L.moe_rmsnorm_quant_rows_bwd_workspace_bytes(rows, H) if g is not None else 0
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev) if nbytes else None
    with nv.on_device(dev):
        rc = L.moe_rmsnorm_quant_rows_bwd(d.data_ptr(), x.data_ptr(), nv.dtype_code(x, "hidden"), nv.ptr(g),
                                          nv.dtype_code(g, "gamma") if g is not None else nv.DT_BF16, nv.ptr(r), eps, rows, H,
                                          d_x.data_ptr(), nv.ptr(d_g), nv.ptr(ws), nbytes, nv.stream_ptr(dev))
    nv.check(rc, "rmsnorm_quant_rows_bwd")
    return d_x, d_g


def dequantize_rows(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """Codes ``[..., H]`` (int8 or float8_e4m3fn) with scales ``[...]`` -> the values they stand for, rounded once to ``dtype``."""
    c = nv.require_device_tensor(codes, "codes")
    if c.dtype not in _CODES:
        kernel_assert(False, f"codes must be int8 or float8_e4m3fn but got {c.dtype}")
    if c.dim() < 1 or c.shape[-1] >= 1 << 24:
        kernel_assert(False, f"codes must have rows of fewer than 2^24 but got {tuple(c.shape)}")
    s = nv.require_device_tensor(scales, "scales")
    if s.dtype != torch.float32 or s.shape != c.shape[:-1] or s.device != c.device:
        kernel_assert(False, f"scales must be float32 {tuple(c.shape[:-1])} on {c.device} but got {s.dtype} {tuple(s.shape)} on {s.device}")
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        kernel_assert(False, f"dtype must be bfloat16, float16 or float32 but got {dtype}")
    dev = c.device
    out = torch.empty(c.shape, dtype=dtype, device=dev)
    if out.numel():
        with nv.on_device(dev):
            rc = nv.lib().moe_dequantize_rows(c.data_ptr(), _CODES[c.dtype], s.data_ptr(), s.numel(), c.shape[-1], out.data_ptr(),
                                              nv.dtype_code(out, "dtype"), nv.stream_ptr(dev))
        nv.check(rc, "dequantize_rows")
    return out
