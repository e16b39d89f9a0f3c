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


# (Few rows are bound by the host's side of a call: what is asked of a tensor is asked once.)
def _rows(t, what):
    """The tensor, its type's code and its shape."""
    t = nv.require_device_tensor(t, what)
    code, shape = nv.dtype_code(t, what), t.shape
    if len(shape) < 1 or not 1 <= shape[-1] <= MAX_H:
        kernel_assert(False, f"{what} must have rows of 1 to {MAX_H} values but got {tuple(shape)}")
    return t, code, shape


def _alike(t, what, like):
    t = nv.require_device_tensor(t, what)
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        kernel_assert(False, f"{what} must be {like.dtype} {tuple(like.shape)} on {like.device} but got {t.dtype} {tuple(t.shape)} "
                             f"on {t.device}")
    return t


def _gamma(gamma, H, dev):
    """The tensor and its type's code."""
    g = nv.require_device_tensor(gamma, "gamma")
    code = nv.dtype_code(g, "gamma")
    if g.numel() != H or g.shape[-1:] != (H,) or g.device != dev:
        kernel_assert(False, f"gamma must hold {H} values on {dev} but got {tuple(g.shape)} on {g.device}")
    return g, code


def _eps(eps):
    eps = float(eps)
    if not eps >= 0:
        kernel_assert(False, f"Epsilon must be positive but got {eps}")
    return eps


def rmsnorm_quant_rows(hidden: torch.Tensor, gamma: Optional[torch.Tensor] = None, eps: float = 1e-6, do_norm: bool = True,
                       residual: Optional[torch.Tensor] = None, code_dtype: torch.dtype = torch.int8):
    """``hidden`` ``[..., H]`` -> codes ``[..., H]`` (``torch.int8`` or ``torch.float8_e4m3fn``) and scales ``[...]`` (fp32), and with
    ``residual`` (hidden's shape and type) ``hidden + residual`` rounded to that type, which is what is normalised.

    y = s / sqrt(mean(s^2) + eps) * gamma (``gamma`` None: ones; ``do_norm=False``: y = s, and no gamma);
    scale = max(max|y|, 2^-100) / M, code = y * (M / max(max|y|, 2^-100)) to nearest, M = 127 or 448.  A row of zeros has codes 0; a row
    whose y is not finite has the scale NaN and codes 0."""
    x, dt, shape = _rows(hidden, "hidden")
    codes_dt = _CODES.get(code_dtype)
    if codes_dt is None:
        kernel_assert(False, f"code_dtype must be int8 or float8_e4m3fn but got {code_dtype}")
    eps = _eps(eps)
    H, dev = shape[-1], x.device
    g, g_dt = None, nv.DT_BF16
    if gamma is not None:
        kernel_assert(do_norm, "gamma must be None without the norm")
        g, g_dt = _gamma(gamma, H, dev)
    r = out_r = None
    if residual is not None:
        r = _alike(residual, "residual", x)
        out_r = torch.empty_like(x)
    codes = torch.empty_like(x, dtype=code_dtype)
    scales = x.new_empty(shape[:-1], dtype=torch.float32)
    rows = scales.numel()
    if rows:
        with nv.on_device(dev):
            rc = nv.lib().moe_rmsnorm_quant_rows(x.data_ptr(), dt, nv.ptr(r), nv.ptr(g), g_dt, 1 if do_norm else 0, eps, rows, H, codes_dt,
                                                 codes.data_ptr(), scales.data_ptr(), nv.ptr(out_r), nv.stream_ptr(dev))
        nv.check(rc, "rmsnorm_quant_rows")
    return (codes, scales) if residual is None else (codes, scales, out_r)


def rmsnorm_quant_rows_bwd(d_normed: torch.Tensor, hidden: torch.Tensor, gamma: Optional[torch.Tensor], eps: float = 1e-6,
                           d_residual: Optional[torch.Tensor] = None):
    """Gradient of the norm from that of its values, ``d_normed`` ``[..., H]``; ``hidden`` is what was normalised (with a residual: the sum
    that came back), of the same type.  The rounding to codes passes gradients on as they are.  ``d_residual``: gradient of the sum
    from its other uses, added.  Returns the gradient of the sum, which is ``hidden``'s and ``residual``'s alike, and that of ``gamma``
    (its shape and type; None without one)."""
    x, dt, shape = _rows(hidden, "hidden")
    d = _alike(d_normed, "d_normed", x)
    r = _alike(d_residual, "d_residual", x) if d_residual is not None else None
    eps = _eps(eps)
    H, dev = shape[-1], x.device
    rows = x.numel() // H
    g, g_dt = _gamma(gamma, H, dev) if gamma is not None else (None, nv.DT_BF16)
    d_x = torch.empty_like(x)
    d_g = torch.empty_like(g) if g is not None else None
    if rows == 0:
        return d_x, d_g.zero_() if d_g is not None else None
    L = nv.lib()
    nbytes = L.moe_rmsnorm_quant_rows_bwd_workspace_bytes(rows, H) if g is not None else 0
    ws = x.new_empty(nbytes // 4, dtype=torch.float32) if nbytes else None
    with nv.on_device(dev):
        rc = L.moe_rmsnorm_quant_rows_bwd(d.data_ptr(), x.data_ptr(), dt, nv.ptr(g), g_dt, nv.ptr(r), eps, rows, H, d_x.data_ptr(),
                                          nv.ptr(d_g), nv.ptr(ws), nbytes, nv.stream_ptr(dev))
    nv.check(rc, "rmsnorm_quant_rows_bwd")
    return d_x, d_g


def dequantize_rows(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """Codes ``[..., H]`` (int8 or float8_e4m3fn) with scales ``[...]`` -> the values they stand for, rounded once to ``dtype``."""
    c = nv.require_device_tensor(codes, "codes")
    code, shape, dev = _CODES.get(c.dtype), c.shape, c.device
    if code is None:
        kernel_assert(False, f"codes must be int8 or float8_e4m3fn but got {c.dtype}")
    if len(shape) < 1 or shape[-1] >= 1 << 24:
        kernel_assert(False, f"codes must have rows of fewer than 2^24 but got {tuple(shape)}")
    s = nv.require_device_tensor(scales, "scales")
    if s.dtype != torch.float32 or s.shape != shape[:-1] or s.device != dev:
        kernel_assert(False, f"scales must be float32 {tuple(shape[:-1])} on {dev} but got {s.dtype} {tuple(s.shape)} on {s.device}")
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        kernel_assert(False, f"dtype must be bfloat16, float16 or float32 but got {dtype}")
    out = torch.empty_like(c, dtype=dtype)
    if out.numel():
        with nv.on_device(dev):
            rc = nv.lib().moe_dequantize_rows(c.data_ptr(), code, s.data_ptr(), s.numel(), shape[-1], out.data_ptr(),
                                              nv.dtype_code(out, "dtype"), nv.stream_ptr(dev))
        nv.check(rc, "dequantize_rows")
    return out
