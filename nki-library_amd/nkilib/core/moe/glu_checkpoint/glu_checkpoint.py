"""The gated activation ``act(gate) * up`` of an expert with its inputs kept in 8 bits, and its backward pass from them.

The reference keeps ``gate_up_activations_T`` in bf16 for the backward pass (moe_cte.py:145-150).  A record holds the same
values in half the bytes: ``codes`` uint8 ``[R, 2, I]`` (e4m3; gate, then up) and ``scales`` uint8 ``[R, 2, ceil(I/32)]`` (E8M0,
one per 32 neighbours of I), row r as slot r of the block table.  A value is ``code * 2**(scale - 127)``, off by at most half a
step of e4m3 (1/16 of it, or 1/1024 of the scale where that is more); the scale is the smallest power of two that keeps the
largest finite value of its group within 448.  Infinities and NaN become NaN and leave their neighbours alone.

    h, codes, scales = glu_checkpoint(gate_up)                        # gate_up [R, 2, I]: a program's own products
    codes, scales    = pack_gate_up_checkpoint(gate_up_activations_T)  # [N, 2, I, B]: what moe_cte returned
    d_gate_up, h     = glu_checkpoint_bwd(codes, scales, d_h)

Where values are clamped, the record alone does not tell a clamped value from one that is rounded to its limit: see ``clamped`` of
``glu_checkpoint_bwd``.

With ``token_position_to_id`` (one id per row) and ``n_tokens``, rows of padding slots (ids outside ``[0, n_tokens)``) have no part
in a result, whatever they hold, and are zero in every output.

Plain calls, outside of torch's autograd: what they return has no graph, also where an input requires a gradient.
"""

import ctypes
from typing import Optional

import torch

from .... import _native as nv
from ...utils.common_types import ActFnType
from ...utils.kernel_assert import kernel_assert


def _ids(token_position_to_id, n_tokens, R, device):
    if token_position_to_id is None:
        return None, 0
    t = nv.require_device_tensor(token_position_to_id, "token_position_to_id")
    if t.dim() != 1:
        t = t.reshape(-1)
    if t.dtype != torch.int32 or t.numel() != R or t.device != device:
        kernel_assert(False, f"token_position_to_id must be int32 of {R} rows on {device} but is {t.dtype} of {t.numel()} on "
                             f"{t.device}")
    if n_tokens is None or int(n_tokens) < 0:
        kernel_assert(False, "token_position_to_id needs n_tokens")
    return t, int(n_tokens)


def _clamps(gate_upper, gate_lower, up_upper, up_lower):
    mask, values = 0, (ctypes.c_float * 4)()
    for i, (bit, v) in enumerate(((nv.CLAMP_GATE_HI, gate_upper), (nv.CLAMP_GATE_LO, gate_lower), (nv.CLAMP_UP_HI, up_upper),
                                  (nv.CLAMP_UP_LO, up_lower))):
        if v is not None:
            mask |= bit
            values[i] = float(v)
    return mask, values if mask else None


def _act(activation_function):
    if not isinstance(activation_function, ActFnType):
        kernel_assert(False, f"activation_function must be an ActFnType but got {activation_function}")
    return activation_function.value


def _record(codes, scales):
    codes = nv.require_device_tensor(codes, "codes")
    scales = nv.require_device_tensor(scales, "scales")
    if codes.dtype != torch.uint8 or codes.dim() != 3 or codes.shape[1] != 2 or codes.shape[2] < 1:
        kernel_assert(False, f"codes must be uint8 [R, 2, I] but got {codes.dtype} {tuple(codes.shape)}")
    R, _, I = codes.shape
    if scales.dtype != torch.uint8 or scales.shape != (R, 2, (I + 31) // 32) or scales.device != codes.device:
        kernel_assert(False, f"scales must be uint8 [{R}, 2, {(I + 31) // 32}] on {codes.device} but got {scales.dtype} "
                             f"{tuple(scales.shape)} on {scales.device}")
    return codes, scales, R, I


def _new_clamped(R, I, device, wanted):
    return torch.empty((R, 2, (I + 7) // 8), dtype=torch.uint8, device=device) if wanted else None


def _new_record(R, I, device):
    return (torch.empty((R, 2, I), dtype=torch.uint8, device=device),
            torch.empty((R, 2, (I + 31) // 32), dtype=torch.uint8, device=device))


def glu_checkpoint(gate_up: torch.Tensor, activation_function: ActFnType = ActFnType.SiLU,
                   gate_clamp_upper_limit: Optional[float] = None, gate_clamp_lower_limit: Optional[float] = None,
                   up_clamp_upper_limit: Optional[float] = None, up_clamp_lower_limit: Optional[float] = None,
                   token_position_to_id: Optional[torch.Tensor] = None, n_tokens: Optional[int] = None,
                   return_clamped: bool = False):
    """``gate_up`` ``[R, 2, I]`` (bfloat16, float16 or float32) -> ``intermediate`` ``[R, I]`` of its type, ``codes`` and
    ``scales`` of the clamped gate and up values.  The intermediate is computed from the values themselves, not from the
    record.  With ``return_clamped`` also ``clamped`` uint8 ``[R, 2, ceil(I/8)]``, for ``glu_checkpoint_bwd``: bit i of byte v is set
    where value ``8 v + i`` of the row lay at its limit or beyond."""
    x = nv.require_device_tensor(gate_up, "gate_up")
    if x.dim() != 3 or x.shape[1] != 2 or x.shape[2] < 1:
        kernel_assert(False, f"gate_up must be [R, 2, I] but got {tuple(x.shape)}")
    R, _, I = x.shape
    dev = x.device
    dt, act = nv.dtype_code(x, "gate_up"), _act(activation_function)
    ids, n_tokens = _ids(token_position_to_id, n_tokens, R, dev)
    mask, clamps = _clamps(gate_clamp_upper_limit, gate_clamp_lower_limit, up_clamp_upper_limit, up_clamp_lower_limit)
    h = torch.empty((R, I), dtype=x.dtype, device=dev)
    codes, scales = _new_record(R, I, dev)
    clamped = _new_clamped(R, I, dev, return_clamped)
    if R:
        with nv.on_device(dev):
            rc = nv.lib().moe_glu_checkpoint_clamped(x.data_ptr(), dt, R, I, act, mask, clamps, nv.ptr(ids), n_tokens, h.data_ptr(),
                                                     codes.data_ptr(), scales.data_ptr(), nv.ptr(clamped), nv.stream_ptr(dev))
        nv.check(rc, "glu_checkpoint")
    return (h, codes, scales, clamped) if return_clamped else (h, codes, scales)


def pack_gate_up_checkpoint(gate_up_activations_T: torch.Tensor, token_position_to_id: Optional[torch.Tensor] = None,
                            n_tokens: Optional[int] = None, gate_clamp_upper_limit: Optional[float] = None,
                            gate_clamp_lower_limit: Optional[float] = None, up_clamp_upper_limit: Optional[float] = None,
                            up_clamp_lower_limit: Optional[float] = None, return_clamped: bool = False):
    """The bf16 checkpoint ``[N, 2, I, B]`` that ``moe_cte`` returned (projections after scale, bias and clamp) -> ``codes`` and
    ``scales`` of ``R = N * B`` rows.  With ``return_clamped`` and the layer's limits (which have no other use here) also ``clamped``
    uint8 ``[R, 2, ceil(I/8)]``, for ``glu_checkpoint_bwd``: set where the checkpoint holds a limit's bf16, within half a step of
    which (2^-8) it does not tell either."""
    x = nv.require_device_tensor(gate_up_activations_T, "gate_up_activations_T")
    if x.dtype != torch.bfloat16 or x.dim() != 4 or x.shape[1] != 2 or x.shape[2] < 1:
        kernel_assert(False, f"gate_up_activations_T must be bfloat16 [N, 2, I, B] but got {x.dtype} {tuple(x.shape)}")
    N, _, I, B = x.shape
    dev = x.device
    ids, n_tokens = _ids(token_position_to_id, n_tokens, N * B, dev)
    mask, clamps = _clamps(gate_clamp_upper_limit, gate_clamp_lower_limit, up_clamp_upper_limit, up_clamp_lower_limit)
    if mask and not return_clamped:
        kernel_assert(False, "limits are for return_clamped: the checkpoint's values are clamped already")
    codes, scales = _new_record(N * B, I, dev)
    clamped = _new_clamped(N * B, I, dev, return_clamped)
    if N * B:
        with nv.on_device(dev):
            rc = nv.lib().moe_pack_gate_up_checkpoint_clamped(x.data_ptr(), N, I, B, mask, clamps, nv.ptr(ids), n_tokens,
                                                              codes.data_ptr(), scales.data_ptr(), nv.ptr(clamped), nv.stream_ptr(dev))
        nv.check(rc, "pack_gate_up_checkpoint")
    return (codes, scales, clamped) if return_clamped else (codes, scales)


def glu_checkpoint_bwd(codes: torch.Tensor, scales: torch.Tensor, d_intermediate: torch.Tensor,
                       activation_function: ActFnType = ActFnType.SiLU, gate_clamp_upper_limit: Optional[float] = None,
                       gate_clamp_lower_limit: Optional[float] = None, up_clamp_upper_limit: Optional[float] = None,
                       up_clamp_lower_limit: Optional[float] = None, token_position_to_id: Optional[torch.Tensor] = None,
                       n_tokens: Optional[int] = None, return_intermediate: bool = True, clamped: Optional[torch.Tensor] = None):
    """Gradient of ``act(gate) * up`` at the recorded values: ``d_intermediate`` ``[R, I]`` -> ``d_gate_up`` ``[R, 2, I]`` of its
    type and, with ``return_intermediate``, the recomputed ``intermediate`` ``[R, I]`` (the other factor of the down weights'
    gradient; ``None`` without).  Where a recorded value lies at or beyond its limit, its gradient is zero.  A clamped value
    is recorded as its limit rounded to e4m3 (7.2 as 7.0, or 7.5, as the group's scale has it), so the limit is taken as the record
    holds it: no clamped value passes a gradient.  Values that were not clamped but are recorded alike, up to half a step (1/16)
    inside the limit, pass none either: with ``clamped`` as the forward pass returned it, all of those do and what it has marked does
    not."""
    codes, scales, R, I = _record(codes, scales)
    d = nv.require_device_tensor(d_intermediate, "d_intermediate")
    if d.shape != (R, I) or d.device != codes.device:
        kernel_assert(False, f"d_intermediate must be [{R}, {I}] on {codes.device} but is {tuple(d.shape)} on {d.device}")
    dev = d.device
    dt, act = nv.dtype_code(d, "d_intermediate"), _act(activation_function)
    ids, n_tokens = _ids(token_position_to_id, n_tokens, R, dev)
    mask, clamps = _clamps(gate_clamp_upper_limit, gate_clamp_lower_limit, up_clamp_upper_limit, up_clamp_lower_limit)
    if clamped is not None:
        clamped = nv.require_device_tensor(clamped, "clamped")
        if clamped.dtype != torch.uint8 or clamped.shape != (R, 2, (I + 7) // 8) or clamped.device != dev:
            kernel_assert(False, f"clamped must be uint8 [{R}, 2, {(I + 7) // 8}] on {dev} but is {clamped.dtype} "
                                 f"{tuple(clamped.shape)} on {clamped.device}")
    d_gate_up = torch.empty((R, 2, I), dtype=d.dtype, device=dev)
    h = torch.empty((R, I), dtype=d.dtype, device=dev) if return_intermediate else None
    if R:
        with nv.on_device(dev):
            rc = nv.lib().moe_glu_checkpoint_bwd_clamped(codes.data_ptr(), scales.data_ptr(), nv.ptr(clamped), d.data_ptr(), dt, R, I,
                                                         act, mask, clamps, nv.ptr(ids), n_tokens, d_gate_up.data_ptr(), nv.ptr(h),
                                                         nv.stream_ptr(dev))
        nv.check(rc, "glu_checkpoint_bwd")
    return d_gate_up, h


def dequantize_checkpoint(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The values ``[R, 2, I]`` that a record stands for (bfloat16 holds them exactly)."""
    codes, scales, R, I = _record(codes, scales)
    dev = codes.device
    out = torch.empty((R, 2, I), dtype=dtype, device=dev)
    dt = nv.dtype_code(out, "dtype")
    if R:
        with nv.on_device(dev):
            rc = nv.lib().moe_dequantize_checkpoint(codes.data_ptr(), scales.data_ptr(), 2 * R, I, out.data_ptr(), dt,
                                                    nv.stream_ptr(dev))
        nv.check(rc, "dequantize_checkpoint")
    return out
