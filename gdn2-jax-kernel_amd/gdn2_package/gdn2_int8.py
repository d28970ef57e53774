"""Rows in 8 bits with a scale for each, and their matrix product (serving):

    q, scale, h = gdn2_rms_norm_int8(x, weight, residual=None, eps=1e-6)
    q, scale = gdn2_quantize_int8(x)
    x = gdn2_dequantize_int8(q, scale, dtype=torch.bfloat16)
    y = gdn2_int8_matmul(q, scale, w, w_scale, bias=None, out_dtype=torch.bfloat16)

A row t is held as q = round(127 t / max|t|) (ties to even; in float32, t times 127 (1 / max|t|),
so that a value within three roundings of a tie may go either way) and scale = max|t| / 127;
it stands for q * scale.  A row of zeros has scale 0; one that holds NaN or an infinity
has scale NaN and q = 0, so that all that is computed from it is NaN.  The weight of a
linear layer, (N,K) as torch.nn.Linear holds it, is quantised once with
``gdn2_quantize_int8(weight)``: a scale for each output channel.

Rows of q start at multiples of 16 bytes: where the width is none, q is a view of a wider
tensor.  The product takes such rows as they are and copies others.  Inference only: as with
the decode step, results carry no gradient, whatever the inputs require.  No counterpart in
the reference.
"""
from __future__ import annotations

import torch

from . import _lib
from .gdn2_fwd import _SUPPORTED_IN, GDN2Error, GDN2ShapeError, _dtype_code, _raise
from .gdn2_norm import _as, _as_rows, _prepare, _row_stride, _tensor


def _empty_q(shape, dev):
    """int8 (..., C), rows at multiples of 16 bytes: the tensor and its row stride."""
    C = shape[-1]
    ld = (C + 15) // 16 * 16
    q = torch.empty((*shape[:-1], ld), dtype=torch.int8, device=dev)
    return (q if ld == C else q[..., :C]), ld


def gdn2_rms_norm_int8(x, weight, residual=None, eps=1e-6):
    """``gdn2_rms_norm`` with y in 8 bits: (q int8 of x's shape, scale float32 of x's shape
    without its last axis, h).  q does not depend on the order of any sum.  Inference only."""
    what = "gdn2_rms_norm_int8"
    xs, ws, rs = _prepare(x, weight, residual, eps, what)
    shape, dev = xs.shape, xs.device
    rows = _as_rows(xs)
    M, C = rows.shape
    q, ld = _empty_q(shape, dev)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    h = r_rows = None
    if rs is not None:
        r_rows = _as_rows(rs)
        h = torch.empty(shape, dtype=rs.dtype, device=dev)
    rc = _lib.launch(
        "gdn2_rms_norm_int8", dev, M, C, _dtype_code(rows.dtype),
        _dtype_code(rows.dtype if h is None else h.dtype), _dtype_code(ws.dtype),
        rows.data_ptr(), _row_stride(rows), None if h is None else r_rows.data_ptr(),
        0 if h is None else _row_stride(r_rows), ws.data_ptr(), float(eps), q.data_ptr(), ld,
        scale.data_ptr(), None if h is None else h.data_ptr())
    if rc:
        _raise(rc, f"{what} (M,C)=({M},{C})")
    if h is None:
        return q, scale, x
    return q, scale, h if h.dtype == residual.dtype else h.to(residual.dtype)


def gdn2_quantize_int8(x):
    """Rows of x (..., C), C <= 32768, in 8 bits: (q int8 of x's shape, scale float32 of x's
    shape without its last axis)."""
    what = "gdn2_quantize_int8"
    _tensor(x, "x", what)
    if x.dim() < 1:
        raise GDN2ShapeError(f"{what}: expected rows, got a scalar")
    if not x.is_floating_point():
        raise GDN2Error(f"{what}: x must be floating point; got {x.dtype}")
    if x.dtype not in _SUPPORTED_IN:
        x = x.float()
    rows = _as_rows(x)
    M, C = rows.shape
    q, ld = _empty_q(x.shape, x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rc = _lib.launch(
        "gdn2_quantize_int8", x.device, M, C, _dtype_code(rows.dtype),
        rows.data_ptr(), _row_stride(rows), q.data_ptr(), ld, scale.data_ptr())
    if rc:
        _raise(rc, f"{what} (M,C)=({M},{C})")
    return q, scale


def _int8_rows(q, scale, names, what, device):
    """q as (M, C) int8 rows of contiguous bytes with one scale each, checked."""
    _tensor(q, names[0], what)
    _tensor(scale, names[1], what)
    if q.dtype != torch.int8 or scale.dtype != torch.float32:
        raise GDN2Error(f"{what}: {names[0]} must be int8 and {names[1]} float32; got {q.dtype}, "
                        f"{scale.dtype}")
    if q.dim() < 1 or scale.shape != q.shape[:-1]:
        raise GDN2ShapeError(f"{what}: {names[1]} must have {names[0]}'s shape without its last "
                             f"axis, {tuple(q.shape[:-1])}; got {tuple(scale.shape)}")
    if q.device != device or scale.device != device:
        raise GDN2Error(f"{what}: all tensors must live on {device}")
    return _as_rows(q), scale.contiguous()


def gdn2_dequantize_int8(q, scale, dtype=torch.bfloat16):
    """The values that rows in 8 bits stand for, q * scale, in float32 or bfloat16."""
    what = "gdn2_dequantize_int8"
    if dtype not in _SUPPORTED_IN:
        raise GDN2Error(f"{what}: dtype must be float32 or bfloat16; got {dtype}")
    rows, s = _int8_rows(q, scale, ("q", "scale"), what, getattr(q, "device", None))
    M, C = rows.shape
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    rc = _lib.launch(
        "gdn2_dequantize_int8", q.device, M, C, _dtype_code(dtype),
        rows.data_ptr(), _row_stride(rows), s.data_ptr(), out.data_ptr())
    if rc:
        _raise(rc, f"{what} (M,C)=({M},{C})")
    return out


def _wide_rows(q):
    """(q, row stride) with rows at multiples of 16 bytes, at most 16 MiB apart, that are
    readable up to the next multiple of 16; q itself where it is laid out so."""
    M, K = q.shape
    ld = q.stride(0) if M > 1 else (K + 15) // 16 * 16
    end = (K + 15) // 16 * 16
    if ld % 16 == 0 and end <= ld <= 1 << 24 and q.data_ptr() % 16 == 0 and (
            K == end or M == 0 or
            q.untyped_storage().nbytes() >= q.storage_offset() + (M - 1) * ld + end):
        return q, ld
    wide = torch.empty((M, end), dtype=torch.int8, device=q.device)
    wide[:, :K] = q
    return wide, end


def gdn2_int8_matmul(q, scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """q * scale times (weight * weight_scale)^T, plus bias.

    q (..., K) int8 with scale (...); weight (N, K) int8 with weight_scale (N,); bias (N,)
    or None.  Returns (..., N) in out_dtype (float32 or bfloat16).  The sums over K are
    exact integers (K <= 131071), scaled in float32 and rounded once.  Inference only."""
    what = "gdn2_int8_matmul"
    if out_dtype not in _SUPPORTED_IN:
        raise GDN2Error(f"{what}: out_dtype must be float32 or bfloat16; got {out_dtype}")
    dev = getattr(q, "device", None)
    x, sx = _int8_rows(q, scale, ("q", "scale"), what, dev)
    w, sw = _int8_rows(weight, weight_scale, ("weight", "weight_scale"), what, dev)
    if weight.dim() != 2 or w.shape[1] != x.shape[1]:
        raise GDN2ShapeError(f"{what}: weight must be (N, {x.shape[1]}); got "
                             f"{tuple(weight.shape)}")
    (M, K), N = x.shape, w.shape[0]
    if bias is not None:
        _tensor(bias, "bias", what)
        if tuple(bias.shape) != (N,):
            raise GDN2ShapeError(f"{what}: bias must be ({N},); got {tuple(bias.shape)}")
        if bias.device != dev or not bias.is_floating_point():
            raise GDN2Error(f"{what}: bias must be floating point, on {dev}")
        bias = _as(bias, torch.float32).contiguous()
    x, ldx = _wide_rows(x)
    w, ldw = _wide_rows(w)
    out = torch.empty((*q.shape[:-1], N), dtype=out_dtype, device=dev)
    rc = _lib.launch(
        "gdn2_int8_matmul", dev, M, N, K, _dtype_code(out_dtype),
        x.data_ptr(), ldx, sx.data_ptr(), w.data_ptr(), ldw, sw.data_ptr(),
        None if bias is None else bias.data_ptr(), out.data_ptr())
    if rc:
        _raise(rc, f"{what} (M,N,K)=({M},{N},{K})")
    return out
