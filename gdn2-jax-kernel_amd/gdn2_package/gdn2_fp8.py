"""Values in 8-bit floating point with a scale for each block of 128, and products of them:

    q, scale = gdn2_quantize_fp8(x)                    # rows, blocks of 1 x 128
    q, scale = gdn2_quantize_fp8(w, blocks=True)       # a weight, blocks of 128 x 128
    x = gdn2_dequantize_fp8(q, scale, dtype=torch.bfloat16)
    y = gdn2_fp8_matmul(q, scale, w, w_scale, bias=None, out_dtype=torch.bfloat16)
    y = gdn2_fp8_linear(x, w, bias=None)               # autograd

A block's scale is the smallest power of two s with max|t| <= 448 s, and its values are held as
e4m3(t / s) (torch.float8_e4m3fn, ties to even): the one rounding there is.  A block of zeros has
scale 0; one that holds NaN or an infinity has scale NaN and q = 0, so that all that is computed
from it is NaN.  The product takes any float32 scales whose products with each other are zero or
normal float32 numbers, so a weight may come from a checkpoint that was quantised otherwise.

Rows of q start at multiples of 16 bytes: where the width is none, q is a view of a wider
tensor; the scales of rows are laid out block by block (a transposed view).  The product takes both
as they are and copies others.  Quantisation and gdn2_fp8_matmul are inference only: as with
the decode step, their results carry no gradient, whatever the inputs require.  No counterpart
in the reference.
"""
from __future__ import annotations

import torch

from . import _lib
from .gdn2_conv import _floating, _ptr
from .gdn2_fwd import _SUPPORTED_IN, GDN2Error, GDN2ShapeError, _dtype_code, _raise
from .gdn2_norm import _INT_MAX, _as, _as_rows, _forward_mode, _gradients, _row_stride, _tensor

_BLOCK = 128
_E4M3 = torch.float8_e4m3fn


def _count(n):
    """Blocks of n values."""
    return (n + _BLOCK - 1) // _BLOCK


def _empty_q(M, C, dev):
    """e4m3 (M, C), rows at multiples of 16 bytes: the tensor and its row stride."""
    ld = (C + 15) // 16 * 16
    q = torch.empty((M, ld), dtype=_E4M3, device=dev)
    return (q if ld == C else q[:, :C]), ld


def gdn2_quantize_fp8(x, blocks=False):
    """x (..., C) in 8 bits: q (float8_e4m3fn of x's shape) and scale (float32), (..., ceil(C / 128))
    for rows, or with blocks=True for a matrix (N, C) (ceil(N / 128), ceil(C / 128))."""
    what = "gdn2_quantize_fp8"
    _tensor(x, "x", what)
    if x.dim() < 1 or (blocks and x.dim() != 2):
        raise GDN2ShapeError(f"{what}: expected {'a matrix' if blocks else 'rows'}; got "
                             f"{tuple(x.shape)}")
    if x.shape[-1] < 1:
        raise GDN2ShapeError(f"{what}: no columns in {tuple(x.shape)}")
    if not x.is_floating_point():
        raise GDN2Error(f"{what}: x must be floating point; got {x.dtype}")
    if x.dtype not in _SUPPORTED_IN:
        x = x.float()
    rows = _as_rows(x)
    M, C = rows.shape
    q, ld = _empty_q(M, C, x.device)
    kb = _count(C)
    s = torch.empty((_count(M), kb) if blocks else (kb, M), dtype=torch.float32, device=x.device)
    rc = _lib.launch("gdn2_quantize_fp8", x.device, M, C, _dtype_code(rows.dtype), rows.data_ptr(),
                     _row_stride(rows), int(blocks), q.data_ptr(), ld, s.data_ptr(), None, 0, None,
                     None, None)
    if rc:
        _raise(rc, f"{what} (M,C)=({M},{C})")
    if blocks:
        return q, s
    if x.dim() == 2:
        return q, s.t()
    lead = x.shape[:-1]
    return q.unflatten(0, lead) if lead else q.view(x.shape), s.view(kb, *lead).movedim(0, -1)


def _scaled_rows(q, scale, names, what, device, blocks):
    """(q, its rows (M, C), the scale, whether it is one for blocks of 128 x 128), checked.
    blocks: that such scales are allowed."""
    _tensor(q, names[0], what)
    _tensor(scale, names[1], what)
    if q.dtype != _E4M3 or scale.dtype != torch.float32:
        raise GDN2Error(f"{what}: {names[0]} must be float8_e4m3fn and {names[1]} float32; got "
                        f"{q.dtype}, {scale.dtype}")
    if q.device != device or scale.device != device:
        raise GDN2Error(f"{what}: all tensors must live on {device}")
    if q.dim() < 1 or q.shape[-1] < 1:
        raise GDN2ShapeError(f"{what}: no columns in {names[0]} {tuple(q.shape)}")
    per_row = (*q.shape[:-1], _count(q.shape[-1]))
    per_block = (_count(q.shape[0]), per_row[-1]) if blocks and q.dim() == 2 else None
    if scale.shape not in (per_row, per_block):
        more = f" or {per_block}" if per_block else ""
        raise GDN2ShapeError(f"{what}: {names[1]} must have shape {per_row}{more} for "
                             f"{names[0]} {tuple(q.shape)}; got {tuple(scale.shape)}")
    # one row has a scale of its own and is a block of rows: the same
    return _as_rows(q), scale, scale.shape != per_row


def gdn2_dequantize_fp8(q, scale, dtype=torch.bfloat16):
    """The values that q stands for with the scales of its rows, or of its blocks of 128 x 128, in
    float32 or bfloat16."""
    what = "gdn2_dequantize_fp8"
    if dtype not in _SUPPORTED_IN:
        raise GDN2Error(f"{what}: dtype must be float32 or bfloat16; got {dtype}")
    rows, s, blocks = _scaled_rows(q, scale, ("q", "scale"), what, getattr(q, "device", None), True)
    M, C = rows.shape
    s = s if blocks else _by_block(s, M).t()
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    rc = _lib.launch(
        "gdn2_dequantize_fp8", q.device, M, C, _dtype_code(dtype), rows.data_ptr(),
        _row_stride(rows), _BLOCK if blocks else 1, s.data_ptr(),
        (_lib.ctypes.c_longlong * 2)(*s.stride()), out.data_ptr())
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
    wide = torch.empty((M, end), dtype=q.dtype, device=q.device)
    wide[:, :K] = q
    return wide, end


def _by_block(scale, M):
    """Scales (..., blocks) of M rows as (blocks, M), dense; a copy only where they are not laid
    out so."""
    if scale.dim() == 2 and scale.stride() == (1, M):
        return scale.t()
    return scale.movedim(-1, 0).reshape(scale.shape[-1], M).contiguous()


def gdn2_fp8_matmul(q, scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """What q stands for times what the weight stands for, transposed, plus bias.

    q (..., K) float8_e4m3fn with scale (..., ceil(K / 128)); weight (N, K) with weight_scale
    (ceil(N / 128), ceil(K / 128)) or, a scale for each row, (N, ceil(K / 128)); bias (N,) or
    None.  Returns (..., N) in out_dtype (float32 or bfloat16).  For float32 the products of a
    block are added in float32.  For bfloat16 they are added by the 8-bit matrix instruction, which is
    faster: of eight neighbouring products it drops, towards zero, what lies below 2^-13 of the
    largest, so that small products are lost beside large ones that cancel.  A caller who
    needs them takes a float32 result and rounds it.  Blocks are scaled and added in float32 and
    the result is rounded once, for either type.  Inference only."""
    what = "gdn2_fp8_matmul"
    if out_dtype not in _SUPPORTED_IN:
        raise GDN2Error(f"{what}: out_dtype must be float32 or bfloat16; got {out_dtype}")
    dev = getattr(q, "device", None)
    x, sx, _ = _scaled_rows(q, scale, ("q", "scale"), what, dev, False)
    w, sw, blocks = _scaled_rows(weight, weight_scale, ("weight", "weight_scale"), what, dev, True)
    if weight.dim() != 2 or w.shape[1] != x.shape[1]:
        raise GDN2ShapeError(f"{what}: weight must be (N, {x.shape[1]}); got "
                             f"{tuple(weight.shape)}")
    if bias is not None:
        bias = _as(_floating(bias, "bias", (w.shape[0],), dev, what), torch.float32).contiguous()
    (M, K), N = x.shape, w.shape[0]
    sx = _by_block(sx, M)
    sw = sw.contiguous() if blocks else _by_block(sw, N)
    x, ldx = _wide_rows(x)
    w, ldw = _wide_rows(w)
    out = torch.empty((*q.shape[:-1], N), dtype=out_dtype, device=dev)
    rc = _lib.launch(
        "gdn2_fp8_matmul", dev, M, N, K, _dtype_code(out_dtype), x.data_ptr(), ldx,
        sx.data_ptr(), M, w.data_ptr(), ldw, _BLOCK if blocks else 1, sw.data_ptr(),
        _count(K) if blocks else N, _ptr(bias), out.data_ptr())
    if rc:
        _raise(rc, f"{what} (M,N,K)=({M},{N},{K})")
    return out


def _launch_linear(x, weight, bias, need_x, need_w):
    """(y, what the backward needs of x and the weight)"""
    rows, shape, dev, L = _as_rows(x), x.shape, x.device, _lib.lib()
    if weight.stride(1) != 1 and weight.shape[1] != 1:
        weight = weight.contiguous()
    (M, K), N = rows.shape, weight.shape[0]
    bias = None if bias is None else _as(bias, torch.float32).contiguous()
    y = torch.empty((*shape[:-1], N), dtype=x.dtype, device=dev)
    kept = torch.empty(L.gdn2_fp8_linear_kept_bytes(M, N, K, need_x, need_w), dtype=torch.uint8,
                       device=dev) if need_x or need_w else None
    nbytes = L.gdn2_fp8_linear_workspace_bytes(M, N, K, 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = _lib.launch(
        "gdn2_fp8_linear_fwd", dev, M, N, K, _dtype_code(x.dtype), rows.data_ptr(),
        _row_stride(rows), weight.data_ptr(), _row_stride(weight), _ptr(bias), need_x, need_w,
        y.data_ptr(), _ptr(kept), ws.data_ptr(), nbytes)
    if rc:
        _raise(rc, f"gdn2_fp8_linear (M,N,K)=({M},{N},{K})")
    return y, kept


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        # the gradients' operands are made with the forward's: their inputs are read once
        need_x, need_w = ctx.needs_input_grad[:2]
        y, kept = _launch_linear(x, weight, bias, need_x, need_w)
        ctx.save_for_backward(kept)
        ctx.kept, ctx.shape, ctx.dtype = (need_x, need_w), x.shape, x.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        return _gradients(_Fp8Linear._grads, ctx, dy)

    @staticmethod
    def _grads(ctx, dy):
        kept, = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        rows, dev, L = _as_rows(_as(dy, ctx.dtype)), dy.device, _lib.lib()
        (M, N), K = rows.shape, ctx.shape[-1]
        dx = torch.empty(ctx.shape, dtype=ctx.dtype, device=dev) if need_x else None
        dw = torch.empty((N, K), dtype=ctx.dtype, device=dev) if need_w else None
        db = torch.empty(N, dtype=torch.float32, device=dev) if need_b else None
        nbytes = L.gdn2_fp8_linear_workspace_bytes(M, N, K, 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = _lib.launch(
            "gdn2_fp8_linear_bwd", dev, M, N, K, _dtype_code(ctx.dtype), rows.data_ptr(),
            _row_stride(rows), _ptr(kept), *ctx.kept, _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(),
            nbytes)
        if rc:
            _raise(rc, f"gdn2_fp8_linear_bwd (M,N,K)=({M},{N},{K})")
        return dx, dw, db if db is None else _as(db, ctx.bias_dtype)


def gdn2_fp8_linear(x, weight, bias=None):
    """x weight^T + bias as a linear layer that multiplies in 8 bits, for training.

    x (..., K), weight (N, K), bias (N,); x and weight float32 or bfloat16 (mixed or other types
    are widened to float32).  Returns (..., N) in x's type.  Forward: x in rows of 1 x 128, the
    weight in blocks of 128 x 128.  Backward: the gradient of x from the output's in rows and the
    weight's blocks, that of the weight from the output's gradient and x in blocks of 128 tokens;
    the bias's is the sum of the output's gradient as it comes.  All three products add as
    gdn2_fp8_matmul does for results of that type: float32 inputs in float32, bfloat16 ones by the
    8-bit matrix instruction.  Between the passes x and the weight are kept in 8 bits.  Differentiable in x, weight and bias in reverse mode (tangents of
    forward mode raise NotImplementedError): gradients pass through the roundings as if they were
    none.  To serve, quantise the weight once and call gdn2_fp8_matmul."""
    what = "gdn2_fp8_linear"
    _tensor(x, "x", what)
    if not isinstance(weight, torch.Tensor):
        raise TypeError(f"{what}: weight must be a torch tensor")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise GDN2ShapeError(f"{what}: weight must be (N, K) for x (..., K); got "
                             f"{tuple(weight.shape)} for x {tuple(x.shape)}")
    if max(weight.shape) > _INT_MAX:   # ctypes would cut it to 32 bits
        raise GDN2ShapeError(f"{what}: sizes past 2^31 - 1 in {tuple(weight.shape)}")
    if not x.is_floating_point():
        raise GDN2Error(f"{what}: x must be floating point; got {x.dtype}")
    weight = _floating(weight, "weight", weight.shape, x.device, what)
    if bias is not None:
        bias = _floating(bias, "bias", weight.shape[:1], x.device, what)
    t = x.dtype if x.dtype in _SUPPORTED_IN and weight.dtype == x.dtype else torch.float32
    xs, w = _as(x, t), _as(weight, t)
    if x.numel() == 0:   # no values, and gradients of zero
        y = xs @ w.t()
        return _as(y if bias is None else y + bias, x.dtype)
    # tangents go to the autograd function too, which refuses them
    if _forward_mode() or torch.is_grad_enabled() and (
            xs.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)):
        y = _Fp8Linear.apply(xs, w, bias)
    else:
        y, _ = _launch_linear(xs, w, bias, False, False)
    return _as(y, x.dtype)
