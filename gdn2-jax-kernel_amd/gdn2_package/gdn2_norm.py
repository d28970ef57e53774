"""RMS norm with the residual's addition:

    y, h = gdn2_rms_norm(x, weight, residual=None, eps=1e-6)        # autograd

h = x + residual, returned in the residual's type (the residual stream), and
y = h w / sqrt(mean(h^2) + eps) over the last axis.  Without a residual h is x itself.
``gdn2_int8.gdn2_rms_norm_int8`` gives y in 8 bits.  No counterpart in the reference.

x is float32 or bfloat16, the residual has x's type or is float32, the weight (C,) is
float32 or bfloat16: then h is rounded to the residual's type first, and y is the norm of
h as it is returned.  Other types are widened to float32, a bfloat16 residual of a float32
x too: then y is the norm of the float32 sum, and h is rounded to the residual's type
only when it is returned.

Float32 arithmetic: squares of values past 1.8e19 overflow, and y is 0 in such a row.
Rows may be strided as long as their values are contiguous.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .gdn2_fwd import _SUPPORTED_IN, GDN2Error, GDN2ShapeError, _dtype_code, _raise


def _tensor(t, name, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch tensor")
    if not t.is_cuda:
        raise GDN2Error(f"{what}: {name} must live on the ROCm device; no CPU path")


def _as(t, dt):
    return t if t.dtype == dt else t.to(dt)


_INT_MAX = 2 ** 31 - 1


def _forward_mode():
    """Whether inputs could carry tangents (a level of forward mode is open)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def _gradients(grads, ctx, *cotangents):
    """grads(ctx, *cotangents); where a graph of it is asked for, its results raise if they are
    differentiated.  once_differentiable sees to that where a cotangent requires a gradient, but
    the results depend on the inputs too, whatever the cotangents are."""
    if not torch.is_grad_enabled():
        return grads(ctx, *cotangents)
    return once_differentiable(grads)(
        ctx, *(c if c is None else c.detach().requires_grad_() for c in cotangents))


def _as_rows(x):
    """x as (M, C) rows of contiguous values; a copy only where there is no such view."""
    C = x.shape[-1]
    if C > _INT_MAX or x.numel() > _INT_MAX * C:   # ctypes would cut them to 32 bits
        raise GDN2ShapeError(f"gdn2: more than 2^31 - 1 rows or columns in {tuple(x.shape)}")
    if x.dim() != 2:
        x = x.reshape(-1, C) if C else x.reshape(0, 0)
    return x if x.stride(1) == 1 or C == 1 else x.contiguous()


def _row_stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _prepare(x, weight, residual, eps, what):
    """(x, residual, weight) of supported types, checked; rows are not formed yet."""
    if not isinstance(weight, torch.Tensor):
        raise TypeError(f"{what}: weight must be a torch tensor")
    _tensor(x, "x", what)
    _tensor(weight, "weight", what)
    if x.dim() < 1 or weight.shape != x.shape[-1:]:
        raise GDN2ShapeError(f"{what}: weight must have the shape of x's last axis; got "
                             f"{tuple(weight.shape)} for x {tuple(x.shape)}")
    if not x.is_floating_point() or not weight.is_floating_point():
        raise GDN2Error(f"{what}: x and weight must be floating point")
    if weight.device != x.device:
        raise GDN2Error(f"{what}: weight must live on {x.device}")
    if not float(eps) >= 0.0:
        raise GDN2Error(f"{what}: eps = {eps!r} must not be negative")
    if residual is not None:
        _tensor(residual, "residual", what)
        if residual.shape != x.shape:
            raise GDN2ShapeError(f"{what}: residual must have x's shape {tuple(x.shape)}; got "
                                 f"{tuple(residual.shape)}")
        if residual.device != x.device or not residual.is_floating_point():
            raise GDN2Error(f"{what}: residual must be floating point, on {x.device}")
    if x.dtype not in _SUPPORTED_IN:
        x = x.float()
    if weight.dtype not in _SUPPORTED_IN:
        weight = weight.float()
    if residual is not None and residual.dtype != x.dtype:
        residual = residual.float()
    return x, weight.contiguous(), residual


def _launch_fwd(x, weight, residual, eps, keep):
    """(y, h, rstd) of x's shape; h None without a residual, rstd of each row if kept."""
    shape, dev = x.shape, x.device
    x = _as_rows(x)
    M, C = x.shape
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    h = rstd = None
    if residual is not None:
        residual = _as_rows(residual)
        h = torch.empty(shape, dtype=residual.dtype, device=dev)
    if keep:
        rstd = torch.empty(M, dtype=torch.float32, device=dev)
    ptr = lambda t: None if t is None else t.data_ptr()
    rc = _lib.launch(
        "gdn2_rms_norm", dev, M, C, _dtype_code(x.dtype),
        _dtype_code(x.dtype if h is None else h.dtype), _dtype_code(weight.dtype), x.data_ptr(),
        _row_stride(x), ptr(residual), 0 if h is None else _row_stride(residual),
        weight.data_ptr(), eps, y.data_ptr(), ptr(h), ptr(rstd))
    if rc:
        _raise(rc, f"gdn2_rms_norm (M,C)=({M},{C})")
    return y, h, rstd


class _RmsNorm(torch.autograd.Function):
    # Shapes are dealt with inside, and the wrapper that refuses second derivatives is called only
    # where they could be asked for: every node and call of a small layer's backward counts.
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = _launch_fwd(x, weight, residual, eps, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.x_dtype, ctx.has_residual = x.dtype, h is not None
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        return _gradients(_RmsNorm._grads, ctx, dy, dh)

    @staticmethod
    def _grads(ctx, dy, dh):
        h, weight, rstd = ctx.saved_tensors
        shape, dev, L = h.shape, h.device, _lib.lib()
        M, C = rstd.shape[0], shape[-1]
        h = h.contiguous()
        dy = None if dy is None else _as(dy, ctx.x_dtype).contiguous()
        dh = None if dh is None else _as(dh, h.dtype).contiguous()
        dx = torch.empty(shape, dtype=ctx.x_dtype, device=dev)
        dr = torch.empty(shape, dtype=h.dtype, device=dev) \
            if ctx.has_residual and h.dtype != ctx.x_dtype else None
        dw = torch.empty(C, dtype=weight.dtype, device=dev)
        nbytes = L.gdn2_rms_norm_bwd_workspace_bytes(M, C)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        ptr = lambda t: None if t is None else t.data_ptr()
        rc = _lib.launch(
            "gdn2_rms_norm_bwd", dev, M, C, _dtype_code(ctx.x_dtype), _dtype_code(h.dtype),
            _dtype_code(weight.dtype), h.data_ptr(), weight.data_ptr(), rstd.data_ptr(), ptr(dy),
            ptr(dh), dx.data_ptr(), ptr(dr), dw.data_ptr(), ws.data_ptr(), nbytes)
        if rc:
            _raise(rc, f"gdn2_rms_norm_bwd (M,C)=({M},{C})")
        return dx, dw, (dx if dr is None else dr) if ctx.has_residual else None, None


def gdn2_rms_norm(x, weight, residual=None, eps=1e-6):
    """(y, h) with h = x + residual (x itself without one) and y = h w / sqrt(mean(h^2) + eps).

    x (..., C) with C <= 16384, weight (C,), residual of x's shape.  y has x's shape and type,
    h the residual's.  Differentiable in x, weight and residual, through y and h, in reverse mode
    (tangents of forward mode raise NotImplementedError).  Shapes and types are checked before
    any launch (GDN2ShapeError, GDN2Error)."""
    what = "gdn2_rms_norm"
    xs, w, rs = _prepare(x, weight, residual, eps, what)
    # tangents go to the autograd function too, which refuses them
    if _forward_mode() or torch.is_grad_enabled() and (
            xs.requires_grad or w.requires_grad or (rs is not None and rs.requires_grad)):
        res = _RmsNorm.apply(xs, w, rs, float(eps))
        y, h = (res, None) if rs is None else res
    else:
        y, h, _ = _launch_fwd(xs, w, rs, float(eps), False)
    if y.dtype != x.dtype:
        y = y.to(x.dtype)
    if h is None:
        return y, x
    return y, h if h.dtype == residual.dtype else h.to(residual.dtype)
