"""Gated linear recurrence, elementwise over the channels:

    h_t = e^{g_t} h_{t-1} + b_t x_t

    out, h_final = gdn2_gated_scan(x, g, b=None, h0=None)          # autograd
    out, state = gdn2_gated_scan_step(x, g, b=None, state=None)    # one token

The recurrent layer that hybrid stacks put between matrix-state (GDN-2) layers;
``g`` is the log decay in GDN-2's convention and must not be positive in use (the
sums of g over any run of tokens have to stay below 88).  ``g = -inf`` at a token (or
below -2.3e38, as masks of float32's or bfloat16's lowest value are) starts a new
sequence there: nothing of what came before, NaN included, enters it, and no gradient
leaves it.  No counterpart in the reference.

Arithmetic is float32.  x and b are float32 or bfloat16 (mixed or other types are
widened to float32), g float32 (or bfloat16 with bfloat16 inputs); ``out`` has x's
type and shape, states are float32.  Inputs may be strided as long as their
channels are contiguous (the parts of one projection's output); others are copied.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .gdn2_fwd import _SUPPORTED_IN, GDN2Error, GDN2ShapeError, _dtype_code, _raise
from .gdn2_norm import _forward_mode, _gradients

_Strides = ctypes.c_longlong * 2


def _types(x, g, b, what):
    """(input type, g's type) of a call, as the GDN-2 forward chooses them."""
    for t in (x, g) if b is None else (x, g, b):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: x, g, b must be torch tensors")
        if not t.is_cuda or t.device != x.device:
            raise GDN2Error(f"{what}: inputs must live on one ROCm device; no CPU path")
        if t.shape != x.shape:
            raise GDN2ShapeError(f"{what}: g and b must have x's shape {tuple(x.shape)}; got "
                                 f"{tuple(t.shape)}")
        if not t.is_floating_point():
            raise GDN2Error(f"{what}: inputs must be floating point; got {t.dtype}")
    dt = x.dtype
    if dt not in _SUPPORTED_IN or (b is not None and b.dtype != dt):
        dt = torch.float32
    bf16 = dt == torch.bfloat16 and g.dtype == torch.bfloat16
    return dt, torch.bfloat16 if bf16 else torch.float32


def _as(t, dt):
    return t if t is None or t.dtype == dt else t.to(dt)


def _state_in(h, shape, device, what, name):
    if not isinstance(h, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch tensor")
    if h.shape != shape:
        raise GDN2ShapeError(f"{what}: {name} must have shape {tuple(shape)}; got "
                             f"{tuple(h.shape)}")
    if h.device != device:
        raise GDN2Error(f"{what}: {name} must live on {device}")
    return _as(h, torch.float32).contiguous()


def _rows(x):
    """(pointer, strides) of a (B,T,C) or (B,T,H,D) tensor, copied where its channels are
    apart.  The copy is returned too, to outlive the launch."""
    if x.is_contiguous():
        return x, x.data_ptr(), None
    if x.dim() == 4:
        x = x.reshape(*x.shape[:2], x.shape[2] * x.shape[3])
    if x.stride(2) != 1 and x.shape[2] != 1:
        x = x.contiguous()
        return x, x.data_ptr(), None
    return x, x.data_ptr(), _Strides(x.stride(0), x.stride(1))


def _sizes(x):
    """(shape, B, T, C)"""
    s = x.shape
    return s, s[0], s[1], s[2] if len(s) == 3 else s[2] * s[3]


def _launch_fwd(x, g, b, h0, keep):
    shape, B, T, C = _sizes(x)
    state = (B, *shape[2:])
    dev, L, code = x.device, _lib.lib(), _dtype_code(x.dtype)
    x, px, sx = _rows(x)
    g, pg, sg = _rows(g)
    pb = sb = None
    if b is not None:
        b, pb, sb = _rows(b)
    out = torch.empty(shape, dtype=x.dtype, device=dev)
    h_final = torch.empty(state, dtype=torch.float32, device=dev)
    kept = ws = None
    if keep:
        kept = torch.empty(L.gdn2_gated_scan_kept_bytes(B, T, C, code) // 4, dtype=torch.float32,
                           device=dev)
    nbytes = L.gdn2_gated_scan_workspace_bytes(B, T, C, code)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = _lib.launch(
        "gdn2_gated_scan_fwd", dev, B, T, C, code, _dtype_code(g.dtype), px, sx, pg, sg, pb, sb,
        None if h0 is None else h0.data_ptr(), out.data_ptr(), h_final.data_ptr(),
        kept.data_ptr() if keep and T else None, None if ws is None else ws.data_ptr(), nbytes)
    if rc:
        _raise(rc, f"gdn2_gated_scan_fwd (B,T,C)=({B},{T},{C})")
    return out, h_final, kept


class _GatedScan(torch.autograd.Function):
    # Shapes are dealt with inside, and the wrapper that refuses second derivatives is called only
    # where they could be asked for: every node and call of a small layer's backward counts.
    @staticmethod
    def forward(ctx, x, g, b, h0):
        out, h_final, kept = _launch_fwd(x, g, b, h0, True)
        ctx.save_for_backward(x, g, b, kept)
        ctx.has_h0 = h0 is not None
        ctx.set_materialize_grads(False)
        return out, h_final

    @staticmethod
    def backward(ctx, dout, dh_final):
        return _gradients(_GatedScan._grads, ctx, dout, dh_final)

    @staticmethod
    def _grads(ctx, dout, dh_final):
        x, g, b, kept = ctx.saved_tensors
        shape, B, T, C = _sizes(x)
        dev, L, code = x.device, _lib.lib(), _dtype_code(x.dtype)
        if T == 0:
            zero = [None if t is None else torch.zeros_like(t) for t in (x, g, b)]
            dh0 = None if not ctx.has_h0 or dh_final is None else dh_final.clone()
            return (*zero, dh0)
        x, px, sx = _rows(x)
        g, pg, sg = _rows(g)
        pb = sb = pd = sd = db = dh0 = ws = None
        if b is not None:
            b, pb, sb = _rows(b)
            db = torch.empty(shape, dtype=b.dtype, device=dev)
        if dout is not None:
            dout, pd, sd = _rows(_as(dout, x.dtype))
        if dh_final is not None:
            dh_final = _as(dh_final, torch.float32).contiguous()
        dx = torch.empty(shape, dtype=x.dtype, device=dev)
        dg = torch.empty(shape, dtype=g.dtype, device=dev)
        if ctx.has_h0:
            dh0 = torch.empty((B, *shape[2:]), dtype=torch.float32, device=dev)
        nbytes = L.gdn2_gated_scan_workspace_bytes(B, T, C, code)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        ptr = lambda t: None if t is None else t.data_ptr()
        rc = _lib.launch(
            "gdn2_gated_scan_bwd", dev, B, T, C, code, _dtype_code(g.dtype), px, sx, pg, sg, pb,
            sb, pd, sd, ptr(dh_final), kept.data_ptr(), dx.data_ptr(), dg.data_ptr(), ptr(db),
            ptr(dh0), ptr(ws), nbytes)
        if rc:
            _raise(rc, f"gdn2_gated_scan_bwd (B,T,C)=({B},{T},{C})")
        return dx, dg, db, dh0


def gdn2_gated_scan(x, g, b=None, h0=None):
    """h_t = e^{g_t} h_{t-1} + b_t x_t over the second axis.

    x, g, b: (B,T,C) or (B,T,H,D), one shape; ``b=None`` stands for ones; h0 (B,C) or
    (B,H,D), default zeros.  Returns ``out`` (all h_t, x's shape and type) and
    ``h_final`` (float32, h0's shape).  Differentiable in x, g, b and h0, through out
    and h_final, in reverse mode (tangents of forward mode raise NotImplementedError); gradients
    come in each input's type.  T may be 0 (h_final = h0).
    Shapes and types are checked before any launch (GDN2ShapeError, GDN2Error)."""
    what = "gdn2_gated_scan"
    dt, gdt = _types(x, g, b, what)
    shape = x.shape
    if len(shape) not in (3, 4):
        raise GDN2ShapeError(f"{what}: expected (B,T,C) or (B,T,H,D) inputs, got {tuple(shape)}")
    if max(_sizes(x)[1:]) >= 2 ** 31:   # ctypes would cut them to 32 bits
        raise GDN2ShapeError(f"{what}: sizes past 2^31 - 1 in {tuple(shape)}")
    state = torch.Size((shape[0], *shape[2:]))
    if h0 is not None:
        h0 = _state_in(h0, state, x.device, what, "h0")
    out_dt = x.dtype
    x, g, b = _as(x, dt), _as(g, gdt), _as(b, dt)
    # tangents go to the autograd function too, which refuses them
    if _forward_mode() or torch.is_grad_enabled() and (
            x.requires_grad or g.requires_grad or (b is not None and b.requires_grad) or
            (h0 is not None and h0.requires_grad)):
        out, h_final = _GatedScan.apply(x, g, b, h0)
    else:
        out, h_final, _ = _launch_fwd(x, g, b, h0, False)
    if out.dtype != out_dt:
        out = out.to(out_dt)
    return out, h_final


def gdn2_gated_scan_step(x, g, b=None, state=None, inplace=False):
    """One token of ``gdn2_gated_scan`` for decoding.

    x, g, b: one shape (B, ...) without a token axis; state: float32 of that shape
    (default zeros).  Returns ``out`` (x's type) and the new state; ``inplace=True``
    updates ``state`` itself, which must then be a contiguous float32 tensor.
    Inference only: as with the decode step, results carry no gradient, whatever the
    inputs require."""
    what = "gdn2_gated_scan_step"
    dt, gdt = _types(x, g, b, what)
    dev, shape = x.device, x.shape
    if inplace:
        if not isinstance(state, torch.Tensor) or state.dtype != torch.float32 or \
                not state.is_contiguous():
            raise GDN2Error(f"{what}: inplace needs a contiguous float32 state")
    h_in = None if state is None else _state_in(state, shape, dev, what, "state")
    out_dt = x.dtype
    x, g = _as(x, dt).contiguous(), _as(g, gdt).contiguous()
    b = None if b is None else _as(b, dt).contiguous()
    h_out = state if inplace else torch.empty(shape, dtype=torch.float32, device=dev)
    out = torch.empty(shape, dtype=dt, device=dev)
    rc = _lib.launch(
        "gdn2_gated_scan_step", dev, x.numel(), _dtype_code(dt), _dtype_code(gdt), x.data_ptr(),
        g.data_ptr(), None if b is None else b.data_ptr(),
        None if h_in is None else h_in.data_ptr(), h_out.data_ptr(), out.data_ptr())
    if rc:
        _raise(rc, f"{what} {tuple(shape)}")
    return _as(out, out_dt), h_out
