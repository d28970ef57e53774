"""Short causal convolution over each channel, in front of a mixer or a scan:

    y_t = act(bias + sum_{k < W} weight[k] x_{t - W + 1 + k}),   W = 2, 3 or 4

    y, state = gdn2_short_conv(x, weight, bias=None, state=None)        # autograd
    y, state = gdn2_short_conv_step(x, weight, bias=None, state=None)   # one token

The state holds the last W - 1 inputs, oldest first, in x's type: those of one call continue
the sequence in the next.  A token marked in ``starts`` begins a sequence (a packed batch):
nothing of what came before enters it, NaN included, and no gradient passes it.  No counterpart
in the reference.

Sums are float32.  x is float32 or bfloat16 (other types are widened to float32), weight and
bias are used in float32.  The convolution's x may be strided as long as its channels are contiguous;
otherwise it is copied, as the step's is wherever it is not dense.
"""
from __future__ import annotations

import torch

from . import _lib
from .gdn2_fwd import _SUPPORTED_IN, GDN2Error, GDN2ShapeError, _dtype_code, _raise
from .gdn2_norm import _INT_MAX, _forward_mode, _gradients, _tensor
from .gdn2_scan import _as, _rows, _sizes

_ACTIVATIONS = {None: 0, "silu": 1}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _floating(t, name, shape, device, what):
    """t, checked to be a floating point tensor of that shape there."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch tensor")
    if t.shape != shape:
        raise GDN2ShapeError(f"{what}: {name} must have shape {tuple(shape)}; got "
                             f"{tuple(t.shape)}")
    if t.device != device:
        raise GDN2Error(f"{what}: {name} must live on {device}")
    if not t.is_floating_point():
        raise GDN2Error(f"{what}: {name} must be floating point; got {t.dtype}")
    return t


def _starts(starts, B, T, device, what):
    """``starts`` as dense bytes, checked."""
    if starts is None:
        return None
    if not isinstance(starts, torch.Tensor):
        raise TypeError(f"{what}: starts must be a torch tensor")
    if starts.dtype != torch.bool or tuple(starts.shape) != (B, T):
        raise GDN2ShapeError(f"{what}: starts must be bool ({B}, {T}); got {starts.dtype} "
                             f"{tuple(starts.shape)}")
    if starts.device != device:
        raise GDN2Error(f"{what}: starts must live on {device}")
    return starts.contiguous()


def _prepare(x, weight, bias, state, activation, lead, what):
    """(x, weight, bias, state) of supported types, checked; x has `lead` axes before its
    channels, which may be (C,) or (H, D)."""
    _tensor(x, "x", what)
    if x.dim() not in (lead + 1, lead + 2):
        raise GDN2ShapeError(f"{what}: expected {lead} axes and (C) or (H,D) channels, got "
                             f"{tuple(x.shape)}")
    if not x.is_floating_point():
        raise GDN2Error(f"{what}: x must be floating point; got {x.dtype}")
    if activation not in _ACTIVATIONS:
        raise GDN2Error(f"{what}: activation must be None or 'silu'; got {activation!r}")
    channels = x.shape[lead:]
    if not isinstance(weight, torch.Tensor):
        raise TypeError(f"{what}: weight must be a torch tensor")
    W = weight.shape[-1] if weight.dim() else 0
    if weight.shape[:-1] != channels or not 2 <= W <= 4:
        raise GDN2ShapeError(f"{what}: weight must be (*{tuple(channels)}, W) with W = 2, 3 or 4; "
                             f"got {tuple(weight.shape)}")
    if max(x.shape) > _INT_MAX or channels.numel() > _INT_MAX:   # ctypes would cut them
        raise GDN2ShapeError(f"{what}: sizes past 2^31 - 1 in {tuple(x.shape)}")
    weight = _floating(weight, "weight", weight.shape, x.device, what)
    if bias is not None:
        bias = _floating(bias, "bias", channels, x.device, what)
    if state is not None:
        state = _floating(state, "state", (x.shape[0], W - 1, *channels), x.device, what)
    dt = x.dtype if x.dtype in _SUPPORTED_IN else torch.float32
    f32 = lambda t: None if t is None else _as(t, torch.float32).contiguous()
    return (_as(x, dt), f32(weight), f32(bias),
            None if state is None else _as(state, dt).contiguous())


def _launch_fwd(x, weight, bias, state, starts, silu):
    shape, B, T, C = _sizes(x)
    W = weight.shape[-1]
    code = _dtype_code(x.dtype)
    x, px, sx = _rows(x)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    last = torch.empty((B, W - 1, *shape[2:]), dtype=x.dtype, device=x.device)
    rc = _lib.launch("gdn2_short_conv_fwd", x.device, B, T, C, W, code, silu, px, sx,
                     weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(starts), y.data_ptr(),
                     last.data_ptr())
    if rc:
        _raise(rc, f"gdn2_short_conv (B,T,C,W)=({B},{T},{C},{W})")
    return y, last


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, starts, silu):
        ctx.save_for_backward(x, weight, bias, state, starts)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return _launch_fwd(x, weight, bias, state, starts, silu)

    @staticmethod
    def backward(ctx, dy, dlast):
        return _gradients(_ShortConv._grads, ctx, dy, dlast)

    @staticmethod
    def _grads(ctx, dy, dlast):
        x, weight, bias, state, starts = ctx.saved_tensors
        shape, B, T, C = _sizes(x)
        W, dev, L = weight.shape[-1], x.device, _lib.lib()
        x, px, sx = _rows(x)
        pd = sd = db = ds = None
        if dy is not None:
            dy, pd, sd = _rows(_as(dy, x.dtype))
        if dlast is not None:
            dlast = _as(dlast, x.dtype).contiguous()
        dx = torch.empty(shape, dtype=x.dtype, device=dev)
        dw = torch.empty(weight.shape, dtype=torch.float32, device=dev)
        if bias is not None:
            db = torch.empty(bias.shape, dtype=torch.float32, device=dev)
        if state is not None:
            ds = torch.empty(state.shape, dtype=x.dtype, device=dev)
        nbytes = L.gdn2_short_conv_bwd_workspace_bytes(B, T, C, W)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = _lib.launch(
            "gdn2_short_conv_bwd", dev, B, T, C, W, _dtype_code(x.dtype), ctx.silu, px, sx,
            weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(starts), pd, sd, _ptr(dlast),
            dx.data_ptr(), dw.data_ptr(), _ptr(db), _ptr(ds), ws.data_ptr(), nbytes)
        if rc:
            _raise(rc, f"gdn2_short_conv_bwd (B,T,C,W)=({B},{T},{C},{W})")
        return dx, dw, db, ds, None, None


def gdn2_short_conv(x, weight, bias=None, state=None, activation="silu", starts=None):
    """The convolution over the second axis of x, (B,T,C) or (B,T,H,D).

    weight: x's channel axes and W (oldest tap first); bias: x's channel axes; state (B,W-1,C) or
    (B,W-1,H,D), default zeros; activation "silu" or None; starts: bool (B,T).  Returns y (x's
    shape and type) and the new state (x's type), in which inputs from before the last start are
    zero.  Differentiable in x, weight, bias and state, through y and the new state, in reverse
    mode (tangents of forward mode raise NotImplementedError).  T may be 0 (the state comes
    back)."""
    what = "gdn2_short_conv"
    xs, w, b, s = _prepare(x, weight, bias, state, activation, 2, what)
    B, T = xs.shape[:2]
    starts = _starts(starts, B, T, xs.device, what)
    if xs.numel() == 0:
        last = xs.new_zeros((B, w.shape[-1] - 1, *xs.shape[2:])) if s is None else s.clone()
        return x.clone(), _as(last, x.dtype)
    silu = _ACTIVATIONS[activation]
    # tangents go to the autograd function too, which refuses them
    if _forward_mode() or torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (xs, w, b, s)):
        y, last = _ShortConv.apply(xs, w, b, s, starts, silu)
    else:
        y, last = _launch_fwd(xs, w, b, s, starts, silu)
    return _as(y, x.dtype), _as(last, x.dtype)


def gdn2_short_conv_step(x, weight, bias=None, state=None, activation="silu", inplace=False):
    """One token of ``gdn2_short_conv`` for decoding: x (B,C) or (B,H,D).

    Returns y (x's type) and the new state; ``inplace=True`` updates ``state`` itself, which
    must then be contiguous and of the type that is computed in (x's, or float32).  Inference
    only: as with the decode step, results carry no gradient, whatever the inputs require."""
    what = "gdn2_short_conv_step"
    xs, w, b, s = _prepare(x, weight, bias, state, activation, 1, what)
    if inplace and (state is None or s.data_ptr() != state.data_ptr() or s.dtype != state.dtype
                    or not state.is_contiguous()):
        raise GDN2Error(f"{what}: inplace needs a contiguous state of type {xs.dtype}")
    xs = xs.contiguous()
    B, W = xs.shape[0], w.shape[-1]
    C = xs.shape[1:].numel()
    y = torch.empty(xs.shape, dtype=xs.dtype, device=xs.device)
    new = state if inplace else torch.empty((B, W - 1, *xs.shape[1:]), dtype=xs.dtype,
                                            device=xs.device)
    if xs.numel():
        rc = _lib.launch("gdn2_short_conv_step", xs.device, B, C, W, _dtype_code(xs.dtype),
                         _ACTIVATIONS[activation], xs.data_ptr(), w.data_ptr(), _ptr(b), _ptr(s),
                         new.data_ptr(), y.data_ptr())
        if rc:
            _raise(rc, f"{what} (B,C,W)=({B},{C},{W})")
    return _as(y, x.dtype), new if inplace else _as(new, x.dtype)
