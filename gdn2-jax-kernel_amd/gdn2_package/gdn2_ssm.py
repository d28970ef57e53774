"""Selective state space scan with N states a channel:

    d = softplus(dt + dt_bias)                  (dt_softplus=True; else dt + dt_bias)
    h_t[c,n] = e^{d_t[c] A[c,n]} h_{t-1}[c,n] + d_t[c] x_t[c] B_t[n]
    out_t[c] = (sum_n C_t[n] h_t[c,n] + D[c] x_t[c]) silu(z_t[c])

    out, h_final = gdn2_selective_scan(x, dt, A, B, C, D=None, z=None)              # autograd
    out, state = gdn2_selective_scan_step(x, dt, A, B, C, D=None, z=None, state=h)  # one token

B and C may come in G groups, each shared by C / G neighbouring channels.  A is not positive
and d not negative in use (the sums of d A over any run of tokens have to stay below 88); d = 0
leaves a state as it is.  A token marked in ``starts`` begins a sequence (a packed batch):
nothing of what came before enters it, NaN included, and no gradient passes it.  No
counterpart in the reference.

Arithmetic is float32.  x, B, C and z are float32 or bfloat16 (mixed or other types are widened
to float32), dt is of x's type or float32; A, D, dt_bias and the states are float32.  The scan's
inputs may be strided as long as the values of a token are contiguous (the parts of one projection's
output); others are copied.  The step's are copied wherever they are not dense, those parts too.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .gdn2_conv import _floating, _ptr, _starts
from .gdn2_fwd import _SUPPORTED_IN, GDN2Error, GDN2ShapeError, _dtype_code, _raise
from .gdn2_norm import _INT_MAX, _forward_mode, _gradients, _tensor
from .gdn2_scan import _as

_Ptrs5 = ctypes.c_void_p * 5
_Strides5 = ctypes.c_longlong * 10
_MAX_STATES = 64
_MAX_STRIDE = 2 ** 25   # elements from one token to the next that are read in place


def _f32(t):
    if t is None or t.dtype == torch.float32 and t.is_contiguous():
        return t
    return t.to(torch.float32).contiguous()


def _prepare(x, dt, A, B, C, D, z, dt_bias, state, lead, what):
    """The inputs in the types that the kernels take, checked: x, dt, z (*lead, Ch), B, C
    (*lead, G, N).  x has `lead` axes before its channels."""
    _tensor(x, "x", what)
    if x.dim() != lead + 1:
        raise GDN2ShapeError(f"{what}: x must have {lead + 1} axes; got {tuple(x.shape)}")
    if not x.is_floating_point():
        raise GDN2Error(f"{what}: x must be floating point; got {x.dtype}")
    Ch = x.shape[-1]
    if not isinstance(A, torch.Tensor):
        raise TypeError(f"{what}: A must be a torch tensor")
    if A.dim() != 2 or A.shape[0] != Ch or not 1 <= A.shape[1] <= _MAX_STATES:
        raise GDN2ShapeError(f"{what}: A must be ({Ch}, N) with 1 <= N <= {_MAX_STATES}; got "
                             f"{tuple(A.shape)}")
    if max(x.shape) > _INT_MAX:   # ctypes would cut them to 32 bits
        raise GDN2ShapeError(f"{what}: sizes past 2^31 - 1 in {tuple(x.shape)}")
    N, dev, rows = A.shape[1], x.device, x.shape[:-1]
    A = _floating(A, "A", A.shape, dev, what)
    dt = _floating(dt, "dt", x.shape, dev, what)
    if not isinstance(B, torch.Tensor) or not isinstance(C, torch.Tensor):
        raise TypeError(f"{what}: B and C must be torch tensors")
    if B.dim() == lead + 1:
        B = B.unsqueeze(-2)
    if C.dim() == lead + 1:
        C = C.unsqueeze(-2)
    G = B.shape[-2] if B.dim() == lead + 2 else 0
    if G < 1 or Ch % G:
        raise GDN2ShapeError(f"{what}: B must be (..., N) or (..., G, N) with G dividing {Ch}; got "
                             f"{tuple(B.shape)}")
    B = _floating(B, "B", (*rows, G, N), dev, what)
    C = _floating(C, "C", (*rows, G, N), dev, what)
    if z is not None:
        z = _floating(z, "z", x.shape, dev, what)
    if D is not None:
        D = _floating(D, "D", (Ch,), dev, what)
    if dt_bias is not None:
        dt_bias = _floating(dt_bias, "dt_bias", (Ch,), dev, what)
    if state is not None:
        state = _floating(state, "the state", (x.shape[0], Ch, N), dev, what)
    t = x.dtype
    if t not in _SUPPORTED_IN or B.dtype != t or C.dtype != t or (z is not None and z.dtype != t):
        t = torch.float32
    dt = dt if dt.dtype == t else _as(dt, torch.float32)
    return (_as(x, t), dt, _f32(A), _as(B, t), _as(C, t), _f32(D),
            None if z is None else _as(z, t), _f32(dt_bias), _f32(state))


def _row_operand(t):
    """t with a token's values contiguous, and the elements from one batch entry and one token
    to the next.  Strides of axes of one element say nothing."""
    shape = t.shape
    width = shape[2] if len(shape) == 3 else shape[2] * shape[3]
    if t.is_contiguous():
        return t, (shape[1] * width, width)
    s = t.stride()
    inner = s[-1] == 1 or shape[-1] == 1
    if len(shape) == 4:
        inner = inner and (s[2] == shape[3] or shape[2] == 1)
    if inner and (shape[1] == 1 or s[1] <= _MAX_STRIDE):
        return t, (s[0], s[1] if shape[1] > 1 else width)
    return t.contiguous(), (shape[1] * width, width)


def _operands(x, dt, z, B, C):
    """(the tensors, which must outlive the launch; pointers; strides)"""
    kept, ptrs, strides = [], _Ptrs5(), _Strides5()
    for i, t in enumerate((x, dt, z, B, C)):
        if t is not None:
            t, (strides[2 * i], strides[2 * i + 1]) = _row_operand(t)
            ptrs[i] = t.data_ptr()
            kept.append(t)
    return kept, ptrs, strides


def _sizes(x, B):
    return x.shape[0], x.shape[1], x.shape[2], B.shape[2], B.shape[3]


def _launch_fwd(x, dt, A, B, C, D, z, dt_bias, h0, starts, softplus, keep):
    sizes, dev, L = _sizes(x, B), x.device, _lib.lib()
    held, ptrs, strides = _operands(x, dt, z, B, C)
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    h_final = torch.empty((sizes[0], *A.shape), dtype=torch.float32, device=dev)
    kept = None
    if keep:
        kept = torch.empty(L.gdn2_selective_scan_kept_bytes(*sizes) // 4, dtype=torch.float32,
                           device=dev)
    nbytes = L.gdn2_selective_scan_workspace_bytes(*sizes, 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = _lib.launch(
        "gdn2_selective_scan_fwd", dev, *sizes, _dtype_code(x.dtype), _dtype_code(dt.dtype),
        softplus, ptrs, strides, A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(h0), _ptr(starts),
        out.data_ptr(), h_final.data_ptr(), _ptr(kept), ws.data_ptr(), nbytes)
    if rc:
        _raise(rc, f"gdn2_selective_scan (B,T,C,G,N)={sizes}")
    return out, h_final, kept


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, h0, starts, softplus):
        out, h_final, kept = _launch_fwd(x, dt, A, B, C, D, z, dt_bias, h0, starts, softplus, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, starts, kept)
        ctx.softplus, ctx.has_h0 = softplus, h0 is not None
        ctx.set_materialize_grads(False)
        return out, h_final

    @staticmethod
    def backward(ctx, dout, dh_final):
        return _gradients(_SelectiveScan._grads, ctx, dout, dh_final)

    @staticmethod
    def _grads(ctx, dout, dh_final):
        x, dt, A, B, C, D, z, dt_bias, starts, kept = ctx.saved_tensors
        sizes, dev, L = _sizes(x, B), x.device, _lib.lib()
        held, ptrs, strides = _operands(x, dt, z, B, C)
        so = None
        if dout is not None:
            dout, so = _row_operand(_as(dout, x.dtype))
            so = (ctypes.c_longlong * 2)(*so)
        if dh_final is not None:
            dh_final = _as(dh_final, torch.float32).contiguous()
        like = lambda t, d=None: None if t is None else torch.empty(
            t.shape, dtype=d or t.dtype, device=dev)
        outs = [like(t) for t in (x, dt, z, B, C)]
        dA, dD, dbias = like(A), like(D), like(dt_bias)
        dh0 = torch.empty((sizes[0], *A.shape), dtype=torch.float32, device=dev) \
            if ctx.has_h0 else None
        nbytes = L.gdn2_selective_scan_workspace_bytes(*sizes, 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = _lib.launch(
            "gdn2_selective_scan_bwd", dev, *sizes, _dtype_code(x.dtype), _dtype_code(dt.dtype),
            ctx.softplus, ptrs, strides, A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(starts),
            _ptr(dout), so, _ptr(dh_final), kept.data_ptr(), _Ptrs5(*(_ptr(t) for t in outs)),
            dA.data_ptr(), _ptr(dD), _ptr(dbias), _ptr(dh0), ws.data_ptr(), nbytes)
        if rc:
            _raise(rc, f"gdn2_selective_scan_bwd (B,T,C,G,N)={sizes}")
        dx, ddt, dz, dB, dC = outs
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dh0, None, None


def gdn2_selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, h0=None,
                        starts=None):
    """The scan over the second axis.

    x, dt, z (Bt,T,Ch); A (Ch,N) with N <= 64; B, C (Bt,T,N) or (Bt,T,G,N); D, dt_bias (Ch,);
    h0 (Bt,Ch,N), default zeros; starts bool (Bt,T).  Without D its term, without z the gate is
    left out.  Returns out (x's shape and type) and h_final (float32, h0's shape).
    Differentiable in all of them but starts, through out and h_final, in reverse mode (tangents of
    forward mode raise NotImplementedError); gradients come in each input's type.  T may be 0
    (h_final = h0).  Shapes and types are checked before any launch."""
    what = "gdn2_selective_scan"
    args = _prepare(x, dt, A, B, C, D, z, dt_bias, h0, 2, what)
    starts = _starts(starts, x.shape[0], x.shape[1], x.device, what)
    h = args[-1]
    if x.numel() == 0:
        shape = (x.shape[0], *A.shape)
        return x.clone(), h.clone() if h is not None else torch.zeros(
            shape, dtype=torch.float32, device=x.device)
    softplus = int(bool(dt_softplus))
    # tangents go to the autograd function too, which refuses them
    if _forward_mode() or torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in args):
        out, h_final = _SelectiveScan.apply(*args, starts, softplus)
    else:
        out, h_final, _ = _launch_fwd(*args, starts, softplus, False)
    return _as(out, x.dtype), h_final


def gdn2_selective_scan_step(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False,
                             state=None, inplace=False):
    """One token of ``gdn2_selective_scan`` for decoding: x, dt, z (Bt,Ch), B, C (Bt,N) or
    (Bt,G,N); state (Bt,Ch,N), default zeros.

    Returns out (x's type) and the new state (float32); ``inplace=True`` updates ``state``
    itself, which must then be a contiguous float32 tensor.  Inference only: as with the decode
    step, results carry no gradient, whatever the inputs require."""
    what = "gdn2_selective_scan_step"
    if inplace and (not isinstance(state, torch.Tensor) or state.dtype != torch.float32 or
                    not state.is_contiguous()):
        raise GDN2Error(f"{what}: inplace needs a contiguous float32 state")
    xs, ds, A, B, C, D, zs, dt_bias, h = _prepare(x, dt, A, B, C, D, z, dt_bias, state, 1, what)
    xs, ds, B, C = xs.contiguous(), ds.contiguous(), B.contiguous(), C.contiguous()
    zs = None if zs is None else zs.contiguous()
    Bt, Ch = xs.shape
    G, N = B.shape[1:]
    out = torch.empty(xs.shape, dtype=xs.dtype, device=xs.device)
    new = state if inplace else torch.empty((Bt, Ch, N), dtype=torch.float32, device=xs.device)
    if xs.numel():
        rc = _lib.launch(
            "gdn2_selective_scan_step", xs.device, Bt, Ch, G, N, _dtype_code(xs.dtype),
            _dtype_code(ds.dtype), int(bool(dt_softplus)), xs.data_ptr(), ds.data_ptr(),
            A.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(D), _ptr(zs), _ptr(dt_bias), _ptr(h),
            new.data_ptr(), out.data_ptr())
        if rc:
            _raise(rc, f"{what} (B,C,G,N)=({Bt},{Ch},{G},{N})")
    return _as(out, x.dtype), new
