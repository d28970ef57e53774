"""C ABI of the short convolution, the selective scan and the 8-bit floating-point operators
(include/gdn2.h), CPU only: every call below is refused before a launch, or only computes a size."""
import ctypes

import pytest

from gdn2_package import _lib

F32, BF16 = _lib.GDN2_F32, _lib.GDN2_BF16
P = [0x100000 * (i + 1) for i in range(16)]          # never dereferenced
BIG = 2 ** 31 - 1
E = _lib


def pointers(*p):
    return (ctypes.c_void_p * 5)(*p)


def conv_fwd(B=2, T=60, C=64, W=4, dt=F32, silu=1, x=P[0], w=P[1], bias=P[2], state=P[3], y=P[4],
             last=P[5]):
    return _lib.lib().gdn2_short_conv_fwd(None, B, T, C, W, dt, silu, x, None, w, bias, state, None,
                                          y, last)


def conv_bwd(B=2, T=60, C=64, W=4, dt=F32, silu=1, x=P[0], w=P[1], bias=P[2], state=P[3], dx=P[4],
             dw=P[5], ws=P[6], wsb=1 << 40):
    return _lib.lib().gdn2_short_conv_bwd(None, B, T, C, W, dt, silu, x, None, w, bias, state, None,
                                          P[7], None, P[8], dx, dw, P[9], P[10], ws, wsb)


def conv_step(B=2, C=64, W=4, dt=F32, silu=1, x=P[0], w=P[1], bias=P[2], state=P[3], y=P[4],
              last=P[5]):
    return _lib.lib().gdn2_short_conv_step(None, B, C, W, dt, silu, x, w, bias, state, last, y)


@pytest.mark.parametrize("f", [conv_fwd, conv_bwd, conv_step])
def test_conv_refusals(f):
    assert f(B=-1) == E.ERR_SHAPE and f(C=0) == E.ERR_SHAPE and f(C=BIG) == E.ERR_SHAPE
    assert f(W=1) == E.ERR_SHAPE and f(W=5) == E.ERR_SHAPE
    assert f(dt=2) == E.ERR_DTYPE and f(silu=2) == E.ERR_FLAGS
    for name in ("x", "w"):
        assert f(**{name: None}) == E.ERR_NULL, name
    assert f(x=P[0] + 2) == E.ERR_ALIGN and f(dt=BF16, x=P[0] + 1) == E.ERR_ALIGN
    assert f(w=P[1] + 2) == E.ERR_ALIGN and f(bias=P[2] + 1) == E.ERR_ALIGN
    assert f(state=P[3] + 2) == E.ERR_ALIGN


def test_conv_refusals_by_direction():
    for f in (conv_fwd, conv_bwd):
        assert f(B=0) == E.ERR_SHAPE and f(T=-1) == E.ERR_SHAPE and f(T=BIG) == E.ERR_SHAPE
        assert f(T=0) == E.ERR_SEQ_LEN and f(B=1 << 24, T=1 << 20) == E.ERR_SHAPE
    assert conv_fwd(y=None) == E.ERR_NULL and conv_fwd(last=None) == E.ERR_NULL
    assert conv_fwd(last=P[3]) == E.ERR_FLAGS      # the state is read by other workgroups
    assert conv_step(y=None) == E.ERR_NULL and conv_step(last=None) == E.ERR_NULL
    assert conv_step(B=0) == E.OK
    for name in ("dx", "dw", "ws"):
        assert conv_bwd(**{name: None}) == E.ERR_NULL, name
    assert conv_bwd(wsb=16) == E.ERR_WORKSPACE
    size = _lib.lib().gdn2_short_conv_bwd_workspace_bytes
    assert size(2, 0, 64, 4) == 0 and size(2, 60, 64, 5) == 0 and size(-1, 60, 64, 4) == 0
    # a row of sums for each workgroup: 8 tokens and 4 runs (64 lanes), or 16 (16 lanes)
    assert size(2, 60, 64, 4) == 2 * 2 * 64 * 5 * 4
    assert size(8, 8192, 768, 4) == 8 * 32 * 768 * 5 * 4   # 64 tokens


def ssm_fwd(B=2, T=60, C=64, G=2, N=16, dt=F32, ddt=F32, sp=1, x=P[0], d=P[1], z=P[2], bm=P[3],
            cm=P[4], A=P[5], h0=P[6], out=P[7], hf=P[8], kept=P[9], ws=P[10], wsb=1 << 40,
            strides=None):
    return _lib.lib().gdn2_selective_scan_fwd(
        None, B, T, C, G, N, dt, ddt, sp, pointers(x, d, z, bm, cm), strides, A, P[11], P[12], h0,
        None, out, hf, kept, ws, wsb)


def ssm_bwd(B=2, T=60, C=64, G=2, N=16, dt=F32, ddt=F32, sp=1, x=P[0], d=P[1], z=P[2], bm=P[3],
            cm=P[4], A=P[5], dx=P[7], dz=P[8], dA=P[6], kept=P[9], ws=P[10], wsb=1 << 40,
            strides=None):
    return _lib.lib().gdn2_selective_scan_bwd(
        None, B, T, C, G, N, dt, ddt, sp, pointers(x, d, z, bm, cm), strides, A, P[11], P[12], None,
        P[13], None, None, kept, pointers(dx, P[14], dz, P[15], P[15]), dA, None, None, None, ws,
        wsb)


@pytest.mark.parametrize("f", [ssm_fwd, ssm_bwd])
def test_scan_refusals(f):
    for bad in (dict(B=0), dict(T=-1), dict(C=0), dict(G=0), dict(G=3), dict(G=65), dict(N=0),
                dict(N=65), dict(T=BIG), dict(C=BIG, G=1), dict(B=1 << 20, T=1 << 20),
                dict(C=1 << 24, B=64)):
        assert f(**bad) == E.ERR_SHAPE, bad
    assert f(T=0) == E.ERR_SEQ_LEN
    assert f(dt=2) == E.ERR_DTYPE and f(ddt=BF16) == E.ERR_DTYPE and f(dt=BF16, ddt=5) == E.ERR_DTYPE
    assert f(sp=2) == E.ERR_FLAGS
    for name in ("x", "d", "bm", "cm", "A", "ws", "kept") if f is ssm_bwd else \
            ("x", "d", "bm", "cm", "A", "ws"):
        assert f(**{name: None}) == E.ERR_NULL, name
    assert f(x=P[0] + 2) == E.ERR_ALIGN and f(dt=BF16, bm=P[3] + 1) == E.ERR_ALIGN
    assert f(dt=BF16, d=P[1] + 2) == E.ERR_ALIGN     # float32 dt
    assert f(kept=P[9] + 8) == E.ERR_ALIGN and f(ws=P[10] + 8) == E.ERR_ALIGN
    assert f(wsb=16) == E.ERR_WORKSPACE
    far = (ctypes.c_longlong * 10)(*([1 << 40, 1 << 20] * 5))
    assert f(strides=far, ws=None) == E.ERR_NULL      # those are fine
    far[3] = (1 << 25) + 1
    assert f(strides=far) == E.ERR_SHAPE
    far[3] = -1
    assert f(strides=far) == E.ERR_SHAPE


def test_scan_refusals_by_direction():
    assert ssm_fwd(out=None) == E.ERR_NULL and ssm_fwd(hf=None) == E.ERR_NULL
    assert ssm_fwd(h0=P[8]) == E.ERR_FLAGS            # h0 is read by other workgroups
    assert ssm_bwd(dx=None) == E.ERR_NULL and ssm_bwd(dA=None) == E.ERR_NULL
    assert ssm_bwd(dz=None) == E.ERR_NULL and ssm_bwd(dz=None, z=None, ws=None) == E.ERR_NULL


def test_scan_sizes():
    kept = _lib.lib().gdn2_selective_scan_kept_bytes
    ws = _lib.lib().gdn2_selective_scan_workspace_bytes
    # a state for every 16 tokens, N padded to 16; rows of B and C of 2 groups
    assert kept(2, 33, 10, 2, 9) == 2 * 3 * 10 * 16 * 4 + 2 * 33 * 2 * 2 * 16 * 4
    assert kept(8, 8192, 768, 1, 16) == 8 * 512 * 768 * 16 * 4 + 8 * 8192 * 2 * 16 * 4
    # one chunk: the rows alone, or the partial sums of one tile of a group, of A, and of D and bias
    assert ws(2, 16, 10, 2, 9, 0) == 2 * 16 * 2 * 2 * 16 * 4
    assert ws(2, 16, 10, 2, 9, 1) == 2 * 16 * 2 * 2 * 16 * 4 + 2 * 10 * 16 * 4 + 2 * 2 * 10 * 4
    # chunks of 128 tokens: a state and a sum of steps for each of them
    assert ws(8, 8192, 768, 1, 16, 0) == 8 * 64 * 768 * (16 + 1) * 4 + 8 * 8192 * 2 * 16 * 4
    for bad in ((0, 5, 8, 1, 4), (2, -1, 8, 1, 4), (2, 5, 8, 3, 4), (2, 5, 8, 1, 65)):
        assert kept(*bad) == 0 and ws(*bad, 0) == 0 and ws(*bad, 1) == 0


def test_scan_step_refusals():
    def f(B=2, C=64, G=2, N=16, dt=F32, ddt=F32, sp=0, x=P[0], d=P[1], A=P[2], bm=P[3], cm=P[4],
          h=P[5], out=P[6]):
        return _lib.lib().gdn2_selective_scan_step(None, B, C, G, N, dt, ddt, sp, x, d, A, bm, cm,
                                                   None, None, None, None, h, out)
    for bad in (dict(B=-1), dict(C=0), dict(G=3), dict(N=65), dict(G=0)):
        assert f(**bad) == E.ERR_SHAPE, bad
    assert f(B=0) == E.OK and f(sp=3) == E.ERR_FLAGS and f(dt=7) == E.ERR_DTYPE
    for name in ("x", "d", "A", "bm", "cm", "h", "out"):
        assert f(**{name: None}) == E.ERR_NULL, name
    assert f(h=P[5] + 2) == E.ERR_ALIGN and f(x=P[0] + 2) == E.ERR_ALIGN


def test_fp8_refusals():
    L = _lib.lib()

    def mm(M=4, N=8, K=40, od=F32, x=P[0], ldx=48, sx=P[1], lsx=4, w=P[2], ldw=48, rb=128, sw=P[3],
           lsw=8, bias=None, out=P[4]):
        return L.gdn2_fp8_matmul(None, M, N, K, od, x, ldx, sx, lsx, w, ldw, rb, sw, lsw, bias, out)
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(K=BIG), dict(ldx=40), dict(ldw=32),
                dict(rb=64), dict(lsx=3), dict(lsw=0), dict(rb=1, lsw=7), dict(M=BIG), dict(N=BIG),
                dict(ldx=(1 << 24) + 16), dict(M=1 << 22, N=8200, lsx=1 << 22)):
        assert mm(**bad) == E.ERR_SHAPE, bad
    assert mm(od=4) == E.ERR_DTYPE and mm(M=0) == E.OK
    for name in ("x", "sx", "w", "sw", "out"):
        assert mm(**{name: None}) == E.ERR_NULL, name
    assert mm(x=P[0] + 8) == E.ERR_ALIGN and mm(ldw=56) == E.ERR_ALIGN
    assert mm(bias=P[5] + 1) == E.ERR_ALIGN and mm(out=P[4] + 2) == E.ERR_ALIGN

    def q(M=4, C=40, dt=F32, x=P[0], blocks=0, qq=P[1], ld=48, s=P[2], qt=P[3], ldt=16, st=P[4],
          part=P[5], sums=P[6]):
        return L.gdn2_quantize_fp8(None, M, C, dt, x, C, blocks, qq, ld, s, qt, ldt, st, part, sums)
    for bad in (dict(M=-1), dict(C=0), dict(C=BIG), dict(ld=40), dict(ldt=4), dict(M=BIG)):
        assert q(**bad) == E.ERR_SHAPE, bad
    assert q(dt=8) == E.ERR_DTYPE and q(blocks=2) == E.ERR_FLAGS and q(M=0) == E.OK
    for bad in (dict(x=None), dict(s=None), dict(st=None), dict(qq=None, qt=None), dict(part=None),
                dict(sums=None), dict(qq=None, blocks=1)):
        assert q(**bad) == E.ERR_NULL, bad
    assert q(qq=P[1] + 8) == E.ERR_ALIGN and q(qt=P[3] + 8) == E.ERR_ALIGN
    assert q(x=P[0] + 2) == E.ERR_ALIGN and q(part=P[5] + 2) == E.ERR_ALIGN

    two = (ctypes.c_longlong * 2)(1, 4)
    d = lambda M=4, C=40, dt=F32, qq=P[0], rb=1, s=P[1], out=P[2], st=two: \
        L.gdn2_dequantize_fp8(None, M, C, dt, qq, 48, rb, s, st, out)
    assert d(C=0) == E.ERR_SHAPE and d(C=BIG) == E.ERR_SHAPE and d(rb=16) == E.ERR_SHAPE
    assert d(qq=None) == E.ERR_NULL and d(s=None) == E.ERR_NULL and d(st=None) == E.ERR_NULL
    assert d(dt=5) == E.ERR_DTYPE and d(out=P[2] + 2) == E.ERR_ALIGN and d(M=0) == E.OK


def test_fp8_linear_refusals():
    L = _lib.lib()

    def fwd(M=4, N=8, K=40, dt=F32, x=P[0], w=P[1], y=P[2], kept=P[3], ws=P[4], wsb=1 << 40):
        return L.gdn2_fp8_linear_fwd(None, M, N, K, dt, x, K, w, K, None, 1, 1, y, kept, ws, wsb)

    def bwd(M=4, N=8, K=40, dt=F32, dy=P[0], kept=P[3], kx=1, kw=1, dx=P[1], dw=P[2], ws=P[4],
            wsb=1 << 40):
        return L.gdn2_fp8_linear_bwd(None, M, N, K, dt, dy, N, kept, kx, kw, dx, dw, None, ws, wsb)
    for f in (fwd, bwd):
        for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(M=BIG), dict(N=(1 << 24) + 1),
                    dict(M=1 << 20, N=1 << 16)):
            assert f(**bad) == E.ERR_SHAPE, (f, bad)
        assert f(dt=2) == E.ERR_DTYPE and f(wsb=16) == E.ERR_WORKSPACE
        assert f(kept=None) == E.ERR_NULL and f(ws=None) == E.ERR_NULL
        assert f(kept=P[3] + 8) == E.ERR_ALIGN and f(ws=P[4] + 8) == E.ERR_ALIGN
    assert fwd(M=0) == E.OK and fwd(x=None) == E.ERR_NULL and fwd(w=None) == E.ERR_NULL
    assert fwd(y=None) == E.ERR_NULL and bwd(dy=None) == E.ERR_NULL and bwd(M=0) == E.ERR_SHAPE
    assert bwd(kx=0) == E.ERR_FLAGS and bwd(kw=0) == E.ERR_FLAGS
    kept, ws = L.gdn2_fp8_linear_kept_bytes, L.gdn2_fp8_linear_workspace_bytes
    # x in columns: 300 rows of 208 bytes and two scales each; the weight transposed: 300 rows of 112
    # and, as exponents, 4 bytes each
    assert kept(200, 100, 300, 0, 1) == 300 * 208 + 300 * 2 * 4
    assert kept(200, 100, 300, 1, 0) == 300 * 112 + 300 * 4
    assert kept(200, 100, 300, 1, 1) == kept(200, 100, 300, 0, 1) + kept(200, 100, 300, 1, 0)
    assert kept(200, 100, 300, 0, 0) == 0 and kept(0, 100, 300, 1, 1) == 0
    assert ws(200, 100, 300, 0) == 200 * 304 + 200 * 3 * 4 + 100 * 304 + 100 * 4
    assert ws(200, 100, 300, 1) == 200 * 112 + 800 + 100 * 208 + 100 * 2 * 4 + 2 * 100 * 4


def test_python_refuses_host_tensors():
    """The entry points check types and places before anything else, without a GPU too."""
    import gdn2_package as gp
    import torch
    x, w = torch.zeros((2, 4, 8)), torch.zeros((8, 4))
    q, s = x[0].to(torch.float8_e4m3fn), x[0, :, :1]
    for f in (lambda: gp.gdn2_short_conv(x, w), lambda: gp.gdn2_short_conv_step(x[0], w),
              lambda: gp.gdn2_selective_scan(x, x, w, x[..., :4], x[..., :4]),
              lambda: gp.gdn2_selective_scan_step(x[0], x[0], w, x[0, :, :4], x[0, :, :4]),
              lambda: gp.gdn2_quantize_fp8(x), lambda: gp.gdn2_dequantize_fp8(q, s),
              lambda: gp.gdn2_fp8_matmul(q, s, q, s), lambda: gp.gdn2_fp8_linear(x, w.t())):
        with pytest.raises(gp.GDN2Error):
            f()
    for f in (lambda: gp.gdn2_short_conv(1, w), lambda: gp.gdn2_selective_scan(1, x, w, x, x),
              lambda: gp.gdn2_quantize_fp8(None), lambda: gp.gdn2_fp8_matmul(1, s, q, s),
              lambda: gp.gdn2_fp8_linear(None, w)):
        with pytest.raises(TypeError):
            f()
