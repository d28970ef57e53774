"""C ABI of the gated recurrence, the RMS norm and the 8-bit product (include/gdn2.h), CPU
only: every call below is refused before a launch, or only computes a size."""
import ctypes

import pytest

from gdn2_package import _lib

F32, BF16 = _lib.GDN2_F32, _lib.GDN2_BF16
P = [0x100000 * (i + 1) for i in range(12)]          # never dereferenced
BIG = 2 ** 31 - 1


def strides(*s):
    return (ctypes.c_longlong * 2)(*s)


def scan_fwd(B=2, T=600, C=64, dt=F32, gdt=F32, x=P[0], g=P[1], b=P[2], h0=P[3], out=P[4],
             hf=P[5], kept=P[6], ws=P[7], wsb=1 << 40):
    return _lib.lib().gdn2_gated_scan_fwd(None, B, T, C, dt, gdt, x, None, g, None, b, None, h0,
                                          out, hf, kept, ws, wsb)


def scan_bwd(B=2, T=600, C=64, dt=F32, gdt=F32, kept=P[6], dx=P[4], dg=P[5], db=P[8], ws=P[7],
             wsb=1 << 40, b=P[2], dout=P[3]):
    return _lib.lib().gdn2_gated_scan_bwd(None, B, T, C, dt, gdt, P[0], None, P[1], None, b, None,
                                          dout, None, P[9], kept, dx, dg, db, P[10], ws, wsb)


@pytest.mark.parametrize("f", [scan_fwd, scan_bwd])
def test_scan_refusals(f):
    assert f(B=0) == _lib.ERR_SHAPE and f(C=0) == _lib.ERR_SHAPE and f(T=-1) == _lib.ERR_SHAPE
    assert f(T=BIG) == _lib.ERR_SHAPE and f(C=BIG) == _lib.ERR_SHAPE
    assert f(B=BIG) == _lib.ERR_SHAPE
    assert f(dt=7) == _lib.ERR_DTYPE and f(dt=_lib.GDN2_BF16_F32) == _lib.ERR_DTYPE
    assert f(gdt=BF16) == _lib.ERR_DTYPE and f(dt=BF16, gdt=5) == _lib.ERR_DTYPE
    assert f(ws=None) == _lib.ERR_NULL and f(wsb=16) == _lib.ERR_WORKSPACE
    assert f(b=P[2] + 2) == _lib.ERR_ALIGN
    assert f(dt=BF16, b=P[2] + 1) == _lib.ERR_ALIGN
    assert f(ws=P[7] + 2) == _lib.ERR_ALIGN and f(kept=P[6] + 2) == _lib.ERR_ALIGN
    assert f(ws=P[7] + 8) == _lib.ERR_ALIGN     # 64-bit words, cleared 16 bytes at a time


def test_scan_refusals_by_direction():
    for name in ("x", "g", "out", "hf"):
        assert scan_fwd(**{name: None}) == _lib.ERR_NULL, name
    assert scan_fwd(T=0, hf=None) == _lib.ERR_NULL
    for name in ("kept", "dx", "dg", "db"):
        assert scan_bwd(**{name: None}) == _lib.ERR_NULL, name
    assert scan_bwd(T=0) == _lib.ERR_SEQ_LEN
    assert scan_bwd(dout=P[3] + 2) == _lib.ERR_ALIGN


def test_scan_sizes():
    L = _lib.lib()
    kept, ws = L.gdn2_gated_scan_kept_bytes, L.gdn2_gated_scan_workspace_bytes
    # short axes walk: a kept state for every 128 tokens, no workspace
    assert kept(2, 300, 100, F32) == 3 * 2 * 100 * 4 and ws(2, 300, 100, F32) == 0
    assert kept(2, 0, 100, F32) == 0 and ws(2, 0, 100, F32) == 0
    # long ones: steps of 128 tokens (tiles of 64 channels) or 256 (32); 8 bytes a step and
    # channel, and 64 for each tile's ticket
    assert kept(8, 8192, 768, BF16) == 64 * 8 * 768 * 4
    assert ws(8, 8192, 768, BF16) == 64 * 8 * 768 * 8 + 8 * 12 * 64
    assert kept(8, 8192, 768, F32) == 32 * 8 * 768 * 4
    assert ws(8, 8192, 768, F32) == 32 * 8 * 768 * 8 + 8 * 24 * 64
    assert kept(1, 600, 33, BF16) == 3 * 33 * 4
    # few channels and many tokens: steps of 512 (tiles of 16)
    assert kept(1, 40000, 100, F32) == 79 * 100 * 4
    assert ws(1, 40000, 100, F32) == 79 * 100 * 8 + 7 * 64
    assert ws(1, 600, 33, BF16) == (3 * 33 * 8 + 15) // 16 * 16 + 2 * 64
    for bad in ((0, 5, 5, F32), (5, -1, 5, F32), (5, 5, 0, F32), (5, 5, 5, 9)):
        assert kept(*bad) == 0 and ws(*bad) == 0


def test_scan_step_refusals():
    f = lambda n=8, dt=F32, gdt=F32, x=P[0], g=P[1], out=P[4], ho=P[3], b=None: \
        _lib.lib().gdn2_gated_scan_step(None, n, dt, gdt, x, g, b, None, ho, out)
    assert f(n=-1) == _lib.ERR_SHAPE and f(n=1 << 50) == _lib.ERR_SHAPE
    assert f(n=0) == _lib.OK
    assert f(dt=9) == _lib.ERR_DTYPE and f(gdt=BF16) == _lib.ERR_DTYPE
    for name in ("x", "g", "out", "ho"):
        assert f(**{name: None}) == _lib.ERR_NULL, name
    assert f(b=P[2] + 2) == _lib.ERR_ALIGN


def test_norm_refusals():
    L = _lib.lib()

    def norm(M=4, C=64, xd=F32, rd=F32, wd=F32, x=P[0], r=P[1], w=P[2], eps=1e-6, y=P[3], h=P[4],
             rstd=P[5]):
        return L.gdn2_rms_norm(None, M, C, xd, rd, wd, x, C, r, C, w, eps, y, h, rstd)

    def norm8(M=4, C=64, xd=F32, rd=F32, wd=F32, x=P[0], r=P[1], w=P[2], eps=1e-6, y=P[3], h=P[4],
              ld=None, scale=P[5]):
        ld = (C + 15) // 16 * 16 if ld is None else ld
        return L.gdn2_rms_norm_int8(None, M, C, xd, rd, wd, x, C, r, C, w, eps, y, ld, scale, h)

    def bwd(M=4, C=64, xd=F32, rd=F32, wd=F32, x=P[0], w=P[2], y=P[3], h=P[4], dw=P[6], ws=P[7],
            wsb=1 << 40):
        return L.gdn2_rms_norm_bwd(None, M, C, xd, rd, wd, x, w, P[5], h, None, y, None, dw, ws,
                                   wsb)
    for f in (norm, norm8, bwd):
        assert f(M=-1) == _lib.ERR_SHAPE and f(C=0) == _lib.ERR_SHAPE
        assert f(C=16385) == _lib.ERR_SHAPE
        assert f(xd=3) == _lib.ERR_DTYPE and f(rd=BF16) == _lib.ERR_DTYPE
        assert f(wd=2) == _lib.ERR_DTYPE
        for name in ("x", "w", "y"):
            assert f(**{name: None}) == _lib.ERR_NULL, (f, name)
        assert f(x=P[0] + 2) == _lib.ERR_ALIGN
    for f in (norm, norm8):
        assert f(eps=-1.0) == _lib.ERR_SHAPE and f(eps=float("nan")) == _lib.ERR_SHAPE
        assert f(h=None) == _lib.ERR_NULL and f(M=0) == _lib.OK
    assert norm8(ld=63) == _lib.ERR_SHAPE and norm8(ld=80) == _lib.ERR_ALIGN
    assert norm8(y=P[3] + 8) == _lib.ERR_ALIGN and norm8(scale=None) == _lib.ERR_NULL
    assert bwd(dw=None) == _lib.ERR_NULL and bwd(ws=None) == _lib.ERR_NULL
    assert bwd(wsb=0) == _lib.ERR_WORKSPACE
    size = L.gdn2_rms_norm_bwd_workspace_bytes
    # a row of partial sums for each workgroup: of four waves up to 1024 columns, else of a row
    assert size(10, 64) == 3 * 64 * 4
    assert size(1 << 20, 768) == 512 * 768 * 4 and size(1 << 20, 4096) == 512 * 4096 * 4
    assert size(2000, 4096) == 500 * 4096 * 4 and size(300, 4096) == 256 * 4096 * 4
    assert size(0, 64) == 0 and size(4, 16385) == 0 and size(-1, 4) == 0


def test_int8_refusals():
    L = _lib.lib()

    def mm(M=4, N=8, K=40, od=F32, x=P[0], ldx=48, sx=P[1], w=P[2], ldw=48, sw=P[3], bias=None,
           out=P[4]):
        return L.gdn2_int8_matmul(None, M, N, K, od, x, ldx, sx, w, ldw, sw, bias, out)
    assert mm(M=-1) == _lib.ERR_SHAPE and mm(N=0) == _lib.ERR_SHAPE and mm(K=0) == _lib.ERR_SHAPE
    assert mm(K=131072, ldx=1 << 20, ldw=1 << 20) == _lib.ERR_SHAPE
    assert mm(ldx=40) == _lib.ERR_SHAPE and mm(ldw=32) == _lib.ERR_SHAPE
    assert mm(M=BIG) == _lib.ERR_SHAPE and mm(N=BIG) == _lib.ERR_SHAPE
    assert mm(M=1 << 30, N=1 << 30) == _lib.ERR_SHAPE
    assert mm(ldx=(1 << 24) + 16) == _lib.ERR_SHAPE and mm(ldw=(1 << 24) + 16) == _lib.ERR_SHAPE
    assert mm(N=(1 << 26) + 1) == _lib.ERR_SHAPE and mm(M=1 << 24, N=8200) == _lib.ERR_SHAPE
    assert mm(od=4) == _lib.ERR_DTYPE and mm(M=0) == _lib.OK
    for name in ("x", "sx", "w", "sw", "out"):
        assert mm(**{name: None}) == _lib.ERR_NULL, name
    assert mm(x=P[0] + 8) == _lib.ERR_ALIGN and mm(ldw=56) == _lib.ERR_ALIGN
    assert mm(bias=P[5] + 1) == _lib.ERR_ALIGN and mm(out=P[4] + 2) == _lib.ERR_ALIGN
    q = lambda M=4, C=40, dt=F32, x=P[0], qq=P[1], ld=48, s=P[2]: \
        L.gdn2_quantize_int8(None, M, C, dt, x, C, qq, ld, s)
    assert q(C=32769, ld=32784) == _lib.ERR_SHAPE and q(ld=39) == _lib.ERR_SHAPE
    assert q(ld=64) == _lib.ERR_ALIGN and q(qq=P[1] + 4) == _lib.ERR_ALIGN
    assert q(dt=8) == _lib.ERR_DTYPE and q(x=None) == _lib.ERR_NULL and q(M=0) == _lib.OK
    d = lambda M=4, C=40, dt=F32, qq=P[0], s=P[1], out=P[2]: \
        L.gdn2_dequantize_int8(None, M, C, dt, qq, 48, s, out)
    assert d(C=0) == _lib.ERR_SHAPE and d(C=BIG) == _lib.ERR_SHAPE
    assert d(qq=None) == _lib.ERR_NULL and d(s=None) == _lib.ERR_NULL
    assert d(dt=5) == _lib.ERR_DTYPE and d(out=P[2] + 2) == _lib.ERR_ALIGN


def test_python_refuses_host_tensors():
    """The entry points check types and places before anything else, without a GPU too."""
    import gdn2_package as gp
    import torch
    x = torch.zeros((2, 4, 8))
    for f in (lambda: gp.gdn2_gated_scan(x, x), lambda: gp.gdn2_gated_scan_step(x, x),
              lambda: gp.gdn2_rms_norm(x, x[0, 0]), lambda: gp.gdn2_rms_norm_int8(x, x[0, 0]),
              lambda: gp.gdn2_quantize_int8(x),
              lambda: gp.gdn2_dequantize_int8(x.to(torch.int8), x[..., 0]),
              lambda: gp.gdn2_int8_matmul(x.to(torch.int8), x[..., 0], x[0].to(torch.int8),
                                          x[0, :, 0])):
        with pytest.raises(gp.GDN2Error):
            f()
    for f in (lambda: gp.gdn2_gated_scan(1, x), lambda: gp.gdn2_rms_norm(x, 1),
              lambda: gp.gdn2_quantize_int8(None), lambda: gp.gdn2_int8_matmul(1, x, x, x)):
        with pytest.raises(TypeError):
            f()


def test_rows_past_32_bits_are_refused():
    """ctypes keeps the low 32 bits of a size: 2^32 + 3 rows would run as 3."""
    from gdn2_package import GDN2ShapeError, gdn2_norm
    import torch
    L = _lib.lib()
    assert L.gdn2_rms_norm_bwd_workspace_bytes(2 ** 32 + 3, 8) == \
        L.gdn2_rms_norm_bwd_workspace_bytes(3, 8)
    one = torch.zeros((1, 1, 1))
    for shape in ((2 ** 31, 1, 1), (2 ** 17, 2 ** 15 + 1, 1), (1, 1, 2 ** 32 + 8), (0, 3, 2 ** 31)):
        x = one[:0].expand(shape) if 0 in shape else one.expand(shape)
        with pytest.raises(GDN2ShapeError):
            gdn2_norm._as_rows(x)
    assert gdn2_norm._as_rows(one[0].expand(2 ** 31 - 1, 1)).shape == (2 ** 31 - 1, 1)
