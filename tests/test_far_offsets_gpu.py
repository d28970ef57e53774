"""Short convolution, selective scan and 8-bit floating point over tensors of more than 2^31 elements (and 2^32
bytes): what lies at the far end is what the same values give alone."""
import pytest
import torch

import test_selective_scan_gpu as scan
from test_fp8_gpu import check as check_product, held, product

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def test_conv(dev):
    """A long axis, and the same values as many batch entries; the pieces bit for bit."""
    import gdn2_package as gp
    T, C = 2_820_001, 768
    x = torch.empty((1, T, C), dtype=BF16, device=dev).normal_()
    dy = torch.empty_like(x).normal_()
    assert x.numel() > 2 ** 31
    w, b = torch.randn((C, 4), device=dev), torch.randn(C, device=dev)
    y, last = gp.gdn2_short_conv(x.requires_grad_(), w, b)
    dx, = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        for a in (0, T // 2, T - 500):   # from three tokens before on
            n = max(a - 3, 0)
            part = x[:, n:a + 500].clone().requires_grad_()
            with torch.enable_grad():
                z, end = gp.gdn2_short_conv(part, w, b)
            assert torch.equal(z[:, a - n:], y[:, a:a + 500])
            to = a + 500 if a + 500 == T else a + 497
            dpart, = torch.autograd.grad(z, part, dy[:, n:a + 500])
            assert torch.equal(dpart[:, a - n:to - n], dx[:, a:to])
        assert torch.equal(last, x[:, -3:])
        # the same as batch entries
        entries = x[0, :2_820_000].view(2000, 1410, C)
        e, _ = gp.gdn2_short_conv(entries, w, b)
        for i in (0, 1999):
            assert torch.equal(e[i:i + 1], gp.gdn2_short_conv(entries[i:i + 1], w, b)[0])


def test_scan(dev):
    """Many batch entries: the last of them against float64."""
    B, T, C = 1100, 1000, 2048
    big = lambda: torch.empty((B, T, C), dtype=BF16, device=dev)
    small, _, dout, dh = scan.inputs(1, T, C, 1, 16, BF16, BF16, dev, 5)
    leaf = {}
    for n in scan.NAMES:
        v = small[n]
        if n in ("x", "dt", "z"):
            leaf[n] = big().normal_() if n != "dt" else big().uniform_(0.0, 3.0)
            leaf[n][-1] = v[0]
        elif n in ("B", "C", "h0"):
            leaf[n] = v.expand(B, *v.shape[1:]).contiguous()
        else:
            leaf[n] = v
        leaf[n] = leaf[n].clone().requires_grad_() if n not in ("x", "dt", "z") \
            else leaf[n].requires_grad_()
    assert leaf["x"].numel() > 2 ** 31
    out, h = scan.call(leaf, True)
    douts, dhs = big().normal_(), torch.zeros_like(h)
    douts[-1], dhs[-1] = dout[0], dh[0]
    ref = scan.reference(scan.d64(small), None, True, dout.double(), dh.double())
    scan.check(out[-1:], ref["out"])
    scan.check(h[-1:], ref["h_final"])
    own = [n for n in scan.NAMES if n in ("x", "dt", "B", "C", "z", "h0")]
    for n, g in zip(own, torch.autograd.grad((out, h), [leaf[n] for n in own], (douts, dhs))):
        scan.check(g[-1:], ref[n], 2.5)


def test_eight_bits(dev):
    """Rows in 8 bits, back, their product, and results, of more than 2^31 elements each."""
    import gdn2_package as gp
    M, K, N = 530_001, 4096, 4100
    x = torch.empty((M, K), dtype=BF16, device=dev).normal_()
    w = torch.randn((N, K), device=dev).to(BF16)
    q, s = gp.gdn2_quantize_fp8(x)
    wq, ws = gp.gdn2_quantize_fp8(w, blocks=True)
    wv = held(w.double(), 128, 128)[0]
    y = gp.gdn2_fp8_matmul(q, s, wq, ws)
    back = gp.gdn2_dequantize_fp8(q, s)
    assert min(x.numel(), y.numel()) > 2 ** 31
    for a in (0, M // 2, M - 300):
        v, qv, _ = held(x[a:a + 300].double(), 1, 128)
        assert torch.equal(q[a:a + 300].double(), qv) and torch.equal(back[a:a + 300], v.to(BF16))
        check_product(y[a:a + 300], product(v, wv), K)
