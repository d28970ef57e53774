"""RMS norm with the residual's addition (gdn2_rms_norm, its backward) against float64.

Tolerances.  The mean of the squares is a sum of non-negative terms, 32 in a row a thread
and a tree of at most 11 levels; rstd takes half of that error and three roundings of its
own, y two more: fewer than 32 roundings of 2^-24.  dx is a difference of two such
products, one with another such mean: 64 roundings of the terms' magnitudes.  dw adds at most
256 products in a row.  Results in bfloat16 are rounded once more, 2^-8 of their value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32, F32), (BF16, BF16, F32), (BF16, F32, BF16), (BF16, BF16, BF16)]
# widths on both sides of every row layout, odd ones and multiples of 8 and 16 among them
WIDTHS = [1, 7, 64, 100, 512, 513, 1000, 1024, 1032, 2048, 2049, 4096, 5000, 8192, 8200, 16384]


def close(got, ref, mag, n):
    half = 2.0 ** -8 if got.dtype == BF16 else 0.0
    got = got.detach().double().cpu().numpy()
    excess = np.abs(got - ref) - (n * ULP * mag + half * np.abs(ref) + 1e-37)
    assert np.isfinite(got).all() and excess.max() <= 0.0, float(excess.max())


def make(M, C, types, dev, seed):
    x_dt, r_dt, w_dt = types
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device=dev)
    return rand(M, C).to(x_dt), (3 * rand(M, C)).to(r_dt), (1 + 0.3 * rand(C)).to(w_dt), \
        rand(M, C).to(x_dt), rand(M, C).to(r_dt)


def np64(t):
    return t.detach().double().cpu().numpy()


def backward_ref(h, w, dy, dh, eps=1e-6):
    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n, dn = h * rstd, dy * w
    dx = rstd * (dn - n * (dn * n).mean(-1, keepdims=True)) + dh
    mag = rstd * (np.abs(dn) + np.abs(n) * np.abs(dn * n).mean(-1, keepdims=True)) + np.abs(dh)
    return dx, mag, (dy * n).sum(0), np.abs(dy * n).sum(0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("C", WIDTHS)
def test_forward_and_backward(dev, C, types):
    import gdn2_package as gp
    for M in (1, 6):
        x, r, w, dy, dh = make(M, C, types, dev, C + M)
        leaf = [t.clone().requires_grad_() for t in (x, w, r)]
        y, h = gp.gdn2_rms_norm(leaf[0], leaf[1], residual=leaf[2])
        want_h = (np64(x) + np64(r))
        assert y.dtype == x.dtype and h.dtype == r.dtype
        assert torch.equal(h, torch.tensor(want_h).to(r.dtype).to(dev))   # one exact rounding
        hn, wn = np64(h), np64(w)
        ref = hn * wn / np.sqrt((hn * hn).mean(-1, keepdims=True) + 1e-6)
        close(y, ref, np.abs(ref), 32)
        dx, dw, dr = torch.autograd.grad((y, h), leaf, (dy, dh))
        rdx, mdx, rdw, mdw = backward_ref(hn, wn, np64(dy), np64(dh))
        assert (dx.dtype, dw.dtype, dr.dtype) == (x.dtype, w.dtype, r.dtype)
        close(dx, rdx, mdx, 64)
        close(dr, rdx, mdx, 64)
        close(dw, rdw, mdw, 256)


@pytest.mark.parametrize("types", TYPES[:2])
@pytest.mark.parametrize("M,C", [(5000, 24), (4099, 600), (777, 1000), (1030, 4096)])
def test_many_rows(dev, M, C, types):
    """More rows than groups of threads: every group takes several."""
    import gdn2_package as gp
    x, r, w, dy, dh = make(M, C, types, dev, M)
    leaf = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = gp.gdn2_rms_norm(leaf[0], leaf[1], residual=leaf[2], eps=1e-3)
    hn, wn = np64(h), np64(w)
    ref = hn * wn / np.sqrt((hn * hn).mean(-1, keepdims=True) + 1e-3)
    close(y, ref, np.abs(ref), 32)
    dx, dw, dr = torch.autograd.grad((y, h), leaf, (dy, dh))
    rdx, mdx, rdw, mdw = backward_ref(hn, wn, np64(dy), np64(dh), 1e-3)
    close(dx, rdx, mdx, 64)
    close(dr, rdx, mdx, 64)
    close(dw, rdw, mdw, 256)
    again = torch.autograd.grad(gp.gdn2_rms_norm(*leaf[:2], residual=leaf[2], eps=1e-3),
                                leaf, (dy, dh))
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dw, dr)))   # no order that changes


@pytest.mark.parametrize("use", ["y", "h", "both"])
def test_no_residual_and_single_outputs(dev, use):
    import gdn2_package as gp
    x, r, w, dy, dh = make(9, 40, TYPES[0], dev, 3)
    leaf = [t.clone().requires_grad_() for t in (x, w)]
    y, h = gp.gdn2_rms_norm(*leaf)
    assert h is leaf[0]
    dx, dw = torch.autograd.grad(y, leaf, dy)
    rdx, mdx, rdw, mdw = backward_ref(np64(x), np64(w), np64(dy), 0.0)
    close(dx, rdx, mdx, 64)
    close(dw, rdw, mdw, 256)
    leaf = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = gp.gdn2_rms_norm(*leaf[:2], residual=leaf[2])
    outs = {"y": (y,), "h": (h,), "both": (y, h)}[use]
    cot = {"y": (dy,), "h": (dh,), "both": (dy, dh)}[use]
    dx, dw, dr = torch.autograd.grad(outs, leaf, cot)
    rdx, mdx, rdw, mdw = backward_ref(np64(h), np64(w), np64(dy) * (use != "h"),
                                      np64(dh) * (use != "y"))
    close(dx, rdx, mdx, 64)
    close(dr, rdx, mdx, 64)
    close(dw, rdw, mdw, 256)


def test_gradient_against_differences(dev):
    """<gradient, direction> against central differences of the float64 definition."""
    import gdn2_package as gp
    x, r, w, dy, dh = make(4, 33, TYPES[0], dev, 5)
    leaf = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = gp.gdn2_rms_norm(*leaf[:2], residual=leaf[2])
    got = torch.autograd.grad((y, h), leaf, (dy, dh))
    vals, cy, ch = [np64(t) for t in (x, w, r)], np64(dy), np64(dh)

    def loss(v):
        s = v[0] + v[2]
        return (s * v[1] / np.sqrt((s * s).mean(-1, keepdims=True) + 1e-6) * cy).sum() + \
            (s * ch).sum()
    _, mdx, _, mdw = backward_ref(np64(h), vals[1], cy, ch)
    rng = np.random.default_rng(0)
    for i, mag in enumerate((64 * mdx, 256 * mdw, 64 * mdx)):
        d = rng.standard_normal(vals[i].shape)
        up, down = list(vals), list(vals)
        up[i], down[i] = vals[i] + 1e-5 * d, vals[i] - 1e-5 * d
        diff = (loss(up) - loss(down)) / 2e-5
        # the kernel's bound along d, h's own rounding (2^-23 of the row in the formula, up
        # to 33 of them here), and the differences' step^2 and rounding (1e-6)
        tol = ULP * float((mag * np.abs(d)).sum()) * 2 + 1e-6 * (1 + abs(diff))
        assert abs(float((np64(got[i]) * d).sum()) - diff) <= tol


def test_strided_rows_shapes_and_zero_rows(dev):
    import gdn2_package as gp
    x, r, w, dy, dh = make(24, 80, TYPES[1], dev, 7)
    want = gp.gdn2_rms_norm(x, w, residual=r)
    wide = torch.cat([x, r, x], 1)
    got = gp.gdn2_rms_norm(wide[:, :80], w, residual=wide[:, 80:160])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = torch.cat([x[:, :3], x, r], 1)[:, 3:]          # rows off 16 bytes
    got = gp.gdn2_rms_norm(odd[:, :80], w, residual=odd[:, 80:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = gp.gdn2_rms_norm(x.view(2, 3, 4, 80), w, residual=r.view(2, 3, 4, 80))
    assert got[0].shape == (2, 3, 4, 80) and torch.equal(got[0].view(24, 80), want[0])
    t = x.view(4, 6, 80).transpose(0, 1)                  # no view of rows: copied
    y, _ = gp.gdn2_rms_norm(t, w)
    assert torch.equal(y, gp.gdn2_rms_norm(t.contiguous(), w)[0])
    y, _ = gp.gdn2_rms_norm(torch.zeros_like(x), w)
    assert torch.equal(y, torch.zeros_like(x))            # eps keeps a row of zeros finite
    leaf = [t[:0].clone().requires_grad_() for t in (x, r)]
    wl = w.clone().requires_grad_()
    y, h = gp.gdn2_rms_norm(leaf[0], wl, residual=leaf[1])
    assert y.shape == (0, 80)
    (y.sum() + h.sum()).backward()
    assert torch.equal(wl.grad, torch.zeros_like(wl))


@pytest.mark.parametrize("M,C", [(270000, 16), (66000, 1100)])
def test_more_rows_than_a_grid(dev, M, C):
    """Workgroups that take a row (or four) after another: the same as the rows alone."""
    import gdn2_package as gp
    x, r, w, _, _ = make(M, C, TYPES[1], dev, 1)
    cut = 65536 * (4 if C <= 1024 else 1) - 3
    for f in (gp.gdn2_rms_norm, gp.gdn2_rms_norm_int8):
        whole = f(x, w, residual=r)
        for part in (slice(0, 1000), slice(cut, None)):
            for a, b in zip(whole, f(x[part], w, residual=r[part])):
                assert torch.equal(a[part], b)
    q, s = gp.gdn2_quantize_int8(x)
    back = gp.gdn2_dequantize_int8(q, s)
    for part in (slice(0, 1000), slice(cut, None)):
        qp, sp = gp.gdn2_quantize_int8(x[part])
        assert torch.equal(q[part], qp) and torch.equal(s[part], sp)
        assert torch.equal(back[part], gp.gdn2_dequantize_int8(qp, sp))


def test_other_types(dev):
    import gdn2_package as gp
    x, r, w, dy, dh = make(5, 48, TYPES[0], dev, 9)
    y, h = gp.gdn2_rms_norm(x.half().requires_grad_(), w.half(), residual=r.bfloat16())
    assert y.dtype == torch.float16 and h.dtype == BF16
    hn, wn = np64(x.half()) + np64(r.bfloat16()), np64(w.half())
    ref = hn * wn / np.sqrt((hn * hn).mean(-1, keepdims=True) + 1e-6)
    assert np.abs(np64(y) - ref).max() <= 2.0 ** -10 * np.abs(ref).max()
    y.float().sum().backward()


def test_refusals(dev):
    import gdn2_package as gp
    x, w = torch.randn((4, 16), device=dev), torch.ones(16, device=dev)
    for f in (gp.gdn2_rms_norm, gp.gdn2_rms_norm_int8):
        for bad in (lambda: f(x, w[:8]), lambda: f(x, w, residual=x[:2]),
                    lambda: f(torch.zeros((2, 16385), device=dev), torch.zeros(16385, device=dev)),
                    lambda: f(x[:, :0], w[:0])):
            with pytest.raises(gp.GDN2ShapeError):
                bad()
        for bad in (lambda: f(x.cpu(), w), lambda: f(x, w.cpu()), lambda: f(x, w, residual=x.cpu()),
                    lambda: f(x.int(), w), lambda: f(x, w, eps=-1.0),
                    lambda: f(x, w, eps=float("nan"))):
            with pytest.raises(gp.GDN2Error):
                bad()
        with pytest.raises(TypeError):
            f(x, None)


def test_second_derivative_is_refused(dev):
    """create_graph gives the gradients, and their own gradient raises."""
    import gdn2_package as gp
    x = torch.randn(5, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    plain, = torch.autograd.grad(gp.gdn2_rms_norm(x, w)[0].sum(), (x,))
    dx, = torch.autograd.grad(gp.gdn2_rms_norm(x, w)[0].sum(), (x,), create_graph=True)
    assert torch.equal(dx, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), (x,))


def test_gradients_of_higher_ranks(dev):
    """(B, T, H, D) inputs, x a part of a projection: the gradients have the inputs' shapes."""
    import gdn2_package as gp
    base = torch.randn(2, 7, 3, 192, device=dev)
    r = torch.randn(2, 7, 3, 64, device=dev, requires_grad=True)
    w = (1 + 0.1 * torch.randn(64, device=dev)).requires_grad_()
    dy, dh = torch.randn(2, 7, 3, 64, device=dev), torch.randn(2, 7, 3, 64, device=dev)
    got = []
    for x in (base[..., 64:128], base[..., 64:128].reshape(42, 64)):
        x = x.detach().requires_grad_()
        y, h = gp.gdn2_rms_norm(x, w, r.view(x.shape))
        assert y.shape == h.shape == x.shape
        grads = torch.autograd.grad((y, h), (x, w, r), (dy.view(x.shape), dh.view(x.shape)))
        assert grads[0].shape == x.shape
        got.append(grads)
    for a, b in zip(*got):
        assert torch.equal(a.reshape(b.shape), b)


def test_sizes_past_32_bits_are_refused(dev):
    """More rows (or columns, or tokens) than the C interface counts, without memory behind them."""
    import gdn2_package as gp
    many = 2 ** 32 + 5
    x, one = torch.zeros((1, 1), device=dev), torch.ones(1, device=dev)
    rows, wide = x.expand(many, 1), x.expand(1, many)
    q, w = x.to(torch.int8), torch.ones((4, 1), dtype=torch.int8, device=dev)
    for bad in (lambda: gp.gdn2_rms_norm(rows, one), lambda: gp.gdn2_rms_norm_int8(rows, one),
                lambda: gp.gdn2_rms_norm(rows, one, residual=rows),
                lambda: gp.gdn2_quantize_int8(rows), lambda: gp.gdn2_quantize_int8(wide),
                lambda: gp.gdn2_dequantize_int8(q.expand(many, 1), one.expand(many)),
                lambda: gp.gdn2_dequantize_int8(q.expand(1, many), one),
                lambda: gp.gdn2_int8_matmul(q.expand(many, 1), one.expand(many), w, one.expand(4)),
                lambda: gp.gdn2_int8_matmul(q, one, w[:1].expand(many, 1), one.expand(many)),
                lambda: gp.gdn2_gated_scan(x[None].expand(1, many, 1), x[None].expand(1, many, 1)),
                lambda: gp.gdn2_gated_scan(x[None].expand(many, 1, 1), x[None].expand(many, 1, 1)),
                lambda: gp.gdn2_gated_scan(*[x[None, None].expand(1, 2, 2 ** 16, 2 ** 17)] * 2)):
        with pytest.raises(gp.GDN2ShapeError):
            bad()


def test_tangents_are_refused(dev):
    """Forward mode is not there, and no tangent is dropped without a word."""
    import gdn2_package as gp
    from torch.autograd import forward_ad
    x, r = torch.randn(2, 5, 64, device=dev)
    w = torch.ones(64, device=dev)
    want = gp.gdn2_rms_norm(x, w, residual=r)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            assert all(torch.equal(a, b) for a, b in zip(gp.gdn2_rms_norm(x, w, residual=r), want))
            dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
            for call in (lambda: gp.gdn2_rms_norm(dual(x), w), lambda: gp.gdn2_rms_norm(x, dual(w)),
                         lambda: gp.gdn2_rms_norm(x.half(), w, residual=dual(r))):
                with pytest.raises(NotImplementedError):
                    call()


@pytest.mark.parametrize("residual", [False, True])
def test_a_penalty_on_the_gradient_is_refused(dev, residual):
    """A loss that holds its own gradient raises, also where the cotangent was a constant and the
    rest of the loss could go on without the penalty's part."""
    import gdn2_package as gp
    leaf = [torch.randn(5, 64, device=dev, requires_grad=True) for _ in range(2)]
    w = torch.ones(64, device=dev, requires_grad=True)
    y, _ = gp.gdn2_rms_norm(leaf[0], w, residual=leaf[1] if residual else None)
    loss = y.sum()
    dx, dw = torch.autograd.grad(loss, (leaf[0], w), create_graph=True)
    for penalty in (dx.square().sum(), dw.square().sum()):
        with pytest.raises(RuntimeError):
            (loss + penalty).backward(retain_graph=True)
    for got, want in zip(torch.autograd.grad(loss, (leaf[0], w)), (dx, dw)):
        assert torch.equal(got, want)     # without it nothing is in the way


@pytest.mark.parametrize("x_dt,r_dt", [(F32, BF16), (torch.float16, BF16), (BF16, torch.float16),
                                       (torch.float16, torch.float16), (F32, torch.float64)])
def test_widened_residuals(dev, x_dt, r_dt):
    """A residual of a type that the kernels do not take: y is the norm of the float32 sum, in 8
    bits too, and h is that sum rounded to the residual's type."""
    import gdn2_package as gp
    x, r, w, _, _ = make(7, 104, (x_dt, r_dt, F32), dev, 4)
    y, h = gp.gdn2_rms_norm(x, w, residual=r)
    q, scale, h8 = gp.gdn2_rms_norm_int8(x, w, residual=r)
    assert y.dtype == x_dt and h.dtype == h8.dtype == r_dt
    total = x.float() + r.float()
    assert torch.equal(h, total.to(r_dt)) and torch.equal(h8, h)
    ref = np64(total) * np64(w) / np.sqrt((np64(total) ** 2).mean(-1, keepdims=True) + 1e-6)
    if x_dt == F32:
        close(y, ref, np.abs(ref), 32)
    want, whole = gp.gdn2_rms_norm(total, w)
    assert whole is total and torch.equal(y, want.to(x_dt))
    want = gp.gdn2_rms_norm_int8(total, w)
    assert torch.equal(q, want[0]) and torch.equal(scale, want[1])


@pytest.mark.parametrize("types", [(BF16, BF16, F32), (F32, F32, F32)])
def test_norm_is_that_of_the_returned_stream(dev, types):
    """Residuals that the kernels take: y is the norm of h as it is returned."""
    import gdn2_package as gp
    x, r, w, _, _ = make(7, 104, types, dev, 6)
    y, h = gp.gdn2_rms_norm(x, w, residual=r)
    assert torch.equal(y, gp.gdn2_rms_norm(h, w)[0])
