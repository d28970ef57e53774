"""Gated linear recurrence (gdn2_gated_scan, its backward, gdn2_gated_scan_step) against
the recurrence in float64.

Tolerances.  Every value is a sum of terms, each multiplied on its way by decays
in (0, 1]; m is the same sum with the terms' magnitudes.  A term passes at most 16 tokens
of a run (two roundings each, and the two of e^g), six compositions and eight waves (three
roundings each) and, more weakly the farther it comes, the steps of 128 tokens or more: fewer
than 128 roundings of 2^-24 where a step's decay is e^-1 or less, as all the inputs here
have.  So 128 * 2^-24 * m; results in bfloat16 are rounded once more, 2^-8 of their value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 128 * 2.0 ** -24


def recurrence(a, u, h0, fresh):
    """All states of h_t = a_t h_{t-1} + u_t, (B,T,C) float64; `fresh`: h_t = u_t."""
    h, out = h0.copy(), np.empty_like(u)
    for t in range(u.shape[1]):
        h = np.where(fresh[:, t], u[:, t], a[:, t] * np.where(fresh[:, t], 0.0, h) + u[:, t])
        out[:, t] = h
    return out


def reference(x, g, b, h0, dout=None, dh_final=None):
    """Outputs, gradients and the magnitudes of both, float64 (B,T,C)."""
    fresh, a = np.isneginf(g), np.exp(g)
    out = recurrence(a, b * x, h0, fresh)
    mag = recurrence(a, np.abs(b * x), np.abs(h0), fresh)
    if dout is None:
        return out, mag
    T = x.shape[1]

    def back(d, e):
        dh = np.empty_like(d)
        for t in reversed(range(T)):
            dh[:, t] = d[:, t] + e
            e = np.where(fresh[:, t], 0.0, a[:, t] * dh[:, t])
        return dh, e
    dh, dh0 = back(dout, dh_final)
    mdh, mdh0 = back(np.abs(dout), np.abs(dh_final))
    before = np.concatenate([h0[:, None], out[:, :-1]], 1)
    mbefore = np.concatenate([np.abs(h0)[:, None], mag[:, :-1]], 1)
    before, mbefore = np.where(fresh, 0.0, before), np.where(fresh, 0.0, mbefore)
    grads = {"x": (b * dh, np.abs(b) * mdh), "g": (a * before * dh, a * mbefore * mdh),
             "b": (x * dh, np.abs(x) * mdh), "h0": (dh0, mdh0)}
    return out, mag, grads


def check(got, ref, mag, n=1):
    """|got - ref| <= n EPS mag (+ the rounding of a bfloat16 result)."""
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0
    got = got.detach().double().cpu().numpy()
    excess = np.abs(got - ref) - (n * EPS * mag + half * np.abs(ref) + 1e-30)
    assert np.isfinite(got).all() and excess.max() <= 0.0, float(excess.max())


def inputs(B, T, C, dtype, gdtype, dev, seed, low=0.01):
    """Tensors on the device and their float64 values (after rounding to the type)."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((B, T, C))
    g = -low - rng.exponential(0.5, (B, T, C)) * rng.uniform(0.01, 1.0, C)
    b = rng.uniform(0.0, 1.0, (B, T, C))
    h0 = rng.standard_normal((B, C))
    put = lambda a, dt: torch.tensor(a, device=dev).to(dt)
    t = [put(x, dtype), put(g, gdtype), put(b, dtype), put(h0, torch.float32)]
    return t, [v.double().cpu().numpy() for v in t]


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
         (torch.bfloat16, torch.bfloat16)]
# one token, the sides of a run, a wave and a step; channels on and off the 4- and 16-wide tiles
SIZES = [(1, 1, 1), (2, 2, 16), (3, 5, 7), (1, 15, 20), (2, 16, 64), (1, 63, 33), (2, 64, 48),
         (1, 65, 128), (2, 255, 30), (1, 256, 36), (3, 257, 17), (1, 1000, 100), (9, 300, 21)]


@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("B,T,C", SIZES)
def test_forward(dev, B, T, C, dtype, gdtype):
    import gdn2_package as gp
    (x, g, b, h0), (xn, gn, bn, hn) = inputs(B, T, C, dtype, gdtype, dev, T + C)
    for bt, ht in ((b, h0), (None, None), (b, None)):
        out, hf = gp.gdn2_gated_scan(x, g, bt, h0=ht)
        ref, mag = reference(xn, gn, np.ones_like(bn) if bt is None else bn,
                             np.zeros_like(hn) if ht is None else hn)
        assert out.dtype == dtype and out.shape == x.shape and hf.dtype == torch.float32
        check(out, ref, mag)
        check(hf, ref[:, -1], mag[:, -1])


@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("B,T,C", SIZES)
def test_backward(dev, B, T, C, dtype, gdtype):
    import gdn2_package as gp
    ts, (xn, gn, bn, hn) = inputs(B, T, C, dtype, gdtype, dev, T + C + 1)
    rng = np.random.default_rng(5)
    dout = torch.tensor(rng.standard_normal((B, T, C)), device=dev).to(dtype)
    dhf = torch.tensor(rng.standard_normal((B, C)), device=dev).float()
    for gate, state in ((True, True), (False, False)):
        use = {"x": ts[0], "g": ts[1]}
        if gate:
            use["b"] = ts[2]
        if state:
            use["h0"] = ts[3]
        leaf = {n: t.clone().requires_grad_() for n, t in use.items()}
        out, hf = gp.gdn2_gated_scan(leaf["x"], leaf["g"], leaf.get("b"), h0=leaf.get("h0"))
        got = torch.autograd.grad((out, hf), list(leaf.values()), (dout, dhf))
        _, _, ref = reference(xn, gn, bn if gate else np.ones_like(bn),
                              hn if state else np.zeros_like(hn), dout.double().cpu().numpy(),
                              dhf.double().cpu().numpy())
        for n, t in zip(leaf, got):
            assert t.dtype == leaf[n].dtype and t.shape == leaf[n].shape
            check(t, *ref[n], n=2)   # products of two sums


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,C", [(1, 2048, 16), (1, 5000, 20), (1, 4097, 7), (2, 9001, 40),
                                   (1, 513, 64), (3, 1025, 200), (2, 1537, 192), (1, 1500, 999),
                                   (2, 700, 1000), (17, 640, 100), (1, 2049, 1024),
                                   (1, 33001, 77), (2, 32769, 64)])
def test_steps_at_once(dev, B, T, C, dtype):
    """Long axes: every step has its workgroup, tiles of 16, 32 and 64 channels."""
    import gdn2_package as gp
    from gdn2_package import _lib
    code = _lib.GDN2_F32 if dtype == torch.float32 else _lib.GDN2_BF16
    assert _lib.lib().gdn2_gated_scan_workspace_bytes(B, T, C, code) > 0
    ts, (xn, gn, bn, hn) = inputs(B, T, C, dtype, torch.float32, dev, T)
    leaf = [t.clone().requires_grad_() for t in ts]
    out, hf = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
    dout, dhf = torch.randn_like(out), torch.randn_like(hf)
    got = torch.autograd.grad((out, hf), leaf, (dout, dhf))
    ref, mag, grads = reference(xn, gn, bn, hn, dout.double().cpu().numpy(),
                                dhf.double().cpu().numpy())
    check(out, ref, mag)
    check(hf, ref[:, -1], mag[:, -1])
    for n, t in zip(("x", "g", "b", "h0"), got):
        check(t, *grads[n], n=2)


@pytest.mark.parametrize("B,T,C", [(1, 20000, 128), (2, 6000, 300), (4, 2000, 1024), (1, 90000, 100)])
def test_same_results_every_time(dev, B, T, C):
    """The hand-over from step to step leaves no trace of who was first."""
    import gdn2_package as gp
    ts, _ = inputs(B, T, C, torch.float32, torch.float32, dev, 1)
    leaf = [t.requires_grad_() for t in ts]
    dout = torch.randn((B, T, C), device=dev)
    first = None
    for _ in range(4):
        out, hf = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
        res = (out, hf, *torch.autograd.grad((out, hf), leaf, (dout, torch.ones_like(hf))))
        first = first or res
        assert all(torch.equal(a, e) for a, e in zip(res, first))


def test_nan_of_any_payload_does_not_stop_the_hand_over(dev):
    """NaN whose bits are all ones (memory filled with 0xFF) in every input."""
    import gdn2_package as gp
    B, T, C = 1, 1200, 96
    x = torch.full((B, T, C), -1, dtype=torch.int32, device=dev).view(torch.float32)
    fine = torch.rand((B, T, C), device=dev)
    for args in ((x, -fine), (fine, x), (fine, -fine, x), (x, x, x)):
        leaf = [t.clone().requires_grad_() for t in args]
        out, hf = gp.gdn2_gated_scan(*leaf)
        grads = torch.autograd.grad((out, hf), leaf, (x, x[:, 0]))
        assert torch.isnan(out).all() and torch.isnan(hf).all()
        assert all(torch.isnan(t).all() for t in grads)


def test_gradient_against_differences(dev):
    """<gradient, direction> against central differences of the float64 recurrence."""
    import gdn2_package as gp
    B, T, C = 2, 70, 9
    ts, vals = inputs(B, T, C, torch.float32, torch.float32, dev, 11)
    rng = np.random.default_rng(12)
    dout, dhf = rng.standard_normal((B, T, C)), rng.standard_normal((B, C))
    f32 = lambda a: torch.tensor(a, device=dev).float()
    dout, dhf = (f32(a).double().cpu().numpy() for a in (dout, dhf))
    leaf = [t.clone().requires_grad_() for t in ts]
    out, hf = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
    got = torch.autograd.grad((out, hf), leaf, (f32(dout), f32(dhf)))
    _, _, grads = reference(*vals, dout, dhf)

    def loss(v):
        o = recurrence(np.exp(v[1]), v[2] * v[0], v[3], np.zeros(v[0].shape, bool))
        return (o * dout).sum() + (o[:, -1] * dhf).sum()
    step = 1e-5
    for i, n in enumerate(("x", "g", "b", "h0")):
        d = rng.standard_normal(vals[i].shape)
        up, down = list(vals), list(vals)
        up[i], down[i] = vals[i] + step * d, vals[i] - step * d
        diff = (loss(up) - loss(down)) / (2 * step)
        mine = float((got[i].double().cpu().numpy() * d).sum())
        # the kernel's bound along d, and the differences' own step^2 and rounding (1e-6)
        tol = 2 * EPS * float((grads[n][1] * np.abs(d)).sum()) + 1e-6 * (1 + abs(diff))
        assert abs(mine - diff) <= tol, (n, mine, diff, tol)


@pytest.mark.parametrize("T,C", [(500, 24), (2500, 5), (1300, 1100)])
def test_fresh_starts(dev, T, C):
    """g = -inf starts a sequence: equal to separate calls, NaN and infinities before
    it stay there, and no gradient crosses it."""
    import gdn2_package as gp
    (x, g, b, h0), _ = inputs(1, T, C, torch.float32, torch.float32, dev, T)
    cuts = [0, 1, 2, 130, 255, 256, 257, 400, T]
    g[:, cuts[1:-1]] = -torch.inf
    g[:, cuts[2]] = torch.finfo(torch.float32).min      # masks' lowest value: as -inf
    x[:, 131:140] = torch.nan
    x[:, 200, 0] = torch.inf
    leaf = [t.clone().requires_grad_() for t in (x, g, b, h0)]
    out, hf = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
    dout = torch.randn_like(out)
    got = torch.autograd.grad((out, hf), leaf, (dout, torch.zeros_like(hf)))
    for s, e in zip(cuts[:-1], cuts[1:]):
        if s <= 130 < e:
            continue
        first = h0[:1].double().cpu().numpy() if s == 0 else np.zeros((1, C))
        part = [v[:, s:e].double().cpu().numpy() for v in (x, g, b)]
        ref, mag, grads = reference(*part, first, dout[:, s:e].double().cpu().numpy(),
                                    np.zeros((1, C)))
        check(out[:, s:e], ref, mag)
        for n, t in zip(("x", "g", "b"), got):
            check(t[:, s:e], *grads[n], n=2)
    assert torch.isnan(out[:, 131:255]).all() and torch.isfinite(out[:, 255:]).all()
    assert torch.isfinite(got[3]).all()


def test_decays_that_underflow(dev):
    """Finite decays below the exponent's range give zero factors, not fresh starts; long
    runs whose products underflow stay finite."""
    import gdn2_package as gp
    B, T, C = 1, 700, 20
    (x, g, b, h0), (xn, gn, bn, hn) = inputs(B, T, C, torch.float32, torch.float32, dev, 3)
    g[:, ::3] = -300.0
    g[:, 1::3, :5] = -1e30
    gn = g.double().cpu().numpy()
    leaf = [t.clone().requires_grad_() for t in (x, g, b, h0)]
    out, hf = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
    dout = torch.randn_like(out)
    got = torch.autograd.grad(out, leaf, dout)
    ref, mag, grads = reference(xn, gn, bn, hn, dout.double().cpu().numpy(), np.zeros((B, C)))
    check(out, ref, mag)
    for n, t in zip(("x", "g", "b", "h0"), got):
        check(t, *grads[n], n=2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_inputs(dev, dtype):
    """The parts of one projection's output, a sliced time axis, a transposed copy, a
    shared (broadcast) g and an odd storage offset."""
    import gdn2_package as gp
    B, T, H, D = 2, 300, 3, 8
    C = H * D
    proj = torch.randn((B, T, 3 * C), device=dev).to(dtype)
    x, g, b = proj[..., :C], -proj[..., C:2 * C].abs() - 0.01, proj[..., 2 * C:]
    want = gp.gdn2_gated_scan(x.contiguous(), g.contiguous(), b.contiguous())
    for got in (gp.gdn2_gated_scan(x, g, b),
                gp.gdn2_gated_scan(x.transpose(1, 2).contiguous().transpose(1, 2), g, b)):
        assert all(torch.equal(a, e) for a, e in zip(got, want))
    o4, h4 = gp.gdn2_gated_scan(*(t.unflatten(-1, (H, D)) for t in (x, g, b)))
    assert o4.shape == (B, T, H, D) and h4.shape == (B, H, D)
    assert torch.equal(o4.flatten(2), want[0]) and torch.equal(h4.flatten(1), want[1])
    got = gp.gdn2_gated_scan(*(t[:, 40:200] for t in (x, g, b)))
    want = gp.gdn2_gated_scan(*(t[:, 40:200].contiguous() for t in (x, g, b)))
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    odd = torch.randn(B * T * C + 1, device=dev).to(dtype)[1:].view(B, T, C)
    got = gp.gdn2_gated_scan(odd, g, b)
    want = gp.gdn2_gated_scan(odd.clone(), g, b)
    assert all(torch.allclose(a, e, rtol=2.0 ** -7, atol=1e-5) for a, e in zip(got, want))


def test_gradient_of_a_shared_decay(dev):
    """One g for all the channels of a head: its gradient is the sum over them."""
    import gdn2_package as gp
    B, T, H, D = 2, 100, 3, 16
    x = torch.randn((B, T, H, D), device=dev)
    g1 = (-torch.rand((B, T, H, 1), device=dev) - 0.01).requires_grad_()
    out, _ = gp.gdn2_gated_scan(x, g1.expand(B, T, H, D))
    out.square().sum().backward()
    g2 = g1.detach().expand(B, T, H, D).clone().requires_grad_()
    out2, _ = gp.gdn2_gated_scan(x, g2)
    out2.square().sum().backward()
    assert torch.equal(out, out2)
    ref = g2.grad.double().sum(-1, keepdim=True)
    mag = g2.grad.double().abs().sum(-1, keepdim=True)
    assert ((g1.grad.double() - ref).abs() <= D * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (32, 768), (5, 2, 12)])
def test_step(dev, shape, dtype, gdtype):
    import gdn2_package as gp
    rng = np.random.default_rng(1)
    put = lambda a, dt: torch.tensor(a, device=dev).to(dt)
    x, b = put(rng.standard_normal(shape), dtype), put(rng.uniform(0, 1, shape), dtype)
    g, h = put(-rng.exponential(0.5, shape), gdtype), put(rng.standard_normal(shape), torch.float32)
    g.view(-1)[0] = -torch.inf
    hn = h.double().cpu().numpy().copy()
    h.view(-1)[0] = torch.nan          # dropped by the fresh start
    hn.reshape(-1)[0] = 0.0
    before = h.clone()
    xn, bn, gn = (t.double().cpu().numpy() for t in (x, b, g))
    for bt in (b, None):
        out, new = gp.gdn2_gated_scan_step(x, g, bt, state=h)
        u = xn * (bn if bt is not None else 1.0)
        check(new, np.exp(gn) * hn + u, np.exp(gn) * np.abs(hn) + np.abs(u))
        check(out, np.exp(gn) * hn + u, np.exp(gn) * np.abs(hn) + np.abs(u))
        assert torch.equal(h.isnan(), before.isnan()) and new.data_ptr() != h.data_ptr()
    out2, same = gp.gdn2_gated_scan_step(x, g, None, state=h, inplace=True)
    assert same.data_ptr() == h.data_ptr() and torch.equal(h, new) and torch.equal(out, out2)
    out3, new3 = gp.gdn2_gated_scan_step(x, g, b)
    check(new3, xn * bn, np.abs(xn * bn))


def test_step_beyond_a_grid(dev):
    """More values than the launch has threads."""
    import gdn2_package as gp
    n = 65536 * 1024 + 4000
    x, h = torch.randn(n, device=dev).bfloat16(), torch.randn(n, device=dev)
    g = -torch.rand(n, device=dev).bfloat16()
    out, new = gp.gdn2_gated_scan_step(x, g, state=h)
    for part in (slice(0, 5000), slice(n - 9000, n)):
        a, b = gp.gdn2_gated_scan_step(x[part], g[part], state=h[part])
        assert torch.equal(out[part], a) and torch.equal(new[part], b)


def test_prefix_then_steps_equal_the_scan(dev):
    import gdn2_package as gp
    B, T, C = 2, 40, 12
    (x, g, b, h0), (xn, gn, bn, hn) = inputs(B, T, C, torch.float32, torch.float32, dev, 2)
    _, h = gp.gdn2_gated_scan(x[:, :30], g[:, :30], b[:, :30], h0=h0)
    ref, mag = reference(xn, gn, bn, hn)
    for t in range(30, T):
        out, h = gp.gdn2_gated_scan_step(x[:, t], g[:, t], b[:, t], state=h)
        check(out, ref[:, t], mag[:, t])


def test_other_types_and_empty_axis(dev):
    import gdn2_package as gp
    x = torch.randn((2, 9, 8), device=dev, dtype=torch.float16).requires_grad_()
    g = -torch.rand((2, 9, 8), device=dev)
    out, hf = gp.gdn2_gated_scan(x, g, torch.ones_like(x, dtype=torch.bfloat16))
    assert out.dtype == torch.float16 and hf.dtype == torch.float32
    out.float().sum().backward()
    assert x.grad.dtype == torch.float16
    h0 = torch.randn((2, 8), device=dev, requires_grad=True)
    out, hf = gp.gdn2_gated_scan(x[:, :0], g[:, :0], h0=h0)
    assert out.shape == (2, 0, 8) and torch.equal(hf, h0)
    hf.sum().backward()
    assert torch.equal(h0.grad, torch.ones_like(h0))
    with torch.no_grad():
        _, hf = gp.gdn2_gated_scan(x[:, :0], g[:, :0])
    assert torch.equal(hf, torch.zeros((2, 8), device=dev))


def test_only_one_output_used(dev):
    """The cotangent of the output that is not used counts as zero."""
    import gdn2_package as gp
    (x, g, b, h0), (xn, gn, bn, hn) = inputs(1, 300, 8, torch.float32, torch.float32, dev, 8)
    zero = np.zeros_like(hn)
    for pick in (0, 1):
        leaf = [t.clone().requires_grad_() for t in (x, g, b, h0)]
        res = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])[pick]
        res.sum().backward()
        one = np.ones_like(xn)
        _, _, ref = reference(xn, gn, bn, hn, one if pick == 0 else 0 * one,
                              zero if pick == 0 else zero + 1)
        for n, t in zip(("x", "g", "b", "h0"), leaf):
            check(t.grad, *ref[n], n=2)


def test_other_stream_and_graph(dev):
    """On a stream that is not the current default, and replayed from a captured graph."""
    import gdn2_package as gp
    x, b = torch.randn((2, 700, 40), device=dev), torch.rand((2, 700, 40), device=dev)
    g = -torch.rand((2, 700, 40), device=dev) - 0.01
    want = gp.gdn2_gated_scan(x, g, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gp.gdn2_gated_scan(x, g, b)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gp.gdn2_gated_scan(x, g, b)
    for k in range(3):
        x.normal_()
        want = gp.gdn2_gated_scan(x, g, b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, want)), k


def test_refusals(dev):
    import gdn2_package as gp
    x = torch.randn((2, 5, 8), device=dev)
    g = -torch.rand_like(x)
    for bad in (lambda: gp.gdn2_gated_scan(x[0], g[0]),
                lambda: gp.gdn2_gated_scan(x, g[:, :4]),
                lambda: gp.gdn2_gated_scan(x, g, g[..., :4]),
                lambda: gp.gdn2_gated_scan(x, g, h0=torch.zeros((2, 7), device=dev)),
                lambda: gp.gdn2_gated_scan(x[:0], g[:0]),
                lambda: gp.gdn2_gated_scan_step(x, g, state=x[0])):
        with pytest.raises(gp.GDN2ShapeError):
            bad()
    for bad in (lambda: gp.gdn2_gated_scan(x.cpu(), g.cpu()),
                lambda: gp.gdn2_gated_scan(x, g.cpu()),
                lambda: gp.gdn2_gated_scan(x.int(), g),
                lambda: gp.gdn2_gated_scan(x, g, h0=torch.zeros((2, 8))),
                lambda: gp.gdn2_gated_scan_step(x, g, inplace=True),
                lambda: gp.gdn2_gated_scan_step(x, g, state=x.bfloat16(), inplace=True)):
        with pytest.raises(gp.GDN2Error):
            bad()
    with pytest.raises(TypeError):
        gp.gdn2_gated_scan(x, [1.0])
    leaf = x.clone().requires_grad_()
    out, _ = gp.gdn2_gated_scan(leaf, g)
    first, = torch.autograd.grad(out.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):   # no second derivative, and it says so
        first.sum().backward()


def test_second_derivative_is_refused(dev):
    """create_graph gives the gradients, and their own gradient raises."""
    import gdn2_package as gp
    x = torch.randn(2, 9, 16, device=dev, requires_grad=True)
    g = -torch.rand(2, 9, 16, device=dev)
    plain, = torch.autograd.grad(gp.gdn2_gated_scan(x, g)[0].sum(), (x,))
    dx, = torch.autograd.grad(gp.gdn2_gated_scan(x, g)[0].sum(), (x,), create_graph=True)
    assert torch.equal(dx, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), (x,))


# walked in tiles of 16 (4 channels a thread, and one) and 64; steps at once in tiles of 16, 32, 64
STARTS = [(1, 500, 24), (1, 470, 5), (200, 402, 33), (48, 450, 240), (1, 33000, 64),
          (1, 33001, 7), (1, 2500, 40), (2, 1300, 77), (1, 1400, 1100), (1, 1201, 1027)]


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,C", STARTS)
def test_no_decay_passes_a_fresh_start(dev, B, T, C, dtype, bad):
    """NaN and +inf in g: the sequences before and after theirs are what they are alone, states
    and gradients, wherever in a run, a wave or a step the starts and the bad tokens stand."""
    import gdn2_package as gp
    (x, g, b, h0), _ = inputs(B, T, C, dtype, torch.float32, dev, T)
    # sequences start at `cuts`; bad tokens at one's end, right after its start, at several
    # places, and all through one that is longer than a step
    cuts, spoilt = [0, 3, 41, 100, 130, 200, 390], {1: [40], 3: [101], 5: [203, 257, 388]}
    if T > 1200:
        cuts += [400, 1030, 1100]
        spoilt[7] = range(401, 1030)
    cuts += [T - 5, T]
    spoilt[len(cuts) - 2] = [T - 3]
    g[:, cuts[1:-1]] = -torch.inf
    for tokens in spoilt.values():
        g[:, list(tokens)] = bad
    leaf = [t.clone().requires_grad_() for t in (x, g, b, h0)]
    out, hf = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
    dout, dhf = torch.randn_like(out), torch.randn_like(hf)
    got = torch.autograd.grad((out, hf), leaf, (dout, dhf))
    for i, (s, e) in enumerate(zip(cuts[:-1], cuts[1:])):
        if i in spoilt:
            continue
        n64 = lambda t: t.detach().double().cpu().numpy()
        first = n64(h0) if s == 0 else np.zeros((B, C))
        ref, mag, grads = reference(*(n64(t[:, s:e]) for t in (x, g, b)), first,
                                    n64(dout[:, s:e]), n64(dhf) if e == T else np.zeros((B, C)))
        check(out[:, s:e], ref, mag)
        for n, t in zip(("x", "g", "b"), got):
            check(t[:, s:e], *grads[n], n=2)
        if s == 0:
            check(got[3], *grads["h0"], n=2)
    assert not torch.isfinite(out[:, 40]).any() and not torch.isfinite(out[:, 389]).any()


def test_step_after_a_bad_decay(dev):
    import gdn2_package as gp
    x = torch.randn((3, 20), device=dev)
    for bad in (torch.nan, torch.inf):
        _, h = gp.gdn2_gated_scan_step(x, torch.full_like(x, bad), state=torch.ones_like(x))
        assert not torch.isfinite(h).any()
        out, h = gp.gdn2_gated_scan_step(x, torch.full_like(x, -torch.inf), state=h)
        assert torch.equal(out, x) and torch.equal(h, x)


@pytest.mark.parametrize("B,T,C", [(3, 100, 40), (2, 400, 130), (1, 700, 64), (2, 1500, 33),
                                   (1, 2049, 1024), (1, 33000, 20)])
def test_state_updated_in_place(dev, B, T, C):
    """h_final over h0, as the C interface allows: no step reads h0 once another may have
    written h_final."""
    import gdn2_package as gp
    from gdn2_package import _lib
    (x, g, b, h0), _ = inputs(B, T, C, torch.float32, torch.float32, dev, C)
    want, hf = gp.gdn2_gated_scan(x, g, b, h0=h0)
    nbytes = _lib.lib().gdn2_gated_scan_workspace_bytes(B, T, C, _lib.GDN2_F32)
    ws, out = torch.empty(nbytes, dtype=torch.uint8, device=dev), torch.empty_like(x)
    state = h0.clone()
    for _ in range(4):
        state.copy_(h0)
        rc = _lib.launch("gdn2_gated_scan_fwd", x.device, B, T, C, _lib.GDN2_F32, _lib.GDN2_F32,
                         x.data_ptr(), None, g.data_ptr(), None, b.data_ptr(), None,
                         state.data_ptr(), out.data_ptr(), state.data_ptr(), None,
                         ws.data_ptr() if nbytes else None, nbytes)
        assert rc == _lib.OK
        assert torch.equal(out, want) and torch.equal(state, hf)


def test_tangents_are_refused(dev):
    """Forward mode is not there, and no tangent is dropped without a word."""
    import gdn2_package as gp
    from torch.autograd import forward_ad
    x, b = torch.randn(2, 2, 9, 16, device=dev)
    g, h0 = -torch.rand(2, 9, 16, device=dev), torch.randn(2, 16, device=dev)
    want = gp.gdn2_gated_scan(x, g, b, h0=h0)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            assert all(torch.equal(a, e) for a, e in zip(gp.gdn2_gated_scan(x, g, b, h0=h0), want))
            dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
            for call in (lambda: gp.gdn2_gated_scan(dual(x), g),
                         lambda: gp.gdn2_gated_scan(x, dual(g)),
                         lambda: gp.gdn2_gated_scan(x, g, dual(b)),
                         lambda: gp.gdn2_gated_scan(x, g, h0=dual(h0))):
                with pytest.raises(NotImplementedError):
                    call()


@pytest.mark.parametrize("full", [False, True])
def test_a_penalty_on_the_gradient_is_refused(dev, full):
    """A loss that holds its own gradient raises, also where the cotangent was a constant and the
    rest of the loss could go on without the penalty's part."""
    import gdn2_package as gp
    x = torch.randn(2, 9, 16, device=dev, requires_grad=True)
    g = (-torch.rand(2, 9, 16, device=dev)).requires_grad_()
    b, h0 = (torch.rand_like(x), torch.randn(2, 16, device=dev)) if full else (None, None)
    loss = sum(t.sum() for t in gp.gdn2_gated_scan(x, g, b, h0=h0)[:2 if full else 1])
    dx, dg = torch.autograd.grad(loss, (x, g), create_graph=True)
    for penalty in (dx.square().sum(), dg.square().sum()):
        with pytest.raises(RuntimeError):
            (loss + penalty).backward(retain_graph=True)
    for got, want in zip(torch.autograd.grad(loss, (x, g)), (dx, dg)):
        assert torch.equal(got, want)     # without it nothing is in the way


@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("B,T,C", [(200, 130, 33), (48, 300, 256), (256, 600, 20), (64, 1000, 200)])
def test_walk_in_wide_tiles(dev, B, T, C, dtype, gdtype):
    """Short axes with enough tiles of 64 channels: walked in those, 4 channels a thread and one."""
    import gdn2_package as gp
    from gdn2_package import _lib
    code = _lib.GDN2_F32 if dtype == torch.float32 else _lib.GDN2_BF16
    assert _lib.lib().gdn2_gated_scan_workspace_bytes(B, T, C, code) == 0
    assert B * ((C + 63) // 64) >= (192 if T <= 512 else 256)
    ts, (xn, gn, bn, hn) = inputs(B, T, C, dtype, gdtype, dev, T)
    for names in (("x", "g", "b", "h0"), ("x", "g")):
        leaf = {n: ts["xgb".find(n) if n != "h0" else 3].clone().requires_grad_() for n in names}
        out, hf = gp.gdn2_gated_scan(leaf["x"], leaf["g"], leaf.get("b"), h0=leaf.get("h0"))
        dout, dhf = torch.randn_like(out), torch.randn_like(hf)
        got = torch.autograd.grad((out, hf), list(leaf.values()), (dout, dhf))
        ref, mag, grads = reference(xn, gn, bn if "b" in leaf else np.ones_like(bn),
                                    hn if "h0" in leaf else np.zeros_like(hn),
                                    dout.double().cpu().numpy(), dhf.double().cpu().numpy())
        check(out, ref, mag)
        check(hf, ref[:, -1], mag[:, -1])
        for n, t in zip(leaf, got):
            check(t, *grads[n], n=2)


# tiles of 16 (many tokens, few channels), 64 (bfloat16, many channels; float32: 32) and 32
LONG = [(1, 32801, 77), (1, 32900, 64), (2, 1537, 767), (2, 1100, 512), (1, 700, 101),
        (1, 900, 100)]


@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("B,T,C", LONG)
def test_steps_at_once_without_a_gate(dev, B, T, C, dtype, gdtype):
    """Every tile without a gate and with g of either type; the cotangent of one output alone."""
    import gdn2_package as gp
    ts, (xn, gn, bn, hn) = inputs(B, T, C, dtype, gdtype, dev, T + 1)
    zero_out, zero_hf, ones = np.zeros_like(xn), np.zeros_like(hn), np.ones_like(bn)
    for which in (0, 1):
        leaf = [t.clone().requires_grad_() for t in ts[:2]]
        res = gp.gdn2_gated_scan(*leaf)
        cot = torch.randn_like(res[which])
        got = torch.autograd.grad(res[which], leaf, cot)
        cn = cot.double().cpu().numpy()
        ref, mag, grads = reference(xn, gn, ones, zero_hf, zero_out if which else cn,
                                    cn if which else zero_hf)
        check(res[0], ref, mag)
        check(res[1], ref[:, -1], mag[:, -1])
        for n, t in zip(("x", "g"), got):
            check(t, *grads[n], n=2)


@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("B,T,C", [(2, 1537, 767), (1, 700, 60), (1, 33000, 24)])
def test_gated_steps_at_once_of_one_output(dev, B, T, C, dtype, gdtype):
    """With a gate: one channel a thread in tiles of 64, g in bfloat16, one output alone."""
    import gdn2_package as gp
    ts, (xn, gn, bn, hn) = inputs(B, T, C, dtype, gdtype, dev, T + 2)
    for which in (0, 1):
        leaf = [t.clone().requires_grad_() for t in ts]
        res = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
        cot = torch.randn_like(res[which])
        got = torch.autograd.grad(res[which], leaf, cot)
        cn = cot.double().cpu().numpy()
        _, _, grads = reference(xn, gn, bn, hn, np.zeros_like(xn) if which else cn,
                                cn if which else np.zeros_like(hn))
        for n, t in zip(("x", "g", "b", "h0"), got):
            check(t, *grads[n], n=2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,C", [(2, 300, 24), (200, 100, 40), (2, 1300, 768), (1, 33000, 40)])
def test_strides_walked_and_in_steps(dev, B, T, C, dtype):
    """The parts of one projection, rows at an odd offset and cotangents of any layout: the
    results from dense tensors where the accesses are the same, within the bound where not."""
    import gdn2_package as gp
    (x, g, b, h0), (xn, gn, bn, hn) = inputs(B, T, C, dtype, dtype, dev, T + 3)
    dout = torch.randn((B, T, C), device=dev).to(dtype)
    wide = torch.cat([dout, dout], 2)

    def run(x, g, b, dout):
        leaf = [t.detach().requires_grad_() for t in (x, g, b, h0)]
        out, hf = gp.gdn2_gated_scan(*leaf[:3], h0=leaf[3])
        return (out, hf, *torch.autograd.grad((out, hf), leaf, (dout, torch.ones_like(hf))))
    want = run(x, g, b, dout)
    proj = torch.cat([x, g, b], 2)
    parts = [proj[..., i * C:(i + 1) * C] for i in range(3)]
    for got in (run(*parts, wide[..., C:]),
                run(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, g, b, dout))),
                run(x.transpose(1, 2).contiguous().transpose(1, 2), g, b, dout)):
        assert all(torch.equal(a, e) for a, e in zip(got, want))
    odd = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
    got = run(odd(x), odd(g), odd(b), odd(dout))
    ref, mag, grads = reference(xn, gn, bn, hn, dout.double().cpu().numpy(), np.ones_like(hn))
    check(got[0], ref, mag)
    check(got[1], ref[:, -1], mag[:, -1])
    for n, t in zip(("x", "g", "b", "h0"), got[2:]):
        check(t, *grads[n], n=2)
    # a g shared by all channels, and one by all tokens
    for shared in (g[..., :1].expand(B, T, C), g[:, :1].expand(B, T, C)):
        one = gp.gdn2_gated_scan(x, shared, b, h0=h0)
        two = gp.gdn2_gated_scan(x, shared.contiguous(), b, h0=h0)
        assert all(torch.equal(a, e) for a, e in zip(one, two))
