"""Selective state space scan (gdn2_selective_scan, its backward, gdn2_selective_scan_step) against
the recurrence in float64.

Tolerances, in units of 2^-24 of m, the same sums with the terms' magnitudes.  The inputs here have
0.02 <= d |A|.  A term that passes k tokens before it is read picks up, in every token, two roundings of
the product and the sum and the error of e^{d A}: d carries at most 24 roundings (of softplus, or
none), its product with A two more, and where a chunk of 128 tokens is passed at once the sum of
d 128 more; so 16 + 160 d |A| for each token, on a term that has fallen to e^{-k d |A|}:
16 k e^{-k d |A|} <= 16 / (e 0.02) = 300 and 160 k d |A| e^{-k d |A|} <= 59.  With 32 for u = d x B,
(N + 8) for the sum over the states, at most 72, and 16 + 4 |z| <= 40 for the gate: below 512.
Gradients are products of two such sums, of a state's and of an adjoint's: twice that, and sums over
channels and tokens add at most 128 roundings each.  A bfloat16 result is rounded once more, 2^-8
of its value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 512 * 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0")


def reference(t, starts, softplus, dout=None, dh=None):
    """{name: (value, magnitude)} in float64: out, h_final and the gradients of what t holds."""
    x, dt, A = t["x"], t["dt"], t["A"]
    Bt, T, Ch = x.shape
    G, N = t["B"].shape[2:]
    raw = dt if t.get("dt_bias") is None else dt + t["dt_bias"]
    d = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    wide = lambda m: m.repeat_interleave(Ch // G, 2)
    B, C = wide(t["B"]), wide(t["C"])
    a = torch.exp(d[..., None] * A)
    fresh = torch.zeros((Bt, T), dtype=torch.bool, device=x.device) if starts is None else starts
    u = (d * x)[..., None] * B
    h0 = torch.zeros((Bt, Ch, N), dtype=x.dtype, device=x.device) if t.get("h0") is None \
        else t["h0"]

    def scan(u, h):
        res, before = torch.empty_like(u), torch.empty_like(u)
        for i in range(T):
            h = torch.where(fresh[:, i, None, None], 0.0, h)
            before[:, i] = h
            h = a[:, i] * h + u[:, i]
            res[:, i] = h
        return res, before
    h, before = scan(u, h0)
    m, mbefore = scan(u.abs(), h0.abs())
    y, my = (h * C).sum(-1), (m * C.abs()).sum(-1)
    if t.get("D") is not None:
        y, my = y + t["D"] * x, my + (t["D"] * x).abs()
    z = t.get("z")
    gate = torch.ones_like(x) if z is None else z * torch.sigmoid(z)
    res = {"out": (y * gate, my * gate.abs()), "h_final": (h[:, -1], m[:, -1])}
    if dout is None:
        return res

    def back(dy, e, C):
        g = torch.empty_like(u)
        for i in reversed(range(T)):
            g[:, i] = e + dy[:, i, :, None] * C[:, i]
            e = torch.where(fresh[:, i, None, None], 0.0, a[:, i] * g[:, i])
        return g, e
    dy = dout * gate
    if z is not None:
        s = torch.sigmoid(z)
        slope = s * (1 + z * (1 - s))
        res["z"] = (dout * y * slope, (dout * my).abs() * (s * (1 + z.abs())))
    g, dh0 = back(dy, dh, C)
    mg, mdh0 = back(dy.abs(), dh.abs(), C.abs())
    group = lambda v: v.unflatten(2, (G, Ch // G)).sum(3)
    for which, g_, b_, sign in (("value", g, before, lambda v: v), ("mag", mg, mbefore, torch.abs)):
        through = g_ * a * b_
        inner = (g_ * sign(B)).sum(-1)
        D = 0 if t.get("D") is None else sign(t["D"]) * sign(dy)
        dd = (through * sign(A)).sum(-1) + sign(x) * inner
        if softplus:
            dd = dd * torch.sigmoid(raw)
        part = {"x": sign(d) * inner + D, "dt": dd, "A": (through * d[..., None]).sum((0, 1)),
                "B": group(g_ * sign(d * x)[..., None]),
                "C": group((h if which == "value" else m) * sign(dy)[..., None]),
                "D": (sign(dy) * sign(x)).sum((0, 1)), "dt_bias": dd.sum((0, 1)),
                "h0": dh0 if which == "value" else mdh0}
        for n, v in part.items():
            res[n] = (v,) if which == "value" else (res[n][0], v)
    return res


def check(got, ref, n=1.0):
    value, mag = ref
    assert got.shape == value.shape
    half = 2.0 ** -8 if got.dtype == BF16 else 0.0
    excess = (got.double() - value).abs() - (n * EPS * mag + half * value.abs() + 1e-30)
    assert torch.isfinite(got).all() and bool((excess <= 0).all()), float(excess.max())


def inputs(Bt, T, Ch, G, N, dtype, dtdtype, dev, seed, softplus=True):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device=dev)
    uni = lambda *s: torch.rand(s, generator=gen, device=dev)
    t = {"x": rand(Bt, T, Ch).to(dtype), "A": -1.0 - 3.0 * uni(Ch, N),
         "B": rand(Bt, T, G, N).to(dtype), "C": rand(Bt, T, G, N).to(dtype), "D": rand(Ch),
         "z": rand(Bt, T, Ch).to(dtype), "h0": rand(Bt, Ch, N)}
    if softplus:   # raw values from about -3.7 to 1
        t["dt"] = (uni(Bt, T, Ch) * 3.0).to(dtdtype)
        t["dt_bias"] = -3.6 + uni(Ch)
    else:
        t["dt"] = (0.02 + 0.5 * uni(Bt, T, Ch)).to(dtdtype)
        t["dt_bias"] = 0.1 * uni(Ch)
    starts = uni(Bt, T) < 3.0 / (T + 2)
    return t, starts, rand(Bt, T, Ch).to(dtype), rand(Bt, Ch, N)


d64 = lambda t: {n: v.detach().double() for n, v in t.items()}


def call(t, softplus, starts=None):
    import gdn2_package as gp
    return gp.gdn2_selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t.get("D"),
                                  z=t.get("z"), dt_bias=t.get("dt_bias"), dt_softplus=softplus,
                                  h0=t.get("h0"), starts=starts)


TYPES = [(F32, F32), (BF16, F32), (BF16, BF16)]
# one token, the sides of a block of 16, of a chunk of 32, and many chunks; channels on and off a
# wave and a tile, groups of a few channels; states of each padded width and off it
SIZES = [(1, 1, 1, 1, 1), (2, 2, 3, 1, 16), (1, 15, 64, 1, 8), (3, 16, 65, 1, 3), (1, 17, 130, 2, 16),
         (2, 31, 36, 3, 24), (1, 32, 20, 20, 5), (2, 33, 70, 1, 32), (1, 100, 129, 1, 16),
         (2, 65, 48, 4, 64), (1, 257, 33, 1, 33), (1, 530, 100, 1, 16), (2, 1000, 8, 2, 9)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_backward(dev, size, types):
    for softplus, names, cut in ((True, NAMES, False), (False, NAMES, True),
                                 (True, ("x", "dt", "A", "B", "C"), True)):
        t, starts, dout, dh = inputs(*size, *types, dev, sum(size), softplus)
        if "dt_bias" not in names and softplus:
            t["dt"] = (t["dt"] - 3.0).to(types[1])
        starts = starts if cut else None
        leaf = {n: t[n].clone().requires_grad_() for n in names}
        out, h = call(leaf, softplus, starts)
        assert out.dtype == types[0] and h.dtype == F32
        ref = reference(d64(leaf), starts, softplus, dout.double(), dh.double())
        check(out, ref["out"])
        check(h, ref["h_final"])
        got = torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))
        for n, g in zip(names, got):
            assert g.dtype == leaf[n].dtype, n
            check(g, ref[n], 2.5)
        with torch.no_grad():
            again, same = call(leaf, softplus, starts)
        assert torch.equal(again, out) and torch.equal(same, h)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("size", [(8, 1030, 768, 1, 16), (2, 4100, 200, 2, 16)])
def test_chunks_of_every_length(dev, size, types):
    """Enough waves for chunks of 64 and 128 tokens, and chunks of 32 over a long axis."""
    t, starts, dout, dh = inputs(*size, *types, dev, 7)
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    out, h = call(leaf, True, starts)
    ref = reference(d64(leaf), starts, True, dout.double(), dh.double())
    check(out, ref["out"])
    check(h, ref["h_final"])
    for n, g in zip(NAMES, torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))):
        check(g, ref[n], 2.5)


def test_same_results_every_time(dev):
    t, starts, dout, dh = inputs(2, 700, 200, 2, 16, BF16, BF16, dev, 3)
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    first = None
    for _ in range(3):
        outs = call(leaf, True, starts)
        res = (*outs, *torch.autograd.grad(outs, list(leaf.values()), (dout, dh)))
        first = first or res
        assert all(torch.equal(a, b) for a, b in zip(first, res))


@pytest.mark.parametrize("which", [0, 1])
def test_one_cotangent(dev, which):
    t, starts, dout, dh = inputs(2, 90, 40, 1, 16, F32, F32, dev, 5)
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    outs = call(leaf, True, starts)
    got = torch.autograd.grad(outs[which], list(leaf.values()), (dout, dh)[which])
    ref = reference(d64(leaf), starts, True, dout.double() * (which == 0),
                    dh.double() * (which == 1))
    for n, g in zip(NAMES, got):
        check(g, ref[n], 2.5)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("G,N", [(1, 16), (2, 7), (4, 64), (1, 1)])
def test_pieces_and_steps(dev, G, N, types):
    """A sequence in pieces and token by token follows the recurrence as at once."""
    import gdn2_package as gp
    t, _, _, _ = inputs(3, 70, 24, G, N, *types, dev, N)
    ref = reference(d64(t), None, True)
    part = lambda a, b, h: {**{n: v[:, a:b] if n in ("x", "dt", "B", "C", "z") else v
                               for n, v in t.items()}, "h0": h}
    for cuts in ((1, 69), (40, 30), (33, 1, 36)):
        at, h, outs = 0, t["h0"], []
        for n in cuts:
            out, h = call(part(at, at + n, h), True)
            outs.append(out)
            at += n
        check(torch.cat(outs, 1), ref["out"])
        check(h, ref["h_final"])
    h, own, outs = t["h0"], t["h0"].clone(), []
    for i in range(70):
        kw = dict(D=t["D"], z=t["z"][:, i], dt_bias=t["dt_bias"], dt_softplus=True)
        xs = (t["x"][:, i], t["dt"][:, i], t["A"], t["B"][:, i], t["C"][:, i])
        out, h = gp.gdn2_selective_scan_step(*xs, state=h, **kw)
        again, same = gp.gdn2_selective_scan_step(*xs, state=own, inplace=True, **kw)
        assert torch.equal(out, again) and torch.equal(h, own) and same is own
        outs.append(out)
    check(torch.stack(outs, 1), ref["out"])
    check(h, ref["h_final"])
    # without a state, D, z, bias
    out, h = gp.gdn2_selective_scan_step(t["x"][:, 0], 0.1 + t["dt"][:, 0], t["A"], t["B"][:, 0],
                                         t["C"][:, 0])
    first = {n: t[n][:, :1] for n in ("x", "B", "C")}
    r = reference(d64({**first, "dt": (0.1 + t["dt"][:, :1]), "A": t["A"]}), None, False)
    check(out, (r["out"][0][:, 0], r["out"][1][:, 0]))
    check(h, r["h_final"])


def test_starts_separate(dev):
    """NaN and infinities before a start reach nothing after it, wherever chunks are cut."""
    t, _, dout, dh = inputs(2, 150, 40, 1, 16, F32, F32, dev, 8)
    alone = {n: (v[:, 101:] if n in ("x", "dt", "B", "C", "z") else v) for n, v in t.items()
             if n != "h0"}
    want = call(alone, True)
    cut = torch.zeros((2, 150), dtype=torch.bool, device=dev)
    cut[:, 101] = True
    for name, where in (("x", 100), ("x", 20), ("h0", None), ("B", 99), ("dt", 64)):
        bad = {n: v.clone() for n, v in t.items()}
        if where is None:
            bad[name][:] = torch.nan
        else:
            bad[name][0, where], bad[name][1, where] = torch.nan, torch.inf
        leaf = {n: v.requires_grad_() for n, v in bad.items()}
        out, h = call(leaf, True, cut)
        mag = reference(d64(alone), None, True)
        check(out[:, 101:], mag["out"])
        check(h, mag["h_final"])
        assert torch.isfinite(want[0]).all()
        gx, = torch.autograd.grad((out, h), [leaf["x"]], (dout, dh))
        assert torch.isfinite(gx[:, 101:]).all()
        lost, = torch.autograd.grad(call(leaf, True, cut)[1], [leaf["x"]], dh)
        if name != "dt" and name != "B":
            assert (lost[:, :101] == 0).all()


def test_gradient_of_nan_behind_a_start(dev):
    """A cotangent that is NaN in one sequence leaves the gradients of the one before it."""
    t, _, dout, dh = inputs(1, 120, 24, 1, 16, F32, F32, dev, 9)
    cut = torch.zeros((1, 120), dtype=torch.bool, device=dev)
    cut[:, 50] = True
    dout[:, 70] = torch.nan
    leaf = {n: t[n].clone().requires_grad_() for n in ("x", "dt", "B", "C", "z", "h0")}
    out, h = call({**t, **leaf}, True, cut)
    got = torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))
    for n, g in zip(leaf, got):
        assert torch.isfinite(g if n == "h0" else g[:, :50]).all(), n


def test_padding_with_steps_of_zero(dev):
    """d = 0 leaves the states as they are: a padded batch's states are those of its tokens."""
    t, _, _, _ = inputs(2, 80, 24, 1, 16, F32, F32, dev, 2, False)
    t.pop("dt_bias")
    t["dt"][1, 50:] = 0.0
    _, h = call(t, False)
    short = {n: (v[1:, :50] if n in ("x", "dt", "B", "C", "z") else v[1:] if n == "h0" else v)
             for n, v in t.items()}
    check(h[1:], reference(d64(short), None, False)["h_final"])


def test_far_decays_and_steps(dev):
    """Decays that leave nothing, steps far below and above softplus' bend."""
    t, _, dout, dh = inputs(1, 70, 16, 1, 16, F32, F32, dev, 4)
    t["A"] = t["A"] * 1e4
    t["dt"][:, ::3], t["dt"][:, 1::3] = 60.0, -60.0
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    out, h = call(leaf, True)
    grads = torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))
    assert all(torch.isfinite(v).all() for v in (out, h, *grads))
    ref = reference(d64(leaf), None, True)
    check(h, ref["h_final"])


def test_layouts_and_types(dev):
    """Parts of one projection, odd offsets, transposes, mixed and other types, empty inputs."""
    import gdn2_package as gp
    Bt, T, Ch, N = 2, 45, 24, 16
    t, starts, _, _ = inputs(Bt, T, Ch, 1, N, BF16, BF16, dev, 5)
    want = call(t, True, starts)
    wide = torch.zeros((Bt, T, 3 * Ch + 2 * N + 1), device=dev, dtype=BF16)
    for off in (0, 1):
        parts, at = dict(t), off
        for n, width in (("x", Ch), ("dt", Ch), ("B", N), ("C", N), ("z", Ch)):
            wide[..., at:at + width] = t[n].flatten(2)
            parts[n] = wide[..., at:at + width]
            at += width
        got = call(parts, True, starts)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    turned = {n: v.transpose(0, -1).contiguous().transpose(0, -1) for n, v in t.items()}
    assert all(torch.equal(a, b) for a, b in zip(call(turned, True, starts), want))
    one = {n: (v[:1].expand(3, *v.shape[1:]) if n not in ("A", "D", "dt_bias") else v)
           for n, v in t.items()}
    assert torch.equal(call(one, True)[0][2], call({**t}, True)[0][0])
    leaf = {n: v.clone().requires_grad_() for n, v in t.items()}
    leaf["B"], leaf["A"] = (t[n].to(dt).requires_grad_() for n, dt in (("B", F32), ("A", BF16)))
    out, _ = call(leaf, True)
    assert out.dtype == BF16
    for n, g in zip(leaf, torch.autograd.grad(out.float().square().sum(), list(leaf.values()))):
        assert g.dtype == leaf[n].dtype and g.shape == leaf[n].shape
    half = {n: (v.half() if n in ("x", "B", "C", "z", "dt") else v) for n, v in t.items()}
    assert call(half, True)[0].dtype == torch.float16
    none = {n: (v[:, :0] if n in ("x", "dt", "B", "C", "z") else v) for n, v in t.items()}
    out, h = call(none, True)
    assert out.shape == (Bt, 0, Ch) and torch.equal(h, t["h0"])
    none.pop("h0")
    assert (call(none, True)[1] == 0).all()
    out, h = gp.gdn2_selective_scan(t["x"][:0], t["dt"][:0], t["A"], t["B"][:0], t["C"][:0])
    assert out.shape == (0, T, Ch) and h.shape == (0, Ch, N)


def test_gradient_by_differences(dev):
    """The gradient's projection on a direction against a central difference of the float64
    definition."""
    t, starts, dout, dh = inputs(2, 60, 12, 2, 5, F32, F32, dev, 11)
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    outs = call(leaf, True, starts)
    grads = torch.autograd.grad(outs, list(leaf.values()), (dout, dh))
    gen = torch.Generator(device=dev).manual_seed(2)
    dirs = {n: torch.randn(v.shape, generator=gen, device=dev, dtype=torch.float64)
            for n, v in leaf.items()}

    def value(move):
        r = reference({n: v + move * dirs[n] for n, v in d64(leaf).items()}, starts, True)
        return float((r["out"][0] * dout.double()).sum() + (r["h_final"][0] * dh.double()).sum())
    h = 1e-6
    slope = (value(h) - value(-h)) / (2 * h)
    terms = [g.double() * dirs[n] for n, g in zip(NAMES, grads)]
    got, scale = (float(sum(f(v).sum() for v in terms)) for f in (lambda v: v, torch.abs))
    assert abs(got - slope) <= 1e-5 * scale


def test_graph(dev):
    """A captured training step and a captured decoding step replay as the eager ones."""
    import gdn2_package as gp
    t, starts, dout, dh = inputs(2, 200, 64, 1, 16, BF16, BF16, dev, 4)
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    state = t["h0"].clone()

    def step():
        outs = call(leaf, True, starts)
        return (*(o.detach() for o in outs),
                *torch.autograd.grad(outs, list(leaf.values()), (dout, dh)))

    def token():
        return gp.gdn2_selective_scan_step(
            leaf["x"][:, 0], leaf["dt"][:, 0], leaf["A"], leaf["B"][:, 0], leaf["C"][:, 0],
            dt_bias=leaf["dt_bias"], dt_softplus=True, state=state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), token()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res, tok = step(), token()
    for i in range(4):
        with torch.no_grad():
            leaf["x"].copy_(torch.randn_like(leaf["x"]))
            state.copy_(torch.randn_like(state))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*res, *tok), (*step(), *token())):
            assert torch.equal(a, b)


def test_other_streams(dev):
    t, starts, _, _ = inputs(2, 2000, 64, 1, 16, F32, F32, dev, 6)
    want = call(t, True, starts)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(call(t, True, starts))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_refusals(dev):
    import gdn2_package as gp
    t, starts, _, _ = inputs(2, 5, 8, 2, 4, F32, F32, dev, 1)
    f = lambda **kw: call({**t, **kw}, True, kw.pop("starts", None))
    z = lambda *s: torch.zeros(s, device=dev)
    for bad in (dict(x=z(2, 8)), dict(dt=z(2, 4, 8)), dict(A=z(7, 4)), dict(A=z(8, 65)),
                dict(A=z(8, 0)), dict(B=z(2, 5, 3, 4), C=z(2, 5, 3, 4)), dict(C=z(2, 5, 1, 4)),
                dict(B=z(2, 5, 2, 3)), dict(D=z(7)), dict(z=z(2, 5, 7)), dict(dt_bias=z(1)),
                dict(h0=z(2, 8, 5)), dict(starts=starts[:1]), dict(starts=z(2, 5))):
        with pytest.raises(gp.GDN2ShapeError):
            f(**bad)
    for bad in (dict(x=t["x"].cpu()), dict(A=t["A"].cpu()), dict(h0=t["h0"].cpu()),
                dict(x=t["x"].int()), dict(D=t["D"].int()), dict(starts=starts.cpu())):
        with pytest.raises(gp.GDN2Error):
            f(**bad)
    for bad in (dict(A=1), dict(B=1), dict(dt=None), dict(starts=[1])):
        with pytest.raises(TypeError):
            f(**bad)
    s = lambda **kw: gp.gdn2_selective_scan_step(
        **{**dict(x=t["x"][:, 0], dt=t["dt"][:, 0], A=t["A"], B=t["B"][:, 0], C=t["C"][:, 0]), **kw})
    for bad in (dict(x=t["x"]), dict(state=z(1, 8, 4)), dict(B=z(2, 3))):
        with pytest.raises(gp.GDN2ShapeError):
            s(**bad)
    for bad in (dict(inplace=True), dict(state=t["h0"].bfloat16(), inplace=True),
                dict(state=t["h0"].transpose(1, 2).contiguous().transpose(1, 2), inplace=True)):
        with pytest.raises(gp.GDN2Error):
            s(**bad)
    leaf = t["x"].clone().requires_grad_()
    g, = torch.autograd.grad(f(x=leaf)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        f(x=fwAD.make_dual(t["x"], t["x"]))
