"""Short causal convolution (gdn2_short_conv, its backward, gdn2_short_conv_step) against the
definition in float64.

Tolerances, in units of 2^-24.  With m = |bias| + sum |w x| the value before the activation
carries at most W + 1 <= 5 roundings of m.  silu(v) = v s with s = 1 / (1 + e^-v): e^-v carries
two roundings of its exponent v log2(e) and one of its own, s three more; silu' is below 1.1 and
silu'' below 0.5.  So y is within 16 + 4 |v| of m, and dp = dy silu'(v) within |dy| (16 + 4 |v| + 4 m).
Sums over tokens run over at most 32 tokens of a run, 16 runs of a workgroup and the rows of
partial sums, in float32: 128 for each term at the sizes here.  A bfloat16 result is rounded once
more, 2^-8 of its value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def reference(x, w, bias, state, starts, silu, dy=None, dlast=None, terms=128):
    """Values and the bounds of their errors (without the last rounding), in float64."""
    B, T, C = x.shape
    W = w.shape[1]
    line = torch.cat([torch.zeros(B, W - 1, C, dtype=x.dtype, device=x.device)
                      if state is None else state, x], 1)
    first = torch.zeros(B, T + W - 1, dtype=torch.long, device=x.device)
    if starts is not None:
        first[:, W - 1:] = starts.long().cumsum(1)
    same = [(first[:, k:k + T] == first[:, W - 1:])[..., None] for k in range(W)]
    tap = [torch.where(same[k], line[:, k:k + T], 0.0) for k in range(W)]
    v = sum(tap[k] * w[:, k] for k in range(W))
    m = sum((tap[k] * w[:, k]).abs() for k in range(W))
    if bias is not None:
        v, m = v + bias, m + bias.abs()
    s = torch.sigmoid(v)
    kept = (first[:, T:] == first[:, -1:])[..., None]
    last = torch.where(kept, line[:, T:], 0.0)
    res = {"y": (v * s if silu else v, ULP * (16 + 4 * v.abs()) * m), "last": (last, None)}
    if dy is None:
        return res
    dp = dy * s * (1 + v * (1 - s)) if silu else dy
    ep = ULP * dy.abs() * (16 + 4 * v.abs() + 4 * m)
    dline, eline = torch.zeros_like(line), torch.zeros_like(line)
    dw, ew = torch.zeros_like(w), torch.zeros_like(w)
    for k in range(W):
        dline[:, k:k + T] += torch.where(same[k], dp, 0.0) * w[:, k]
        eline[:, k:k + T] += torch.where(same[k], ep + 8 * ULP * dp.abs(), 0.0) * w[:, k].abs()
        dw[:, k] = (dp * tap[k]).sum((0, 1))
        ew[:, k] = ((ep + terms * ULP * dp.abs()) * tap[k].abs()).sum((0, 1))
    dline[:, T:] += torch.where(kept, dlast, 0.0)
    eline += 4 * ULP * dline.abs()
    eline[:, T:] += 4 * ULP * dlast.abs()
    res.update(x=(dline[:, W - 1:], eline[:, W - 1:]), weight=(dw, ew),
               bias=(dp.sum((0, 1)), (ep + terms * ULP * dp.abs()).sum((0, 1))),
               state=(dline[:, :W - 1], eline[:, :W - 1]))
    return res


def check(got, ref):
    value, bound = ref
    assert got.shape == value.shape
    if bound is None:
        assert torch.equal(got, value.to(got.dtype))
        return
    half = 2.0 ** -8 if got.dtype == BF16 else ULP
    excess = (got.double() - value).abs() - (bound + half * value.abs() + 1e-37)
    assert bool((excess <= 0).all()), float(excess.max())


def inputs(B, T, C, W, dtype, dev, seed, starts=False):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device=dev)
    t = {"x": rand(B, T, C).to(dtype), "weight": rand(C, W), "bias": rand(C),
         "state": rand(B, W - 1, C).to(dtype)}
    cut = torch.rand((B, T), generator=gen, device=dev) < 0.2 if starts else None
    return t, cut, rand(B, T, C).to(dtype), rand(B, W - 1, C).to(dtype)


d64 = lambda t: None if t is None else t.detach().double()
# one token, fewer than the taps, the sides of a run and of a workgroup's runs; channels on and
# off four, and of one, some and many tiles
SIZES = [(1, 1, 1), (2, 2, 4), (3, 3, 7), (1, 5, 64), (2, 8, 12), (1, 31, 100), (2, 33, 260),
         (1, 129, 17), (2, 300, 64), (1, 1025, 20), (5, 130, 257), (1, 4100, 12)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("B,T,C", SIZES)
def test_forward_and_backward(dev, B, T, C, W, dtype):
    import gdn2_package as gp
    for starts in (False, True):
        t, cut, dy, dlast = inputs(B, T, C, W, dtype, dev, T * C + W, starts)
        for names, act in ((("x", "weight", "bias", "state"), "silu"), (("x", "weight"), None)):
            leaf = {n: t[n].clone().requires_grad_() for n in names}
            y, last = gp.gdn2_short_conv(leaf["x"], leaf["weight"], bias=leaf.get("bias"),
                                         state=leaf.get("state"), activation=act, starts=cut)
            assert y.dtype == dtype and last.dtype == dtype
            ref = reference(*(d64(leaf.get(n)) for n in ("x", "weight", "bias", "state")), cut,
                            act == "silu", d64(dy), d64(dlast))
            check(y, ref["y"])
            check(last, ref["last"])
            for n, g in zip(leaf, torch.autograd.grad((y, last), list(leaf.values()),
                                                      (dy, dlast))):
                assert g.dtype == leaf[n].dtype
                check(g, ref[n])
            with torch.no_grad():
                again, same = gp.gdn2_short_conv(leaf["x"], leaf["weight"], bias=leaf.get("bias"),
                                                 state=leaf.get("state"), activation=act, starts=cut)
            assert torch.equal(again, y) and torch.equal(same, last)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,C,W", [(1540, 70, 12, 4), (1600, 133, 7, 3), (800, 1030, 6, 4)])
def test_long_runs(dev, B, T, C, W, dtype):
    """Enough workgroups for the backward's runs of 64 tokens.  A weight's sum: 64 tokens, 16 runs, at
    most 1600 rows of partial sums of which a thread adds every 64th, 25, and 64 of those: 169."""
    import gdn2_package as gp
    for starts in (False, True):
        t, cut, dy, dlast = inputs(B, T, C, W, dtype, dev, T, starts)
        if starts:   # far from each other too
            cut &= torch.arange(T, device=dev) % 32 < 3
        leaf = [t[n].clone().requires_grad_() for n in ("x", "weight", "bias", "state")]
        outs = gp.gdn2_short_conv(leaf[0], leaf[1], bias=leaf[2], state=leaf[3], starts=cut)
        ref = reference(*map(d64, leaf), cut, True, d64(dy), d64(dlast), 192)
        check(outs[0], ref["y"])
        for n, g in zip(("x", "weight", "bias", "state"),
                        torch.autograd.grad(outs, leaf, (dy, dlast))):
            check(g, ref[n])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_cotangent(dev, dtype):
    """Either output may go without a gradient."""
    import gdn2_package as gp
    t, cut, dy, dlast = inputs(2, 40, 24, 4, dtype, dev, 1, True)
    for use in (0, 1):
        leaf = [t[n].clone().requires_grad_() for n in ("x", "weight", "bias", "state")]
        outs = gp.gdn2_short_conv(leaf[0], leaf[1], bias=leaf[2], state=leaf[3], starts=cut)
        got = torch.autograd.grad(outs[use], leaf, (dy, dlast)[use])
        d = [d64(dy) * (use == 0), d64(dlast) * (use == 1)]
        ref = reference(*map(d64, leaf), cut, True, *d)
        for n, g in zip(("x", "weight", "bias", "state"), got):
            check(g, ref[n])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W", [2, 3, 4])
def test_pieces_and_steps(dev, W, dtype):
    """A sequence in pieces, down to single tokens, is the sequence at once, bit for bit."""
    import gdn2_package as gp
    t, _, _, _ = inputs(3, 50, 30, W, dtype, dev, W)
    run = lambda x, s: gp.gdn2_short_conv(x, t["weight"], bias=t["bias"], state=s)
    whole, end = run(t["x"], t["state"])
    for cuts in ([50], [1, 49], [20, 2, 28], [W - 1, 51 - W]):
        s, ys, at = t["state"], [], 0
        for n in cuts:
            y, s = run(t["x"][:, at:at + n], s)
            ys.append(y)
            at += n
        assert torch.equal(torch.cat(ys, 1), whole) and torch.equal(s, end)
    s, own = t["state"], t["state"].clone()
    for i in range(50):
        y, s = gp.gdn2_short_conv_step(t["x"][:, i], t["weight"], bias=t["bias"], state=s)
        z, same = gp.gdn2_short_conv_step(t["x"][:, i], t["weight"], bias=t["bias"], state=own,
                                          inplace=True)
        assert torch.equal(y, whole[:, i]) and torch.equal(z, y) and same is own
    assert torch.equal(s, end) and torch.equal(own, end)
    y, s = gp.gdn2_short_conv_step(t["x"][:, 0], t["weight"])
    w, _ = gp.gdn2_short_conv(t["x"][:, :1], t["weight"])
    assert torch.equal(y, w[:, 0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_starts_separate(dev, dtype):
    """NaN and infinities before a start reach nothing after it, nor do gradients come back."""
    import gdn2_package as gp
    B, T, C, W = 2, 70, 20, 4
    t, _, dy, dlast = inputs(B, T, C, W, dtype, dev, 3)
    cut = torch.zeros((B, T), dtype=torch.bool, device=dev)
    at = 37
    cut[:, at] = True
    x = t["x"].clone()
    x[0, at - 1], x[1, at - 2] = torch.nan, torch.inf
    leaf = [x.requires_grad_(), t["weight"].clone().requires_grad_()]
    y, last = gp.gdn2_short_conv(*leaf, starts=cut)
    alone, end = gp.gdn2_short_conv(t["x"][:, at:], t["weight"])
    assert torch.equal(y[:, at:], alone) and torch.equal(last, end)
    g = torch.autograd.grad((y[:, at:], last), leaf, (dy[:, at:], dlast))
    # the infinity's own token, at - 2, and the three that reach it have no slope to speak of
    assert (g[0][:, :at - 5] == 0).all() and torch.isfinite(g[0][:, at:]).all()
    # every token a start: only the last tap is left; the state stays empty
    every = torch.ones((B, T), dtype=torch.bool, device=dev)
    y, last = gp.gdn2_short_conv(t["x"], t["weight"], state=t["state"] * torch.nan, starts=every,
                                 activation=None)
    want = t["x"].float() * t["weight"][:, -1]
    assert torch.equal(y, want.to(dtype))
    assert (last[:, :-1] == 0).all() and torch.equal(last[:, -1], t["x"][:, -1])


def test_layouts_and_types(dev):
    """Heads, parts of a projection, odd offsets, transposes, other types, empty inputs."""
    import gdn2_package as gp
    B, T, H, D, W = 2, 45, 3, 8, 4
    t, cut, _, _ = inputs(B, T, H * D, W, BF16, dev, 5, True)
    want, end = gp.gdn2_short_conv(t["x"], t["weight"], bias=t["bias"], state=t["state"], starts=cut)
    heads = lambda v: v.unflatten(-1, (H, D))
    y, s = gp.gdn2_short_conv(heads(t["x"]), t["weight"].view(H, D, W), bias=t["bias"].view(H, D),
                              state=heads(t["state"]), starts=cut)
    assert torch.equal(y.flatten(2), want) and torch.equal(s.flatten(2), end)
    wide = torch.randn((B, T, 3 * H * D + 1), device=dev).bfloat16()
    for off in (0, 1, H * D):
        wide[..., off:off + H * D] = t["x"]
        y, s = gp.gdn2_short_conv(wide[..., off:off + H * D], t["weight"], bias=t["bias"],
                                  state=t["state"], starts=cut)
        assert torch.equal(y, want) and torch.equal(s, end)
    other = t["x"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(gp.gdn2_short_conv(other, t["weight"], bias=t["bias"], state=t["state"],
                                          starts=cut)[0], want)
    one = gp.gdn2_short_conv(t["x"][:1].expand(3, -1, -1), t["weight"])[0]
    assert torch.equal(one[2], gp.gdn2_short_conv(t["x"][:1], t["weight"])[0][0])
    y, s = gp.gdn2_short_conv(t["x"].half(), t["weight"].bfloat16())
    assert y.dtype == s.dtype == torch.float16
    leaf = t["weight"].bfloat16().requires_grad_()
    gp.gdn2_short_conv(t["x"], leaf)[0].sum().backward()
    assert leaf.grad.dtype == BF16
    y, s = gp.gdn2_short_conv(t["x"][:, :0], t["weight"], state=t["state"])
    assert y.shape == (B, 0, H * D) and torch.equal(s, t["state"])
    assert gp.gdn2_short_conv(t["x"][:0], t["weight"])[1].shape == (0, W - 1, H * D)


def test_gradient_by_differences(dev):
    """The gradient's projection on a direction against a central difference in float64 of the
    float64 definition."""
    import gdn2_package as gp
    t, cut, dy, dlast = inputs(2, 60, 12, 4, F32, dev, 9, True)
    names = ("x", "weight", "bias", "state")
    leaf = [t[n].clone().requires_grad_() for n in names]
    outs = gp.gdn2_short_conv(leaf[0], leaf[1], bias=leaf[2], state=leaf[3], starts=cut)
    grads = torch.autograd.grad(outs, leaf, (dy, dlast))

    def value(move):
        r = reference(*(d64(v) + move * d for v, d in zip(leaf, dirs)), cut, True)
        return float((r["y"][0] * d64(dy)).sum() + (r["last"][0] * d64(dlast)).sum())
    gen = torch.Generator(device=dev).manual_seed(2)
    dirs = [torch.randn(v.shape, generator=gen, device=dev, dtype=torch.float64) for v in leaf]
    h = 1e-5
    slope = (value(h) - value(-h)) / (2 * h)
    got = float(sum((d64(g) * d).sum() for g, d in zip(grads, dirs)))
    scale = float(sum((d64(g) * d).abs().sum() for g, d in zip(grads, dirs)))
    assert abs(got - slope) <= 1e-6 * scale


def test_graph(dev):
    """A captured training step replays, with the program's own work between the replays."""
    import gdn2_package as gp
    t, cut, dy, dlast = inputs(2, 100, 64, 4, BF16, dev, 4, True)
    leaf = [t[n].clone().requires_grad_() for n in ("x", "weight", "bias", "state")]

    def step():
        outs = gp.gdn2_short_conv(leaf[0], leaf[1], bias=leaf[2], state=leaf[3], starts=cut)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaf, (dy, dlast)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for i in range(4):
        with torch.no_grad():
            leaf[0].copy_(torch.randn_like(leaf[0]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, step()):
            assert torch.equal(a, b)


def test_other_streams(dev):
    import gdn2_package as gp
    t, _, _, _ = inputs(2, 3000, 64, 4, F32, dev, 6)
    want = gp.gdn2_short_conv(t["x"], t["weight"])[0]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(gp.gdn2_short_conv(t["x"], t["weight"])[0])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals(dev):
    import gdn2_package as gp
    x, w = torch.zeros((2, 5, 8), device=dev), torch.zeros((8, 4), device=dev)
    state, b = torch.zeros((2, 3, 8), device=dev), torch.zeros(8, device=dev)
    f, s = gp.gdn2_short_conv, gp.gdn2_short_conv_step
    for bad in (lambda: f(x[0], w), lambda: f(x, w[:, :1]), lambda: f(x, w[:7]),
                lambda: f(x, torch.zeros((8, 5), device=dev)), lambda: f(x, w, bias=b[:7]),
                lambda: f(x, w, state=state[:, :2]), lambda: f(x, w, state=state[:1]),
                lambda: f(x, w, starts=torch.zeros((2, 4), dtype=torch.bool, device=dev)),
                lambda: f(x, w, starts=torch.zeros((2, 5), device=dev)),
                lambda: s(x[:, 0], w, state=state[:1]), lambda: s(x[0, 0], w)):
        with pytest.raises(gp.GDN2ShapeError):
            bad()
    for bad in (lambda: f(x.cpu(), w), lambda: f(x, w.cpu()), lambda: f(x, w, state=state.cpu()),
                lambda: f(x, w, activation="relu"), lambda: f(x.int(), w), lambda: f(x, w.int()),
                lambda: s(x[:, 0], w, inplace=True),
                lambda: s(x[:, 0], w, state=state.bfloat16(), inplace=True),
                lambda: s(x[:, 0], w, state=state.transpose(0, 1).contiguous().transpose(0, 1),
                          inplace=True)):
        with pytest.raises(gp.GDN2Error):
            bad()
    for bad in (lambda: f(1, w), lambda: f(x, 1), lambda: f(x, w, bias=1),
                lambda: f(x, w, starts=[0])):
        with pytest.raises(TypeError):
            bad()
    leaf = torch.randn((1, 4, 8), device=dev, requires_grad=True)
    g, = torch.autograd.grad(f(leaf, w + 1)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        f(fwAD.make_dual(torch.zeros_like(x), x), w)
