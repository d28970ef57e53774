"""8-bit floating point in blocks of 128 (gdn2_quantize_fp8, gdn2_dequantize_fp8), its product
(gdn2_fp8_matmul) and the linear layer trained with it (gdn2_fp8_linear).

q and scale are compared bit for bit with the definition in float64: the scale is a power of two and
t / s exact, so there is one rounding.

The product.  Float32 results: products of e4m3 values are exact, a block's 128 of them are added in
float32 (at most 128 roundings, 2^-24 each, of the sum of the magnitudes), scaled and added to
those of other blocks (three roundings, and K / 128 + 8 additions): (139 + K / 128) 2^-24 of the sum
of the magnitudes.  Bfloat16 results: the 8-bit matrix instruction keeps of eight products at a
time what lies above 2^-13 of the largest one, so the other seven lose at most 7 2^-13 of that one,
which the sum of the magnitudes holds: 2^-10 of it, and 2^-8 of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -24
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def held(t, down, along):
    """(values that t stands for, q values, scales), float64, blocks of down x along."""
    M, K = t.shape
    pad = torch.zeros((-(-M // down) * down, -(-K // along) * along), dtype=torch.float64,
                      device=t.device)
    pad[:M, :K] = t
    cells = pad.view(pad.shape[0] // down, down, pad.shape[1] // along, along)
    top = cells.abs().amax((1, 3))
    scale = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp_min(-126.0))
    wide = scale[:, None, :, None]
    v = cells / wide
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    q = torch.round(v / step) * step
    cut = lambda a: a.expand(cells.shape).reshape(pad.shape)[:M, :K]
    return cut(q * wide), cut(q), torch.where(top == 0, 0.0, scale)


def product(x, w, bias=None):
    """(value, sum of magnitudes) in float64 of what x (M, K) and w (N, K) stand for."""
    y, mag = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
    return (y, mag) if bias is None else (y + bias.double(), mag + bias.double().abs())


def check(got, ref, K):
    value, mag = ref
    bound = (139 + K / 128) * ULP * mag
    if got.dtype == BF16:
        bound = bound + 2.0 ** -10 * mag + 2.0 ** -8 * value.abs()
    excess = (got.double() - value).abs() - bound
    assert got.shape == value.shape and bool((excess <= 0).all()), float(excess.max())


def values(M, K, dtype, dev, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    t = torch.randn((M, K), generator=gen, device=dev)
    return (t * torch.exp(2.0 * torch.randn((M, 1), generator=gen, device=dev))).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [1, 7, 128, 130, 300])
@pytest.mark.parametrize("C", [1, 8, 100, 127, 128, 129, 256, 1000])
def test_quantize_and_back(dev, C, M, dtype):
    import gdn2_package as gp
    x = values(M, C, dtype, dev, M + C)
    for blocks in (False, True):
        q, scale = gp.gdn2_quantize_fp8(x, blocks=blocks)
        v, qv, s = held(x.double(), 128 if blocks else 1, 128)
        assert q.dtype == E4M3 and q.shape == x.shape and scale.dtype == F32
        assert torch.equal(scale.double(), s) and torch.equal(q.double(), qv)
        ld = (C + 15) // 16 * 16
        rows = torch.as_strided(q.view(torch.uint8), (M, ld), (ld, 1))
        assert (rows[:, C:] == 0).all()
        for dt in (F32, BF16):
            back = gp.gdn2_dequantize_fp8(q, scale, dtype=dt)
            assert back.dtype == dt and torch.equal(back, v.to(dt))
    # strided rows, off 16 bytes; batches
    wide = torch.cat([x[:, :1], x, x[:, :1]], 1)
    a, b = gp.gdn2_quantize_fp8(wide[:, 1:-1]), gp.gdn2_quantize_fp8(x)
    assert torch.equal(a[0].double(), b[0].double()) and torch.equal(a[1], b[1])
    q, s = gp.gdn2_quantize_fp8(x[None].expand(2, M, C))
    assert q.shape == (2, M, C) and torch.equal(s[1], b[1])
    assert torch.equal(gp.gdn2_dequantize_fp8(q, s, dtype=F32)[1],
                       gp.gdn2_dequantize_fp8(*b, dtype=F32))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,C", [(1, 5), (130, 100), (300, 257), (128, 128)])
def test_both_directions(dev, M, C, dtype):
    """gdn2_quantize_fp8 of the C ABI with rows and columns at once, the columns' sums, columns
    alone, and blocks both ways."""
    from gdn2_package import _lib
    L, code = _lib.lib(), _lib.GDN2_F32 if dtype == F32 else _lib.GDN2_BF16
    x = values(M, C, dtype, dev, 3)
    kb, mb, up = -(-C // 128), -(-M // 128), lambda n: (n + 15) // 16 * 16
    f32 = lambda *s: torch.full(s, torch.nan, device=dev)
    u8 = lambda *s: torch.full(s, 0x7F, dtype=torch.uint8, device=dev)
    q, qt, part, sums = u8(M, up(C)), u8(C, up(M)), f32(mb, C), f32(C)

    def call(blocks, q, s, qt, st, part=None, sums=None):
        ptr = lambda t: None if t is None else t.data_ptr()
        assert L.gdn2_quantize_fp8(torch.cuda.current_stream().cuda_stream, M, C, code,
                                   x.data_ptr(), C, blocks, ptr(q), up(C), ptr(s), ptr(qt), up(M),
                                   ptr(st), ptr(part), ptr(sums)) == 0

    def same(q, s, t, down):
        _, qv, sv = held(t.double(), down, 128)
        width = t.shape[1]
        assert torch.equal(q.view(E4M3)[:, :width].double(), qv) and (q[:, width:] == 0).all()
        assert torch.equal(s.double(), sv)
    s, st = f32(kb, M), f32(mb, C)
    call(0, q, s, qt, st, part, sums)
    same(q, s.t(), x, 1)
    same(qt, st.t(), x.t(), 1)
    # eight rows, sixteen of those, and the rows of partial sums in turn
    mag = x.double().abs().sum(0)
    assert ((sums.double() - x.double().sum(0)).abs() <= (8 + 16 + mb + 16) * ULP * mag).all()
    qt.fill_(0x7F), st.fill_(torch.nan)
    call(0, None, None, qt, st)
    same(qt, st.t(), x.t(), 1)
    q.fill_(0x7F), qt.fill_(0x7F)
    s, st = f32(mb, kb), f32(kb, mb)
    call(1, q, s, qt, st)
    same(q, s, x, 128)
    same(qt, st, x.t(), 128)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_value(dev, dtype):
    """Every e4m3 value comes back as it is, its neighbours' midpoints go to even, the border of a
    scale is where it is said to be."""
    import gdn2_package as gp
    codes = torch.arange(256, dtype=torch.uint8, device=dev).view(E4M3).double()
    exact = codes[torch.isfinite(codes)]
    ordered = exact.unique()
    mid = (ordered[1:] + ordered[:-1]) / 2        # five bits at most: exact in bfloat16
    x = torch.cat([exact, mid, torch.tensor([448.0], device=dev, dtype=torch.float64)])
    x = torch.nn.functional.pad(x, (0, -len(x) % 127)).view(-1, 127)
    x = torch.cat([x, torch.full((len(x), 1), 448.0, dtype=torch.float64, device=dev)], 1)
    for k in (0, 100, -100):
        t = (x * 2.0 ** k).to(dtype)
        q, s = gp.gdn2_quantize_fp8(t)
        _, qv, sv = held(t.double(), 1, 128)
        assert (s == 2.0 ** k).all() and torch.equal(q.double(), qv) and torch.equal(s.double(), sv)
    for top, s in ((448.0, 1.0), (450.0, 2.0), (224.0, 0.5), (225.0, 1.0), (1.0, 2.0 ** -8)):
        t = torch.full((1, 5), top, device=dev).to(dtype)
        q, got = gp.gdn2_quantize_fp8(t)
        assert float(got) == s and (q.double() * s - top).abs().max() <= top / 16


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_blocks_without_values(dev, dtype):
    """Zeros, NaN, infinities, the largest and the smallest values, each in its block alone."""
    import gdn2_package as gp
    x = torch.randn((8, 300), device=dev).to(dtype)
    x[1, :128], x[2, 7], x[3, 299], x[4, 130] = 0, torch.nan, torch.inf, -torch.inf
    x[5] = x[5].sign() * torch.finfo(dtype).max
    x[6] = x[6].sign() * torch.finfo(dtype).tiny
    x[7] = x[7].sign() * 2.0 ** -133   # a subnormal of either type
    q, s = gp.gdn2_quantize_fp8(x)
    bad = torch.zeros((8, 3), dtype=torch.bool, device=dev)
    bad[2, 0] = bad[3, 2] = bad[4, 1] = True
    assert torch.equal(torch.isnan(s), bad) and float(s[1, 0]) == 0.0
    wide = bad.repeat_interleave(128, 1)[:, :300]
    assert (q.double()[wide] == 0).all()
    v, qv, sv = held(torch.where(wide, 0.0, x.double()), 1, 128)
    assert torch.equal(q.double(), qv) and torch.equal(s[~bad].double(), sv[~bad])
    w, sw = gp.gdn2_quantize_fp8(torch.randn((40, 300), device=dev), blocks=True)
    y = gp.gdn2_fp8_matmul(q[:5], s[:5], w, sw, out_dtype=F32)
    assert torch.isnan(y[2:5]).all() and torch.isfinite(y[:2]).all()
    qb, sb = gp.gdn2_quantize_fp8(x, blocks=True)
    assert torch.isnan(sb).all() and (qb.double() == 0).all()
    e, es = gp.gdn2_quantize_fp8(x[:0])
    assert e.shape == (0, 300) and es.shape == (0, 3)
    assert gp.gdn2_dequantize_fp8(e, es).shape == (0, 300)


def operands(M, N, K, dev, seed, blocks):
    """Finite e4m3 codes of every size with scales of any value, and the values they stand for."""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def codes(r):
        c = torch.randint(0, 256, (r, K), generator=gen, device=dev, dtype=torch.uint8)
        return torch.where((c & 127) == 127, c - 1, c).view(E4M3)
    kb, rand = -(-K // 128), lambda *s: torch.rand(s, generator=gen, device=dev) + 0.01
    q, w, sx = codes(M), codes(N), rand(M, kb)
    sw = rand(-(-N // 128), kb) if blocks else rand(N, kb)
    wide = lambda s, r: s.double().repeat_interleave(r, 0).repeat_interleave(128, 1)
    x64 = q.double() * wide(sx, 1)[:, :K]
    w64 = w.double() * wide(sw, 128 if blocks else 1)[:N, :K]
    return q, sx, w, sw, torch.randn(N, generator=gen, device=dev), x64, w64


KS = [1, 15, 16, 17, 100, 127, 128, 129, 192, 256, 257, 384, 400, 640, 1000]


@pytest.mark.parametrize("blocks", [True, False])
@pytest.mark.parametrize("M", [1, 2, 16, 17, 32, 33, 64, 65, 127, 130, 300])
@pytest.mark.parametrize("N", [1, 7, 16, 64, 65, 136, 200])
def test_product(dev, M, N, blocks):
    import gdn2_package as gp
    for K in KS[(M + N) % 2::2]:
        q, sx, w, sw, bias, x64, w64 = operands(M, N, K, dev, M * N + K, blocks)
        for dt, b in ((F32, bias), (BF16, None)):
            y = gp.gdn2_fp8_matmul(q, sx, w, sw, bias=b, out_dtype=dt)
            assert y.dtype == dt
            check(y, product(x64, w64, b), K)


@pytest.mark.parametrize("blocks", [True, False])
@pytest.mark.parametrize("M,N,K", [(2050, 2100, 200), (4100, 4104, 130), (65600, 70, 40),
                                   (70, 20000, 70), (64, 9000, 2000), (2048, 2048, 1024)])
def test_product_of_many_tiles(dev, M, N, K, blocks):
    """Enough tiles to choose the largest, and long thin products."""
    import gdn2_package as gp
    q, sx, w, sw, bias, x64, w64 = operands(M, N, K, dev, K, blocks)
    for dt, b in ((F32, None), (BF16, bias.bfloat16())):
        check(gp.gdn2_fp8_matmul(q, sx, w, sw, bias=b, out_dtype=dt), product(x64, w64, b), K)


@pytest.mark.parametrize("blocks", [True, False])
@pytest.mark.parametrize("M,N", [(130, 900), (200, 777), (260, 1300)])
def test_product_of_few_tiles(dev, M, N, blocks):
    """A tile for a CU at most: two halves of k of 4 and 4 slices up to 9 and 8, the last one whole,
    of one value or in between."""
    import gdn2_package as gp
    for K in (1023, 1024, 1025, 1157, 1280, 1300, 2048, 2170):
        q, sx, w, sw, bias, x64, w64 = operands(M, N, K, dev, M + K, blocks)
        for dt, b in ((F32, bias), (BF16, None)):
            check(gp.gdn2_fp8_matmul(q, sx, w, sw, bias=b, out_dtype=dt), product(x64, w64, b), K)


def test_layouts(dev):
    """Padding that holds NaN, rows at odd offsets, transposes, batches, scales laid out either way."""
    import gdn2_package as gp
    for M in (9, 90):
        N, K = 140, 175
        q, sx, w, sw, _, x64, w64 = operands(M, N, K, dev, 1, True)
        want = gp.gdn2_fp8_matmul(q, sx, w, sw, out_dtype=F32)
        check(want, product(x64, w64), K)
        bits = lambda t: t.view(torch.uint8)
        wide_q = torch.full((M, 192), 0x7F, dtype=torch.uint8, device=dev)
        wide_w = torch.full((N, 176), 0xFF, dtype=torch.uint8, device=dev)
        wide_q[:, :K], wide_w[:, :K] = bits(q), bits(w)
        off = lambda t, n: torch.cat([bits(t)[:, :n], bits(t)], 1).view(E4M3)[:, n:]
        turned = bits(q).t().contiguous().t().view(E4M3)
        for a in (q, wide_q.view(E4M3)[:, :K], off(q, 1), turned):
            for b in (w, wide_w.view(E4M3)[:, :K], off(w, 5)):
                for s in (sx, sx.t().contiguous().t()):
                    assert torch.equal(gp.gdn2_fp8_matmul(a, s, b, sw, out_dtype=F32), want)
        assert torch.equal(gp.gdn2_fp8_matmul(q, sx, w, sw.t().contiguous().t(), out_dtype=F32), want)
        # the last row's padding is outside the storage: copied, not read
        tight = torch.empty((M - 1) * 176 + K, dtype=torch.uint8, device=dev).as_strided(
            (M, K), (176, 1))
        tight.copy_(bits(q))
        assert torch.equal(gp.gdn2_fp8_matmul(tight.view(E4M3), sx, w, sw, out_dtype=F32), want)
        y = gp.gdn2_fp8_matmul(q.view(3, M // 3, K), sx.view(3, M // 3, 2), w, sw, out_dtype=F32)
        assert y.shape == (3, M // 3, N) and torch.equal(y.view(M, N), want)
        one = gp.gdn2_fp8_matmul(q[0], sx[0], w, sw, out_dtype=F32)
        check(one[None], product(x64[:1], w64), K)
        assert gp.gdn2_fp8_matmul(q[:0], sx[:0], w, sw).shape == (0, N)
        # the same blocks said row by row
        rows = sw.repeat_interleave(128, 0)[:N]
        check(gp.gdn2_fp8_matmul(q, sx, w, rows, out_dtype=F32), product(x64, w64), K)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 5, 7), (33, 130, 64), (130, 64, 300),
                                   (257, 300, 129), (700, 520, 400), (130, 1160, 1157),
                                   (1160, 130, 1030), (2200, 140, 1300)])
def test_linear(dev, M, N, K, dtype):
    import gdn2_package as gp
    x, w, dy = (values(*s, dtype, dev, i) for i, s in enumerate(((M, K), (N, K), (M, N))))
    bias = torch.randn(N, device=dev)
    for b in (bias, None):
        leaf = [t.clone().requires_grad_() for t in (x, w, b) if t is not None]
        y = gp.gdn2_fp8_linear(*leaf)
        assert y.dtype == dtype
        xr, wb = held(x.double(), 1, 128)[0], held(w.double(), 128, 128)[0]
        check(y, product(xr, wb, b), K)
        got = torch.autograd.grad(y, leaf, dy)
        check(got[0], product(held(dy.double(), 1, 128)[0], wb.t()), N)
        check(got[1], product(held(dy.double().t(), 1, 128)[0], held(x.double().t(), 1, 128)[0]), M)
        if b is not None:
            mag = dy.double().abs().sum(0)
            off = (got[2].double() - dy.double().sum(0)).abs()
            assert (off <= (40 + M / 2048) * ULP * mag).all()
        with torch.no_grad():
            assert torch.equal(gp.gdn2_fp8_linear(x, w, b), y)


def test_linear_partial_and_types(dev):
    """Gradients of some inputs alone; batches; mixed and other types; no rows."""
    import gdn2_package as gp
    M, N, K = 40, 30, 200
    x, w, dy = (values(*s, BF16, dev, i) for i, s in enumerate(((M, K), (N, K), (M, N))))
    b = torch.randn(N, device=dev)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(gp.gdn2_fp8_linear(*full), full, dy)
    for i in range(3):
        part = [x, w, b]
        part[i] = part[i].clone().requires_grad_()
        g, = torch.autograd.grad(gp.gdn2_fp8_linear(*part), part[i], dy)
        assert torch.equal(g, want[i])
    leaf = x.view(4, 10, K).clone().requires_grad_()
    y = gp.gdn2_fp8_linear(leaf, w, b)
    g, = torch.autograd.grad(y, leaf, dy.view(4, 10, N))
    assert y.shape == (4, 10, N) and torch.equal(g.view(M, K), want[0])
    # a transposed cotangent, one that is expanded
    wide = dy.t().contiguous().t()
    assert torch.equal(torch.autograd.grad(gp.gdn2_fp8_linear(*full), full[0], wide)[0], want[0])
    g1 = torch.autograd.grad(gp.gdn2_fp8_linear(*full), full, dy[:1].expand(M, N))
    g2 = torch.autograd.grad(gp.gdn2_fp8_linear(*full), full, dy[:1].repeat(M, 1))
    assert all(torch.equal(p, q) for p, q in zip(g1, g2))
    mixed = [x.clone().requires_grad_(), w.float().requires_grad_(), b.bfloat16().requires_grad_()]
    y = gp.gdn2_fp8_linear(*mixed)
    assert y.dtype == BF16
    for p, g in zip(mixed, torch.autograd.grad(y, mixed, dy)):
        assert g.dtype == p.dtype and g.shape == p.shape
    assert gp.gdn2_fp8_linear(x.half(), w.half()).dtype == torch.float16
    none = x[:0].clone().requires_grad_()
    y = gp.gdn2_fp8_linear(none, full[1], full[2])
    assert y.shape == (0, N)
    assert (torch.autograd.grad(y.sum(), full[1])[0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N", [(8, 40), (200, 300), (2100, 2100)])
def test_linear_with_nan(dev, M, N, dtype):
    """NaN and infinities in a block reach every output that it enters, and no other."""
    import gdn2_package as gp
    K = 300
    x, w, dy = (values(*s, dtype, dev, i) for i, s in enumerate(((M, K), (N, K), (M, N))))
    x[:, :] = x.clamp(-100, 100)
    x[2, 140], x[5, 299], dy[3, 7] = torch.nan, torch.inf, -torch.inf
    x[4], dy[:128, 9] = 0.0, 0.0
    leaf = [x.requires_grad_(), w.requires_grad_()]
    y = gp.gdn2_fp8_linear(*leaf)
    bad = torch.zeros(M, dtype=torch.bool, device=dev)
    bad[2] = bad[5] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all() and (y[4] == 0).all()
    dx, dw = torch.autograd.grad(y, leaf, dy)
    assert torch.isnan(dx[3]).all() and torch.isfinite(dx[torch.arange(M, device=dev) != 3]).all()
    lost = torch.zeros((N, K), dtype=torch.bool, device=dev)
    lost[7], lost[:, 140], lost[:, 299] = True, True, True
    assert torch.equal(torch.isnan(dw), lost)


def test_graph(dev):
    """A captured training step of the layer and a captured product replay as the eager ones."""
    import gdn2_package as gp
    M, N, K = 300, 260, 200
    x, w, dy = (values(*s, BF16, dev, i) for i, s in enumerate(((M, K), (N, K), (M, N))))
    leaf = [x.clone().requires_grad_(), w.clone().requires_grad_(),
            torch.randn(N, device=dev, requires_grad=True)]
    wq = gp.gdn2_quantize_fp8(w, blocks=True)

    def step():
        y = gp.gdn2_fp8_linear(*leaf)
        served = gp.gdn2_fp8_matmul(*gp.gdn2_quantize_fp8(leaf[0]), *wq)
        return (y.detach(), served, *torch.autograd.grad(y, leaf, dy))
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
    x, w = values(700, 400, BF16, dev, 1), values(600, 400, BF16, dev, 2)
    want = gp.gdn2_fp8_linear(x, w)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(gp.gdn2_fp8_linear(x, w))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals(dev):
    import gdn2_package as gp
    M, N, K = 10, 20, 200
    q, sx, w, sw, b, _, _ = operands(M, N, K, dev, 1, True)
    x, wf = torch.zeros((M, K), device=dev), torch.zeros((N, K), device=dev)
    f = gp.gdn2_fp8_matmul
    for bad in (lambda: f(q, sx[:, :1], w, sw), lambda: f(q, sx, w[:, :100], sw[:, :1]),
                lambda: f(q, sx, w, sw[:, :1]), lambda: f(q, sx, w, sw, bias=b[:5]),
                lambda: f(q, sx, w[0], sw[0]), lambda: f(q[:, :0], sx[:, :0], w, sw),
                lambda: gp.gdn2_quantize_fp8(x[0, 0]), lambda: gp.gdn2_quantize_fp8(x[:, :0]),
                lambda: gp.gdn2_quantize_fp8(x[0], blocks=True),
                lambda: gp.gdn2_dequantize_fp8(q, sx[:5]),
                lambda: gp.gdn2_fp8_linear(x, wf[:, :5]), lambda: gp.gdn2_fp8_linear(x, wf[0]),
                lambda: gp.gdn2_fp8_linear(x, wf, b[:3])):
        with pytest.raises(gp.GDN2ShapeError):
            bad()
    for bad in (lambda: f(q.cpu(), sx, w, sw), lambda: f(q, sx.cpu(), w, sw),
                lambda: f(q, sx.double(), w, sw), lambda: f(x, sx, w, sw),
                lambda: f(q, sx, w, sw, out_dtype=torch.float16),
                lambda: f(q, sx, w, sw, bias=b.int()), lambda: f(q, sx, w, sw, bias=b.cpu()),
                lambda: gp.gdn2_quantize_fp8(x.int()), lambda: gp.gdn2_quantize_fp8(x.cpu()),
                lambda: gp.gdn2_dequantize_fp8(q, sx, dtype=torch.float16),
                lambda: gp.gdn2_fp8_linear(x, wf.cpu()), lambda: gp.gdn2_fp8_linear(x.int(), wf)):
        with pytest.raises(gp.GDN2Error):
            bad()
    for bad in (lambda: f(1, sx, w, sw), lambda: f(q, sx, w, None), lambda: gp.gdn2_fp8_linear(x, 1),
                lambda: gp.gdn2_quantize_fp8(None), lambda: f(q, sx, w, sw, bias=1)):
        with pytest.raises(TypeError):
            bad()
    leaf = torch.randn((M, K), device=dev, requires_grad=True)
    g, = torch.autograd.grad(gp.gdn2_fp8_linear(leaf, wf + 1).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        gp.gdn2_fp8_linear(fwAD.make_dual(x, x), wf)
