"""Rows in 8 bits (gdn2_rms_norm_int8, gdn2_quantize_int8, gdn2_dequantize_int8) and their
product (gdn2_int8_matmul).

q is compared bit for bit with the same float32 steps in numpy, and with the definition: at
most half a step off, and the three roundings of t * (127 * (1 / m)).  Scales carry fewer than
32 roundings (the norm's).  The product's sums are exact integers: what is left are the
conversion, the two scales and the bias, four roundings, and the one to bfloat16."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def np64(t):
    return t.detach().double().cpu().numpy()


def check_rows(q, scale, t32, rstd):
    """q, scale of rows t32 (numpy float32), the norm's factor rstd (float64, per row)."""
    m = np.abs(t32).max(-1, keepdims=True)
    inv = (np.float32(1) / m) * np.float32(127)
    got = q.cpu().numpy()
    assert np.array_equal(got, np.rint(t32 * inv).astype(np.int8))
    exact = 127.0 * t32.astype(np.float64) / m
    assert np.abs(got - exact).max() <= 0.5 + 127 * 3 * ULP
    ref = m[:, 0].astype(np.float64) * rstd / 127
    assert np.abs(np64(scale) - ref).max() <= (32 * ULP * ref).max()


@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, F32), (BF16, F32, BF16)])
@pytest.mark.parametrize("C", [1, 7, 16, 24, 100, 512, 1000, 1032, 2049, 4096, 5000, 8200, 16384])
def test_norm_in_8_bits(dev, C, types):
    import gdn2_package as gp
    for M in (1, 13):
        gen = torch.Generator(device=dev).manual_seed(C)
        rand = lambda *s: torch.randn(s, generator=gen, device=dev)
        x, r, w = rand(M, C).to(types[0]), rand(M, C).to(types[1]), (1 + rand(C)).to(types[2])
        q, scale, h = gp.gdn2_rms_norm_int8(x, w, residual=r, eps=1e-5)
        assert q.shape == (M, C) and q.dtype == torch.int8 and scale.shape == (M,)
        assert torch.equal(h, torch.tensor(np64(x) + np64(r)).to(types[1]).to(dev))
        t = (h.float() * w.float()).cpu().numpy()
        check_rows(q, scale, t, 1 / np.sqrt((np64(h) ** 2).mean(-1) + 1e-5))
        q2, s2, same = gp.gdn2_rms_norm_int8(h, w, eps=1e-5) if types[0] == types[1] \
            else (q, scale, h)
        assert torch.equal(q2, q) and torch.equal(s2, scale) and same is h
        ld = (C + 15) // 16 * 16
        rows = torch.as_strided(q, (M, ld), (ld, 1))
        assert (rows[:, C:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [1, 5, 16, 250, 768, 3000, 7000, 16385, 32768])
def test_quantize_and_back(dev, C, dtype):
    import gdn2_package as gp
    x = torch.randn((2, 3, C), device=dev).to(dtype)
    q, scale = gp.gdn2_quantize_int8(x)
    assert q.shape == x.shape and scale.shape == (2, 3)
    check_rows(q.reshape(6, C), scale.reshape(6), x.float().reshape(6, C).cpu().numpy(), 1.0)
    for dt in (F32, BF16):
        back = gp.gdn2_dequantize_int8(q, scale, dtype=dt)
        want = (q.float() * scale[..., None]).to(dt)
        assert back.dtype == dt and torch.equal(back, want)
    # strided rows, off 16 bytes
    wide = torch.randn((6, C + 3), device=dev).to(dtype)
    a, b = gp.gdn2_quantize_int8(wide[:, 3:]), gp.gdn2_quantize_int8(wide[:, 3:].clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_without_values(dev, dtype):
    """Zero rows have scale 0, rows with NaN or infinity scale NaN and q = 0; tiny rows
    count as zero; the largest finite ones hold."""
    import gdn2_package as gp
    x = torch.randn((8, 40), device=dev).to(dtype)
    x[1], x[2, 7], x[3, 39], x[4, 0] = 0, torch.nan, torch.inf, -torch.inf
    x[5] *= 1e-38
    x[6] = x[6].sign() * torch.finfo(dtype).max
    q, scale = gp.gdn2_quantize_int8(x)
    assert (q[1:6] == 0).all() and (scale[1] == 0) and (scale[5] == 0)
    assert torch.isnan(scale[2:5]).all() and torch.isfinite(scale[[0, 6, 7]]).all()
    assert (q[6].abs() == 127).all()
    back = gp.gdn2_dequantize_int8(q, scale, dtype=F32)
    assert torch.isnan(back[2:5]).all() and (back[[1, 5]] == 0).all()
    w, sw = gp.gdn2_quantize_int8(torch.randn((9, 40), device=dev))
    y = gp.gdn2_int8_matmul(q, scale, w, sw, out_dtype=F32)
    assert torch.isnan(y[2:5]).all() and (y[[1, 5]] == 0).all()
    x[6] = 1.0   # (a norm's sum of squares would overflow, as in any float32 norm)
    qn, sn, _ = gp.gdn2_rms_norm_int8(x, torch.ones(40, device=dev))
    assert torch.isnan(sn[2:5]).all() and (sn[1] == 0) and (qn[1:5] == 0).all()
    e, es = gp.gdn2_quantize_int8(x[:0])
    assert e.shape == (0, 40) and es.shape == (0,)
    assert gp.gdn2_dequantize_int8(e, es).shape == (0, 40)


def product(q, sx, w, sw, bias=None):
    """(value, sum of the roundings' magnitudes) in float64; the integers are exact."""
    y = (q.double() @ w.double().t()) * sx.double()[:, None] * sw.double()
    mag = y.abs()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag


def check_product(got, ref, mag):
    half = 2.0 ** -8 if got.dtype == BF16 else 0.0
    excess = (got.double() - ref).abs() - (4 * ULP * mag + half * ref.abs())
    assert bool((excess <= 0).all()), float(excess.max())


def operands(M, N, K, dev, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    ints = lambda *s: torch.randint(-128, 128, s, generator=gen, device=dev, dtype=torch.int8)
    rand = lambda n: torch.rand(n, generator=gen, device=dev) + 0.01
    return ints(M, K), rand(M), ints(N, K), rand(N), torch.randn(N, generator=gen, device=dev)


KS = [1, 15, 16, 17, 63, 64, 65, 100, 127, 128, 192, 193, 256, 1000, 1024, 1100]


@pytest.mark.parametrize("M", [1, 2, 16, 17, 32, 33, 63, 64, 65, 127, 128, 130, 300])
@pytest.mark.parametrize("N", [1, 7, 16, 30, 64, 65, 136, 200])
def test_product(dev, M, N):
    import gdn2_package as gp
    for K in KS[(M + N) % 2::2]:
        q, sx, w, sw, bias = operands(M, N, K, dev, M * N + K)
        for dt, b in ((F32, bias), (BF16, None)):
            y = gp.gdn2_int8_matmul(q, sx, w, sw, bias=b, out_dtype=dt)
            assert y.shape == (M, N) and y.dtype == dt
            check_product(y, *product(q, sx, w, sw, b))


@pytest.mark.parametrize("M,N,K", [(2050, 2100, 200), (4100, 4104, 130), (4097, 4353, 64),
                                   (65600, 70, 40), (70, 20000, 70), (64, 9000, 2000)])
def test_product_of_many_tiles(dev, M, N, K):
    """Enough tiles to choose those of 128 x 128 and of 192 x 128, and long thin products."""
    import gdn2_package as gp
    q, sx, w, sw, bias = operands(M, N, K, dev, K)
    for dt, b in ((F32, None), (BF16, bias.bfloat16())):
        y = gp.gdn2_int8_matmul(q, sx, w, sw, bias=b, out_dtype=dt)
        check_product(y, *product(q, sx, w, sw, b))


@pytest.mark.parametrize("M", [3, 70])
def test_longest_sums_of_the_largest_values(dev, M):
    """All -128 over K = 131071: 2^31 - 16384 - 2^31 / 131072, the largest sum there is."""
    import gdn2_package as gp
    K, N = 131071, 20
    q = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((N, K), -128, dtype=torch.int8, device=dev)
    w[1] = 127
    one = lambda n: torch.ones(n, device=dev)
    y = gp.gdn2_int8_matmul(q, one(M), w, one(N), out_dtype=F32)
    want = torch.full((M, N), 16384.0 * K, dtype=torch.float64, device=dev)
    want[:, 1] = -16256.0 * K
    assert torch.equal(y, want.float())


def test_layouts(dev):
    """Padded rows whose padding is not zero, rows at odd offsets, batches, transposes."""
    import gdn2_package as gp
    M, N, K = 90, 40, 75
    q, sx, w, sw, _ = operands(M, N, K, dev, 1)
    want = gp.gdn2_int8_matmul(q, sx, w, sw, out_dtype=F32)
    check_product(want, *product(q, sx, w, sw))
    wide_q = torch.full((M, 96), 77, dtype=torch.int8, device=dev)
    wide_w = torch.full((N, 80), -55, dtype=torch.int8, device=dev)
    wide_q[:, :K], wide_w[:, :K] = q, w
    for a in (q, wide_q[:, :K], torch.cat([q[:, :1], q], 1)[:, 1:], q.t().contiguous().t()):
        for b in (w, wide_w[:, :K], torch.cat([w[:, :5], w], 1)[:, 5:]):
            assert torch.equal(gp.gdn2_int8_matmul(a, sx, b, sw, out_dtype=F32), want)
    # the last row's padding is outside the storage: copied, not read
    tight = torch.empty((M - 1) * 80 + K, dtype=torch.int8, device=dev).as_strided((M, K), (80, 1))
    tight.copy_(q)
    assert torch.equal(gp.gdn2_int8_matmul(tight, sx, w, sw, out_dtype=F32), want)
    y = gp.gdn2_int8_matmul(q.view(2, 45, K), sx.view(2, 45), w, sw, out_dtype=F32)
    assert y.shape == (2, 45, N) and torch.equal(y.view(M, N), want)
    assert gp.gdn2_int8_matmul(q[0], sx[0], w, sw, out_dtype=F32).shape == (N,)
    assert gp.gdn2_int8_matmul(q[:0], sx[:0], w, sw).shape == (0, N)
    assert torch.equal(gp.gdn2_int8_matmul(q, sx[:1].expand(M), w, sw, out_dtype=F32)[0], want[0])


@pytest.mark.parametrize("M,N", [(40, 2100), (200, 13001)])
def test_rows_far_apart(dev, M, N):
    """Row strides up to the largest that is read in place, and past it (copied); results whose
    rows start anywhere."""
    import gdn2_package as gp
    K = 100
    q, sx, w, sw, bias = operands(M, N, K, dev, 2)
    want = gp.gdn2_int8_matmul(q, sx, w, sw, bias, out_dtype=BF16)
    check_product(gp.gdn2_int8_matmul(q, sx, w, sw, out_dtype=F32), *product(q, sx, w, sw))
    for stride in (1 << 24, (1 << 24) + 16):
        far = torch.empty((M - 1) * stride + 112, dtype=torch.int8, device=dev)
        rows = far.as_strided((M, K), (stride, 1))
        rows.copy_(q)
        assert torch.equal(gp.gdn2_int8_matmul(rows, sx, w, sw, bias, out_dtype=BF16), want)
        del far, rows


def test_the_chain_of_a_layer(dev):
    """norm -> 8 bits -> product approximates the float layer within the steps' size."""
    import gdn2_package as gp
    M, C, N = 33, 256, 96
    x, r = torch.randn((M, C), device=dev).bfloat16(), torch.randn((M, C), device=dev).bfloat16()
    g, W = 1 + 0.1 * torch.randn(C, device=dev), torch.randn((N, C), device=dev) / 16
    w, sw = gp.gdn2_quantize_int8(W)
    q, s, h = gp.gdn2_rms_norm_int8(x, g, residual=r)
    y = gp.gdn2_int8_matmul(q, s, w, sw, out_dtype=F32).double()
    hn = h.double()
    yn = hn * g.double() / (hn.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    ref = yn @ W.double().t()
    # each factor is off by at most half its row's step
    bound = (yn.abs() @ (0.5 * sw.double()[:, None].expand(N, C)).t()) + \
        (0.5 * s.double()[:, None].expand(M, C)) @ (W.double().abs() + 0.5 * sw.double()[:, None]).t()
    assert bool(((y - ref).abs() <= 1.001 * bound).all())


def test_other_stream_and_graph(dev):
    import gdn2_package as gp
    x, wn = torch.randn((70, 96), device=dev), torch.ones(96, device=dev)
    W, sW = gp.gdn2_quantize_int8(torch.randn((48, 96), device=dev))

    def chain():
        q, s, h = gp.gdn2_rms_norm_int8(x, wn, residual=x)
        return gp.gdn2_int8_matmul(q, s, W, sW), h
    want = chain()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = chain()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for k in range(3):
        x.normal_()
        want = chain()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, want)), k


def test_refusals(dev):
    import gdn2_package as gp
    q, sx, w, sw, bias = operands(4, 8, 32, dev, 0)
    mm = gp.gdn2_int8_matmul
    for bad in (lambda: mm(q, sx[:3], w, sw), lambda: mm(q, sx, w[:, :16], sw),
                lambda: mm(q, sx, w, sw[:7]), lambda: mm(q, sx, w, sw, bias=bias[:5]),
                lambda: mm(q, sx, w[None], sw[None]), lambda: mm(q[:, :0], sx, w[:, :0], sw),
                lambda: mm(q.new_zeros((1, 131072)), sx[:1], q.new_zeros((1, 131072)), sw[:1]),
                lambda: gp.gdn2_dequantize_int8(q, sx[:2]),
                lambda: gp.gdn2_quantize_int8(torch.zeros((1, 32769), device=dev)),
                lambda: gp.gdn2_quantize_int8(torch.zeros((), device=dev))):
        with pytest.raises(gp.GDN2ShapeError):
            bad()
    for bad in (lambda: mm(q.int(), sx, w, sw), lambda: mm(q, sx.double(), w, sw),
                lambda: mm(q.cpu(), sx.cpu(), w, sw), lambda: mm(q, sx, w.cpu(), sw.cpu()),
                lambda: mm(q, sx, w, sw, bias=bias.int()),
                lambda: mm(q, sx, w, sw, out_dtype=torch.float16),
                lambda: gp.gdn2_dequantize_int8(q, sx, dtype=torch.int32),
                lambda: gp.gdn2_quantize_int8(q), lambda: gp.gdn2_quantize_int8(sx.cpu())):
        with pytest.raises(gp.GDN2Error):
            bad()
    with pytest.raises(TypeError):
        mm(q, 1.0, w, sw)


@pytest.mark.parametrize("K", [384, 385, 513, 1003, 2049])
@pytest.mark.parametrize("M,N", [(500, 400), (70, 9000), (2050, 2100), (4100, 4104)])
def test_product_of_many_slices(dev, M, N, K):
    """K over many more slices than the ring holds, whole ones and not, in tiles of 64 x 64 (the
    first two sizes), 128 x 128 and 192 x 128."""
    import gdn2_package as gp
    q, sx, w, sw, bias = operands(M, N, K, dev, K)
    for dt, b in ((F32, bias), (BF16, None)):
        y = gp.gdn2_int8_matmul(q, sx, w, sw, bias=b, out_dtype=dt)
        check_product(y, *product(q, sx, w, sw, b))


@pytest.mark.parametrize("M,N", [(40, 9000), (128, 25000), (192, 33000)])
def test_longest_sums_in_tiles(dev, M, N):
    """All -128 over K = 131071 in each of the three tiles."""
    import gdn2_package as gp
    K, ld = 131071, 131072
    q = torch.full((M, ld), -128, dtype=torch.int8, device=dev)[:, :K]
    w = torch.full((N, ld), -128, dtype=torch.int8, device=dev)[:, :K]
    w[1::3] = 127
    w[2::3] = 0
    one = lambda n: torch.ones(n, device=dev)
    y = gp.gdn2_int8_matmul(q, one(M), w, one(N), out_dtype=F32)
    row = torch.empty(N, dtype=torch.float64, device=dev)
    row[0::3], row[1::3], row[2::3] = 16384.0 * K, -16256.0 * K, 0.0
    assert torch.equal(y, row.float().expand(M, N))
