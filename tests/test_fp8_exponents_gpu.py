"""The bfloat16 linear layer's products with tiles of 128 x 128 and of 64 x 64 over many slices of 128
values, whose scales the matrix instruction applies: exponents are read four slices at a time, and whole
slices with others behind them run in a loop without branches.  Every block of the sum has a scale of
its own, so that one block's in another's place would show.  Tolerances as in test_fp8_gpu.py."""
import pytest
import torch

from test_fp8_gpu import BF16, check, held, product, values

pytestmark = pytest.mark.gpu


def uneven(M, K, dev, seed):
    """values() with each 128 x 128 block times a power of two from 2^-4 to 2^4."""
    t = values(M, K, BF16, dev, seed)
    gen = torch.Generator(device=dev).manual_seed(seed + 100)
    e = torch.randint(-4, 5, (-(-M // 128), -(-K // 128)), generator=gen, device=dev)
    wide = e.repeat_interleave(128, 0)[:M].repeat_interleave(128, 1)[:, :K]
    return (t.double() * torch.exp2(wide.double())).to(BF16)


# y, dx and dw have more than three 64 x 64 tiles for each of 256 CUs (tiles of 128 x 128, sums of 15 to 18
# slices), or between one and three (tiles of 64 x 64, sums of 10 to 12)
@pytest.mark.parametrize("M,N,K", [(2100, 2050, 2000), (1800, 2304, 1920), (1200, 1300, 1500),
                                   (1153, 1153, 1153)])
def test_linear(dev, M, N, K):
    import gdn2_package as gp
    x, w, dy = uneven(M, K, dev, 1), uneven(N, K, dev, 2), uneven(M, N, dev, 3)
    bias = torch.randn(N, device=dev)
    leaf = [t.requires_grad_() for t in (x, w, bias)]
    y = gp.gdn2_fp8_linear(*leaf)
    xd, wd, dd = (t.detach().double() for t in (x, w, dy))
    wb = held(wd, 128, 128)[0]
    check(y.detach(), product(held(xd, 1, 128)[0], wb, bias.detach()), K)
    dx, dw, _ = torch.autograd.grad(y, leaf, dy)
    check(dx, product(held(dd, 1, 128)[0], wb.t()), N)
    check(dw, product(held(dd.t(), 1, 128)[0], held(xd.t(), 1, 128)[0]), M)
    # a block's share of a sum is far above the tolerance: leaving the second out would not pass
    short = xd.clone()
    short[:, 128:256] = 0
    with pytest.raises(AssertionError):
        check(y.detach(), product(held(short, 1, 128)[0], wb, bias.detach()), K)


@pytest.mark.parametrize("where", ["first", "loop", "last"])
def test_nan_in_one_block(dev, where):
    """A row's block whose scale is NaN reaches that row alone, whichever slice it is."""
    import gdn2_package as gp
    M, N, K = 2100, 2050, 2000
    x, w = uneven(M, K, dev, 4), uneven(N, K, dev, 5)
    at = {"first": 5, "loop": 128 * 5 + 17, "last": K - 1}[where]
    x[1000, at], w[700, at] = torch.nan, torch.inf
    y = gp.gdn2_fp8_linear(x, w)
    bad = torch.zeros((M, N), dtype=torch.bool, device=dev)
    bad[1000], bad[:, 640:768] = True, True
    assert torch.equal(torch.isnan(y), bad)
