"""What gdn2_fp8_matmul and gdn2_fp8_linear keep of a block's products where these are far apart.

A bfloat16 result: the matrix instruction keeps of eight products at a time what lies above 2^-13 of the
largest one, so the other seven lose at most 7 2^-13 < 2^-10 of it.  A float32 result: products are exact
and at most 128 of a block are added in float32; here all sums are below 2^24 times the smallest
product's last bit, so that they are exact.  Scales are powers of two and exact."""
import pytest
import torch

from test_fp8_gpu import BF16, E4M3, F32

pytestmark = pytest.mark.gpu


def far_apart(M, N, K, dev):
    """Codes x, w (float64 values) with a product of 2^15 and one of -2^15 among every sixteen, which cancel,
    and products of 1, 2, 4 and 8 between them."""
    k = torch.arange(K, device=dev)
    # x: 128 at the first of sixteen, -128 at the second, else 2^0 .. 2^3 by k and the row
    x = 2.0 ** ((k[None] + torch.arange(M, device=dev)[:, None]) % 4).double()
    w = torch.where((k[None] + torch.arange(N, device=dev)[:, None]) % 3 == 0, 0.0, 1.0).double()
    x[:, k % 16 == 0], x[:, k % 16 == 1] = 128.0, -128.0
    w[:, k % 16 < 2] = 256.0
    return x, w


@pytest.mark.parametrize("M,N,K", [(5, 40, 640), (24, 70, 1000), (70, 300, 1000), (300, 500, 1100),
                                   (1200, 1300, 1100), (2100, 2100, 1000)])
def test_products_far_apart(dev, M, N, K):
    import gdn2_package as gp
    x, w = far_apart(M, N, K, dev)
    value, mag = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
    kb = -(-K // 128)
    for rows in (N, -(-N // 128)):
        args = (x.to(E4M3), torch.ones((M, kb), device=dev), w.to(E4M3),
                torch.ones((rows, kb), device=dev))
        assert torch.equal(args[0].double(), x) and torch.equal(args[2].double(), w)
        # the pairs of +- 2^15 only cancel where a row's last sixteen are whole
        exact = gp.gdn2_fp8_matmul(*args, out_dtype=F32)
        assert torch.equal(exact.double(), value)
        fast = gp.gdn2_fp8_matmul(*args, out_dtype=BF16)
        bound = 2.0 ** -10 * mag + 2.0 ** -8 * value.abs()
        assert ((fast.double() - value).abs() <= bound).all()
        # a caller who needs the small products rounds a float32 result
        assert torch.equal(exact.to(BF16), value.to(BF16))


@pytest.mark.parametrize("M,N,K", [(24, 70, 640), (300, 500, 1100)])
def test_linear_in_float32(dev, M, N, K):
    """The linear layer over float32 copies of the same values adds in float32."""
    import gdn2_package as gp
    x, w = far_apart(M, N, K, dev)
    # every block's largest value is 128 or 256: scales 2^-1 and 1 (2^-1 and 2^-2 without a remainder), exact
    y = gp.gdn2_fp8_linear(x.float(), w.float())
    assert torch.equal(y.double(), x @ w.t().contiguous())
    fast = gp.gdn2_fp8_linear(x.to(BF16), w.to(BF16))
    mag = x.abs() @ w.abs().t().contiguous()
    value = x @ w.t().contiguous()
    assert ((fast.double() - value).abs() <= 2.0 ** -10 * mag + 2.0 ** -8 * value.abs()).all()
