"""Short convolution with 64 lanes across the channels: forward with four channels a thread, backward with
two and one, and its runs of 64 tokens.  Tolerances as in test_short_conv_gpu.py."""
import pytest
import torch

from test_short_conv_gpu import BF16, F32, check, d64, inputs, reference

pytestmark = pytest.mark.gpu


def both_directions(B, T, C, W, dtype, dev, terms):
    import gdn2_package as gp
    for starts in (False, True):
        t, cut, dy, dlast = inputs(B, T, C, W, dtype, dev, T + C + W, starts)
        if starts and T > 64:   # far from each other too
            cut &= torch.arange(T, device=dev) % 32 < 3
        leaf = [t[n].clone().requires_grad_() for n in ("x", "weight", "bias", "state")]
        outs = gp.gdn2_short_conv(leaf[0], leaf[1], bias=leaf[2], state=leaf[3], starts=cut)
        ref = reference(*map(d64, leaf), cut, True, d64(dy), d64(dlast), terms)
        check(outs[0], ref["y"])
        check(outs[1], ref["last"])
        for n, g in zip(("x", "weight", "bias", "state"),
                        torch.autograd.grad(outs, leaf, (dy, dlast))):
            check(g, ref[n])


# 252: a tile with a lane off; 768 and 1020: several tiles
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("B,T,C", [(1, 1, 256), (2, 2, 256), (2, 40, 252), (1, 70, 768), (3, 133, 256),
                                   (1, 1030, 1020)])
def test_lanes(dev, B, T, C, W, dtype):
    both_directions(B, T, C, W, dtype, dev, 128)


# At least 1536 workgroups of 4 runs of 64 tokens: 128 and 124 channels two a thread, 61 one a thread.
# A weight's sum: 64 tokens, 4 runs, at most 1800 rows of partial sums of which a thread adds every
# 64th, 29, and 64 of those: 161.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,C,W", [(1540, 70, 128, 4), (600, 600, 124, 3), (1600, 133, 61, 4),
                                     (790, 300, 128, 2)])
def test_long_runs(dev, B, T, C, W, dtype):
    from gdn2_package import _lib
    # a row of sums for each 4 runs
    assert _lib.lib().gdn2_short_conv_bwd_workspace_bytes(B, T, C, W) == \
        B * -(-T // 256) * C * (W + 1) * 4
    both_directions(B, T, C, W, dtype, dev, 192)
