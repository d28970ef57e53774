"""So many channels that the kernels which add partial sums have more columns than one launch has
workgroups (CPU: test_launch_sizes_host.py)."""
import pytest
import torch

from test_short_conv_gpu import F32, check, d64, inputs, reference

pytestmark = pytest.mark.gpu


def test_conv_backward(dev):
    """13.6 million channels of 4 taps: 68 million columns, 16 for each of 2^20 workgroups at a time."""
    import gdn2_package as gp
    t, _, dy, dlast = inputs(1, 2, 13_600_004, 4, F32, dev, 1)
    leaf = [t[n].clone().requires_grad_() for n in ("x", "weight", "bias", "state")]
    outs = gp.gdn2_short_conv(leaf[0], leaf[1], bias=leaf[2], state=leaf[3])
    ref = reference(*map(d64, leaf), None, True, d64(dy), d64(dlast))
    check(outs[0], ref["y"])
    for n, g in zip(("x", "weight", "bias", "state"), torch.autograd.grad(outs, leaf, (dy, dlast))):
        check(g, ref[n])


def test_scan_backward(dev):
    """4.2 million channels of 16 states: 75 million columns, 64 for each of 2^20 workgroups at a time.
    Groups of 16 channels, so that a sum over a group is one workgroup's."""
    import test_selective_scan_gpu as scan
    t, _, dout, dh = scan.inputs(1, 2, 1 << 22, 1 << 18, 16, F32, F32, dev, 2)
    leaf = {n: t[n].clone().requires_grad_() for n in scan.NAMES}
    out, h = scan.call(leaf, True)
    ref = scan.reference(scan.d64(leaf), None, True, dout.double(), dh.double())
    scan.check(out, ref["out"])
    scan.check(h, ref["h_final"])
    for n, g in zip(scan.NAMES, torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))):
        scan.check(g, ref[n], 2.5)
