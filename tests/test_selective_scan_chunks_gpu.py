"""Selective scan with chunks of 16, 32, 64 and 128 tokens, of each width of the states, against the
recurrence in float64 (test_selective_scan_chunks_cpu.py: that the sizes are cut so).

Tolerances as in test_selective_scan_gpu.py, whose chunks may have 128 tokens.  The longest sums over tokens
here: A's gradient, 128 tokens of a chunk, at most 1500 chunks' partial sums of which a thread adds every
sixteenth, 94, and 16 of those: 238 roundings beside the 1024 of a product of two sums, below 2.5 x 512."""
import pytest
import torch

from test_selective_scan_chunks_cpu import CHUNKED, STATES, WIDE
from test_selective_scan_gpu import BF16, F32, NAMES, call, check, d64, inputs, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("N", STATES)
@pytest.mark.parametrize("L", CHUNKED)
def test_chunks(dev, L, N, types):
    B, T, C, G = CHUNKED[L]
    for cut in (False, True):
        t, starts, dout, dh = inputs(B, T, C, G, N, *types, dev, L + N)
        starts = starts if cut else None
        names = NAMES if cut else tuple(n for n in NAMES if n not in ("z", "D"))
        leaf = {n: t[n].clone().requires_grad_() for n in names}
        out, h = call(leaf, True, starts)
        ref = reference(d64(leaf), starts, True, dout.double(), dh.double())
        check(out, ref["out"])
        check(h, ref["h_final"])
        for n, g in zip(names, torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))):
            assert g.dtype == leaf[n].dtype, n
            check(g, ref[n], 2.5)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("L", WIDE)
def test_more_channels_than_a_wave(dev, L, types):
    B, T, C, G = WIDE[L]
    t, starts, dout, dh = inputs(B, T, C, G, 16, *types, dev, L)
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    out, h = call(leaf, True, starts)
    ref = reference(d64(leaf), starts, True, dout.double(), dh.double())
    check(out, ref["out"])
    check(h, ref["h_final"])
    for n, g in zip(NAMES, torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))):
        check(g, ref[n], 2.5)


@pytest.mark.parametrize("L", CHUNKED)
def test_starts_at_the_sides_of_chunks(dev, L):
    """Starts at the first, last and middle tokens of chunks and of blocks of 16, several in one chunk,
    and chunks without any between those that have them; NaN before a start reaches nothing after it."""
    B, T, C, G = CHUNKED[L]
    t, _, dout, dh = inputs(B, T, C, G, 16, F32, F32, dev, L)
    at = torch.arange(T, device=dev)
    kinds = [at % L == 0, at % L == L - 1, (at % 16 == 0) & (at // L == 1), at == L + 15,
             (at == 1) | (at == T - 1), (at == L // 2) | (at == L // 2 + 1)]
    starts = torch.stack([kinds[b % len(kinds)] for b in range(B)])
    leaf = {n: t[n].clone().requires_grad_() for n in NAMES}
    out, h = call(leaf, True, starts)
    ref = reference(d64(leaf), starts, True, dout.double(), dh.double())
    check(out, ref["out"])
    check(h, ref["h_final"])
    for n, g in zip(NAMES, torch.autograd.grad((out, h), list(leaf.values()), (dout, dh))):
        check(g, ref[n], 2.5)
    bad = {n: v.clone() for n, v in t.items()}
    starts = torch.zeros_like(starts)
    starts[:, L + 3] = True
    bad["x"][:, L + 2], bad["h0"][:] = torch.nan, torch.inf
    out, h = call(bad, True, starts)
    alone = {n: (v[:, L + 3:] if n in ("x", "dt", "B", "C", "z") else v) for n, v in t.items()
             if n != "h0"}
    ref = reference(d64(alone), None, True)
    check(out[:, L + 3:], ref["out"])
    check(h, ref["h_final"])
