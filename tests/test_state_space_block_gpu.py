"""The short convolution, the selective scan and the 8-bit products together, as the example uses
them: it runs, its gradients are those of its definition, and serving follows training.

Gradients are compared with a float64 block whose products round to 8 bits in the same way and whose
gradients pass those roundings as the layer defines.  What differs is where a float32 value lies so near
the middle of two e4m3 values that it goes the other way: values carry errors of some 1e-5 of
their size, eight such middles lie in each factor of two, so about one in 10^4 values changes by 2^-4
of itself: 6e-4 of a norm for each of the up to five roundings that a gradient passes, 3e-3 in
all, tested at 1e-2.

Serving: prompt and single tokens against the whole sequence at once go the same way but for the order
of sums in the scan, which can turn a bfloat16 rounding (2^-8 of a value, in about one of 10^3) and by it
8-bit ones (2^-4, in about one of 50 values whose neighbour in bfloat16 is taken): below 1% of the rms.
Against the float32 block: a bfloat16 rounding of 2^-9 turns one 8-bit value in 32 (steps of 2^-3 to
2^-4), which then is off by up to a step: 1.6% of a norm for each of the three products' inputs; out is a
product of four factors that come from them (x, dt or B, C, z), which add up: below 10%."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "state_space_block.py"
    spec = importlib.util.spec_from_file_location("state_space_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def held(t, down, along):
    M, K = t.shape
    pad = torch.zeros((-(-M // down) * down, -(-K // along) * along), dtype=t.dtype, device=t.device)
    pad[:M, :K] = t
    cells = pad.view(pad.shape[0] // down, down, pad.shape[1] // along, along)
    s = torch.exp2(torch.ceil(torch.log2(cells.abs().amax((1, 3), keepdim=True) / 448.0))
                   .clamp_min(-126.0))
    v = cells / s
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    return (torch.round(v / step) * step * s).reshape(pad.shape)[:M, :K]


class Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return (held(x.flatten(0, -2), 1, 128) @ held(w, 128, 128).t()).view(*x.shape[:-1], -1)

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        d, rows = dy.flatten(0, -2), x.flatten(0, -2)
        return ((held(d, 1, 128) @ held(w, 128, 128)).view(x.shape),
                held(d.t(), 1, 128) @ held(rows.t(), 1, 128).t())


def block64(params, sizes, x, residual, starts):
    Ci, N, R = sizes
    norm, w_in, w_x, w_dt, w_out, conv, conv_bias, dt_bias, log_A, D = params
    h = x + residual
    y = h * norm / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    x, z = Linear.apply(y, w_in).split(Ci, -1)
    T = x.shape[1]
    seq = torch.nn.functional.pad(starts.long().cumsum(1), (3, 0))
    line = torch.nn.functional.pad(x, (0, 0, 3, 0))
    pre = conv_bias + sum(torch.where((seq[:, k:k + T] == seq[:, 3:])[..., None], line[:, k:k + T],
                                      0.0) * conv[:, k] for k in range(4))
    x = pre * torch.sigmoid(pre)
    dt, B, C = Linear.apply(x, w_x).split((R, N, N), -1)
    d = torch.nn.functional.softplus(dt @ w_dt.t() + dt_bias, threshold=1e9)
    a = torch.exp(d[..., None] * -torch.exp(log_A)) * ~starts[..., None, None]
    s, ys = torch.zeros_like(a[:, 0]), []
    for t in range(T):
        s = a[:, t] * s + (d[:, t] * x[:, t])[..., None] * B[:, t, None]
        ys.append((s * C[:, t, None]).sum(-1))
    y = torch.stack(ys, 1) + D * x
    return Linear.apply(y * z * torch.sigmoid(z), w_out)


def test_gradients(dev):
    mod = example()
    gen = torch.Generator(device=dev).manual_seed(1)
    block = mod.Block(96, 160, 16, 8, dev, gen)
    x, dy = (torch.randn((2, 90, 96), device=dev, generator=gen) for _ in range(2))
    residual = torch.randn((2, 90, 96), device=dev, generator=gen)
    starts = torch.rand((2, 90), device=dev, generator=gen) < 0.03
    leaf = [x.requires_grad_(), *block.parameters()]
    out, _ = block.forward(x, residual, starts)
    got = torch.autograd.grad(out, leaf, dy)
    wide = [p.detach().double().requires_grad_() for p in leaf]
    ref = block64(wide[1:], block.sizes, wide[0], residual.double(), starts)
    want = torch.autograd.grad(ref, wide, dy.double())
    for a, b in zip((out, *got), (ref, *want)):
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) < 1e-2


def test_example_trains_and_serves(dev):
    losses, off, same = example().main(steps=3)
    assert all(0.0 < v < 100.0 for v in losses)
    assert off < 0.1 and same < 0.01
