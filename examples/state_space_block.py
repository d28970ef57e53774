"""A state space block, trained with 8-bit floating-point products and served token by token.

    python examples/state_space_block.py

The block normalises its input, projects it to x and a gate z, runs the short convolution and the
selective scan over x, and projects back onto the residual stream:

    y, h = rms_norm(x + residual);  x, z = y W_in^T;  x = conv(x);  dt, B, C = x W_x^T;
    out = scan(x, dt W_dt^T, A, B, C, z) W_out^T

All projections but the narrow one of the steps (dt) multiply in 8 bits with a scale for each block
of 128.  Serving quantises the weights once, prefills a prompt and then decodes on the states of
the convolution and the scan.
"""
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "gdn2-jax-kernel_amd"))
import gdn2_package as gp  # noqa: E402


class Block:
    """C channels of the stream, Ci of the block, N states each, steps through R values."""

    def __init__(self, C, Ci, N, R, device, generator):
        self.sizes = Ci, N, R
        rand = lambda *s: torch.randn(s, device=device, generator=generator)
        self.norm = torch.ones(C, device=device)
        self.w_in, self.w_x = rand(2 * Ci, C) * C ** -0.5, rand(R + 2 * N, Ci) * Ci ** -0.5
        self.w_dt, self.w_out = rand(Ci, R) * R ** -0.5, rand(C, Ci) * Ci ** -0.5
        self.conv, self.conv_bias = rand(Ci, 4) * 0.5, torch.zeros(Ci, device=device)
        # steps around 0.01 to 0.1, decays of 1 to N a unit of step
        self.dt_bias = torch.linspace(-4.6, -2.3, Ci, device=device)
        self.log_A = torch.arange(1, N + 1, device=device).float().log().repeat(Ci, 1)
        self.D = torch.ones(Ci, device=device)
        for p in self.parameters():
            p.requires_grad_()

    def parameters(self):
        return [self.norm, self.w_in, self.w_x, self.w_dt, self.w_out, self.conv, self.conv_bias,
                self.dt_bias, self.log_A, self.D]

    def forward(self, x, residual, starts=None):
        """(B, T, C) and the stream, with the trainable forms; starts marks packed sequences."""
        Ci, N, R = self.sizes
        y, h = gp.gdn2_rms_norm(x, self.norm, residual=residual)
        x, z = gp.gdn2_fp8_linear(y, self.w_in).split(Ci, -1)
        x, _ = gp.gdn2_short_conv(x, self.conv, bias=self.conv_bias, starts=starts)
        dt, B, C = gp.gdn2_fp8_linear(x, self.w_x).split((R, N, N), -1)
        out, _ = gp.gdn2_selective_scan(x, F.linear(dt, self.w_dt), -torch.exp(self.log_A), B, C,
                                        D=self.D, z=z, dt_bias=self.dt_bias, dt_softplus=True,
                                        starts=starts)
        return gp.gdn2_fp8_linear(out, self.w_out), h


class Server:
    """The block with its weights in 8 bits and its two states."""

    def __init__(self, block):
        self.block = block
        self.w_in, self.w_x, self.w_out = (gp.gdn2_quantize_fp8(w, blocks=True)
                                           for w in (block.w_in, block.w_x, block.w_out))
        self.A = -torch.exp(block.log_A)
        self.w_dt = block.w_dt.bfloat16()
        self.conv = self.scan = None

    def __call__(self, x, residual):
        """A prompt (B, T, C) from the start, or one more token (B, 1, C), bfloat16."""
        b = self.block
        Ci, N, R = b.sizes
        product = lambda t, w: gp.gdn2_fp8_matmul(*gp.gdn2_quantize_fp8(t), *w)
        y, h = gp.gdn2_rms_norm(x, b.norm, residual=residual)
        x, z = product(y, self.w_in).split(Ci, -1)
        more = self.conv is not None
        if more:
            x, _ = gp.gdn2_short_conv_step(x[:, 0], b.conv, bias=b.conv_bias, state=self.conv,
                                           inplace=True)
        else:
            x, self.conv = gp.gdn2_short_conv(x, b.conv, bias=b.conv_bias)
        dt, B, C = product(x, self.w_x).split((R, N, N), -1)
        kw = dict(D=b.D, dt_bias=b.dt_bias, dt_softplus=True)
        dt = F.linear(dt, self.w_dt)
        if more:
            out, _ = gp.gdn2_selective_scan_step(x, dt, self.A, B, C, z=z[:, 0], state=self.scan,
                                                 inplace=True, **kw)
            out = out[:, None]
        else:
            out, self.scan = gp.gdn2_selective_scan(x, dt, self.A, B, C, z=z, **kw)
        return product(out, self.w_out), h


def main(steps=10, B=2, T=200, C=128, Ci=256, N=16, R=16):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(0)
    block = Block(C, Ci, N, R, dev, gen)
    opt = torch.optim.Adam(block.parameters(), lr=1e-3)
    x = torch.randn((B, T, C), device=dev, generator=gen)
    residual = torch.zeros_like(x)
    starts = torch.zeros((B, T), dtype=torch.bool, device=dev)
    starts[:, T // 2] = True                 # two sequences in a row of the batch
    target = torch.roll(x, 1, 1)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = F.mse_loss(block.forward(x, residual, starts)[0], target)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {steps} steps")
    with torch.no_grad():
        xb, rb, cut = x.bfloat16(), residual.bfloat16(), T - 8
        server = Server(block)
        outs = [server(xb[:, :cut], rb[:, :cut])[0]]
        outs += [server(xb[:, t:t + 1], rb[:, t:t + 1])[0] for t in range(cut, T)]
        served, whole = torch.cat(outs, 1).float(), Server(block)(xb, rb)[0].float()
        exact = block.forward(x, residual)[0]
    rms = lambda t: float(t.square().mean().sqrt())
    off, same = rms(served - exact) / rms(exact), rms(served - whole) / rms(whole)
    print(f"serving: off the float32 block by {off:.4f} of its rms; prompt and single tokens off "
          f"the whole sequence at once by {same:.4f}")
    return losses, off, same


if __name__ == "__main__":
    main()
