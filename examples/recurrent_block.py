"""A small hybrid stack, trained in float32 and served in 8 bits.

    python examples/recurrent_block.py

Every block adds its mixer's output to the residual stream:

    y, h = rms_norm(x + residual);   p = y W_in^T;   x = mixer(p) W_out^T;   residual = h

with a GDN-2 mixer (matrix state) in the first block and a gated linear recurrence
(vector state) in the second.  Training runs the trainable forms; serving quantises the
weights once, keeps the norms' and the mixers' outputs in 8 bits between the kernels,
prefills a prompt with the scans and then decodes token by token on the states.
"""
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "gdn2-jax-kernel_amd"))
import gdn2_package as gp  # noqa: E402


class Block:
    """kind "gdn2": projections q,k,v,w,b,g of H heads of D; kind "scan": x,b,g of H D
    channels."""

    def __init__(self, kind, H, D, device, generator):
        self.kind, self.H, self.D = kind, H, D
        C, self.parts = H * D, 6 if kind == "gdn2" else 3
        rand = lambda *s: torch.randn(s, device=device, generator=generator)
        self.norm = torch.ones(C, device=device)
        self.w_in = rand(self.parts * C, C) * C ** -0.5
        self.w_out = rand(C, C) * C ** -0.5
        for p in self.parameters():
            p.requires_grad_()

    def parameters(self):
        return [self.norm, self.w_in, self.w_out]

    def inputs(self, p):
        """The mixer's activated inputs from one projection (B, T, parts H D)."""
        xs = p.unflatten(-1, (self.parts, self.H, self.D)).unbind(2)
        if self.kind == "gdn2":
            q, k, v, w, b, g = xs
            return (F.normalize(q, dim=-1), F.normalize(k, dim=-1), v, torch.sigmoid(w),
                    torch.sigmoid(b), -F.softplus(g.float()))
        x, b, g = xs
        return x, -F.softplus(g.float()), torch.sigmoid(b)

    def mix(self, p, state=None, trainable=False):
        """Mixer over a whole sequence: (B, T, H D) and the final state."""
        xs = self.inputs(p)
        if self.kind == "gdn2":
            f = gp.gdn2_pallas_forward_trainable if trainable else gp.gdn2_pallas_forward
            out, state = f(*xs, self.D ** -0.5, h0=state)
        else:
            out, state = gp.gdn2_gated_scan(*xs, h0=state)
        return out.flatten(2), state

    def step(self, p, state):
        """Mixer over one token, the state updated in place."""
        xs = [x[:, 0] for x in self.inputs(p)]
        if self.kind == "gdn2":
            out, _ = gp.gdn2_decode_step(*xs, self.D ** -0.5, state=state, inplace=True)
        else:
            out, _ = gp.gdn2_gated_scan_step(*xs, state=state, inplace=True)
        return out.flatten(1)[:, None]


def train_forward(blocks, x):
    """(B, T, C) through the stack with the trainable forms."""
    residual = torch.zeros_like(x)
    for blk in blocks:
        y, residual = gp.gdn2_rms_norm(x, blk.norm, residual=residual)
        out, _ = blk.mix(F.linear(y, blk.w_in), trainable=True)
        x = F.linear(out.to(x.dtype), blk.w_out)
    return x + residual


class Server:
    """The stack with its weights in 8 bits; one state for each block."""

    def __init__(self, blocks):
        self.blocks = blocks
        self.weights = [(*gp.gdn2_quantize_int8(b.w_in), *gp.gdn2_quantize_int8(b.w_out))
                        for b in blocks]
        self.states = [None] * len(blocks)

    def __call__(self, x):
        """A prompt (B, T, C) from the start, or one more token (B, 1, C)."""
        residual = torch.zeros_like(x)
        for i, (blk, (wi, si, wo, so)) in enumerate(zip(self.blocks, self.weights)):
            q, s, residual = gp.gdn2_rms_norm_int8(x, blk.norm, residual=residual)
            p = gp.gdn2_int8_matmul(q, s, wi, si)
            if self.states[i] is None:
                out, self.states[i] = blk.mix(p)
            else:
                out = blk.step(p, self.states[i])
            q, s = gp.gdn2_quantize_int8(out)
            x = gp.gdn2_int8_matmul(q, s, wo, so)
        return x + residual


def main(steps=20, B=2, T=200, H=2, D=64):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(0)
    blocks = [Block("gdn2", H, D, dev, gen), Block("scan", H, D, dev, gen)]
    params = [p for b in blocks for p in b.parameters()]
    opt = torch.optim.Adam(params, lr=2e-3)
    # a running mean with decay 0.9 of the inputs as the target
    x = torch.randn((B, T, H * D), device=dev, generator=gen)
    decay = torch.full_like(x, 0.9).log()
    with torch.no_grad():
        target, _ = gp.gdn2_gated_scan(0.1 * x, decay)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = F.mse_loss(train_forward(blocks, x), target)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {steps} steps")
    with torch.no_grad():
        whole = train_forward(blocks, x)
        xb, cut = x.bfloat16(), T - 8
        server = Server(blocks)
        outs = [server(xb[:, :cut])] + [server(xb[:, t:t + 1]) for t in range(cut, T)]
        served = torch.cat(outs, 1).float()
        at_once = Server(blocks)(xb).float()
    rms = whole.square().mean().sqrt()
    off = float((served - whole).square().mean().sqrt() / rms)
    same = float((served - at_once).square().mean().sqrt() / rms)
    print(f"serving in 8 bits: off the float32 stack by {off:.4f} of its rms; prompt and "
          f"single tokens off the whole sequence at once by {same:.4f}")
    return losses, off, same


if __name__ == "__main__":
    main()
