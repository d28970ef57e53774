"""Performance cases of the operators that a state space block adds around the GDN-2 mixer.

Three families, each called as a program that trains or serves such a block calls it:

* ``conv``, ``conv_train``, ``conv_step`` -- the short causal convolution over each channel,
  with its activation: a prompt, forward and backward, one decoding token;
* ``scan``, ``scan_train``, ``scan_step`` -- the selective state space scan
  h_t[c,n] = e^{d_t[c] A[c,n]} h_{t-1}[c,n] + d_t[c] x_t[c] B_t[n],
  y_t[c] = sum_n C_t[n] h_t[c,n] + D[c] x_t[c],  out = y silu(z),  d = softplus(dt + dt_bias);
* ``product``, ``linear_train`` -- matrix product in 8-bit floating point (e4m3) with a scale for
  each block of 128: activations quantised and multiplied with a quantised weight, and a linear
  layer trained that way.

Definitions.  A block's scale is the smallest power of two s with max|t| <= 448 s, and its values
are held as e4m3(t / s), ties to even: rows of an activation or of a gradient in blocks of 1 x 128
along the axis that is summed over, weights in blocks of 128 x 128.  The products sum what those
values stand for.  In the convolution and the scan a token marked in ``starts`` begins a sequence:
nothing from before it enters.

Where ``own`` is false the operators run in their plain form, elementary torch operations in
float32; where it is true the package's entry points are called.
"""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gp():
    path = os.path.join(os.getcwd(), "gdn2-jax-kernel_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gdn2_package
    return gdn2_package


def listed():
    return [
        # one decoding token of 32 sequences through the convolution of q, k and v, 6 heads of 128
        {"name": "conv_step_b32", "kind": "conv_step", "B": 32, "C": 2304, "W": 4,
         "dtype": "bf16", "bias": False},
        # a batch of prompts where nothing is a multiple of anything, continued from a state
        {"name": "conv_odd_f32", "kind": "conv", "B": 3, "T": 1001, "C": 1003, "W": 3,
         "dtype": "f32", "bias": True, "state": True, "starts": False},
        # the training step at the size of the package's headline forward, packed sequences
        {"name": "conv_train_bf16", "kind": "conv_train", "B": 8, "T": 8192, "C": 768, "W": 4,
         "dtype": "bf16", "bias": True, "state": False, "starts": True},
        # one decoding token of 32 sequences: the state is read and written once
        {"name": "scan_step_b32", "kind": "scan_step", "B": 32, "C": 1536, "N": 16, "G": 1,
         "dtype": "bf16", "z": True},
        # one prompt of an odd length continued from a state
        {"name": "scan_prompt_bf16", "kind": "scan", "B": 1, "T": 4001, "C": 1536, "N": 16,
         "G": 1, "dtype": "bf16", "dt32": False, "z": True, "h0": True, "starts": False},
        # prefill at the size of the package's headline forward
        {"name": "scan_b8_bf16", "kind": "scan", "B": 8, "T": 8192, "C": 768, "N": 16, "G": 1,
         "dtype": "bf16", "dt32": False, "z": True, "h0": False, "starts": False},
        # a training step of a layer with twice the model's channels
        {"name": "scan_train_bf16", "kind": "scan_train", "B": 8, "T": 2048, "C": 1536, "N": 16,
         "G": 1, "dtype": "bf16", "dt32": False, "z": True, "h0": False, "starts": False},
        # float32, packed sequences, two groups, states of an odd width, no gate
        {"name": "scan_train_odd_f32", "kind": "scan_train", "B": 2, "T": 1003, "C": 500, "N": 21,
         "G": 2, "dtype": "f32", "dt32": True, "z": False, "h0": True, "starts": True},
        # a projection of one decoding step of 32 sequences: the weight is read once
        {"name": "product_decode", "kind": "product", "M": 32, "K": 4096, "N": 4096,
         "dtype": "bf16", "bias": False},
        # a projection of a prefill of 16384 tokens through a wide layer
        {"name": "product_prefill", "kind": "product", "M": 16384, "K": 4096, "N": 4096,
         "dtype": "bf16", "bias": False},
        # a training step of a projection: three products
        {"name": "linear_train_bf16", "kind": "linear_train", "M": 8192, "K": 2048, "N": 4096,
         "dtype": "bf16", "bias": False},
        # nothing a multiple of anything, a bias, float32
        {"name": "linear_train_odd_f32", "kind": "linear_train", "M": 1001, "K": 1003, "N": 777,
         "dtype": "f32", "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width over [lo, hi]: half of them heads of 64 or 128 channels, half any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.5 else min(hi, max(64, n // 64 * 64))


def draw(rng):
    kind = rng.choice(["conv_step", "conv", "conv_train", "scan_step", "scan", "scan", "scan_train",
                       "scan_train", "product", "product", "linear_train", "linear_train"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    coin = lambda p: rng.random() < p
    if kind.startswith("conv"):
        C, W = _width(rng, 64, 4096), rng.choice([2, 3, 4, 4])
        case = {"kind": kind, "B": _log(rng, 1, 512 if kind == "conv_step" else 16), "C": C,
                "W": W, "dtype": dtype, "bias": coin(0.5)}
        if kind != "conv_step":
            T = max(1, min(32768, 8 * 8192 * 768 // (1 if dtype == "bf16" else 2)
                           // (case["B"] * C)))
            case.update(T=_log(rng, 1, T), state=coin(0.5), starts=coin(0.3))
        return case
    if kind.startswith("scan"):
        C, N = _width(rng, 64, 4096), rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 64)])
        G = rng.choice([1, 1, 2, 4])
        C = max(G, C // G * G)
        case = {"kind": kind, "B": _log(rng, 1, 256 if kind == "scan_step" else 16), "C": C, "N": N,
                "G": G, "dtype": dtype, "z": coin(0.6)}
        if kind != "scan_step":
            most = 8 * 8192 * 768 * 16 if kind == "scan" else 8 * 2048 * 1536 * 16
            T = max(1, min(32768, most // (2 if dtype == "f32" else 1) // (case["B"] * C * N)))
            case.update(T=_log(rng, 1, T), dt32=dtype == "f32" or coin(0.3), h0=coin(0.5),
                        starts=coin(0.3))
        return case
    K, N = _width(rng, 64, 8192), _width(rng, 64, 8192)
    most = 16384 * 4096 * 4096 if kind == "product" else 8192 * 2048 * 4096
    M = _log(rng, 1, max(1, min(16384, most // (K * N), 16384 * 4096 // (2 * max(K, N)))))
    return {"kind": kind, "M": M, "K": K, "N": N, "dtype": dtype, "bias": coin(0.5)}


def _grads_wanted(*tensors):
    for t in tensors:
        if t is not None:
            t.requires_grad_()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, dt = case["kind"], _DT[case["dtype"]]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    s = {"case": case}
    if kind in ("product", "linear_train"):
        M, K, N = case["M"], case["K"], case["N"]
        x, w = rand(M, K), rand(N, K) * K ** -0.5
        x *= torch.exp(0.5 * rand(K))     # channels of different sizes, as activations have them
        s["bias"] = rand(N) if case["bias"] else None
        s["x"] = x.to(dt)
        if kind == "linear_train":
            s["w"], s["dy"] = w.to(dt), (rand(M, N) * torch.exp(rand(M, 1))).to(dt)
            _grads_wanted(s["x"], s["w"], s["bias"])
        else:
            # a weight in 8 bits as checkpoints hold it: a float32 scale of any value for a block
            nb, kb = -(-N // 128), -(-K // 128)
            padded = torch.zeros((nb * 128, kb * 128), device="cuda")
            padded[:N, :K] = w
            top = padded.view(nb, 128, kb, 128).abs().amax((1, 3)).clamp_min(1e-30)
            s["sw"] = top / 448.0
            wide = s["sw"].repeat_interleave(128, 0).repeat_interleave(128, 1)
            q = (padded / wide).clamp(-448, 448).to(torch.float8_e4m3fn)
            s["w"] = q[:N, :-(-K // 16) * 16].contiguous()[:, :K]   # rows at multiples of 16 bytes
        return s
    B, C = case["B"], case["C"]
    if kind == "conv_step":
        s["x"], s["state"] = rand(B, C).to(dt), rand(B, case["W"] - 1, C).to(dt)
    elif kind.startswith("conv"):
        s["x"] = rand(B, case["T"], C).to(dt)
        s["state"] = rand(B, case["W"] - 1, C).to(dt) if case["state"] else None
    if kind.startswith("conv"):
        s["w"] = rand(C, case["W"]) * case["W"] ** -0.5
        s["bias"] = rand(C) if case["bias"] else None
    else:
        N, G = case["N"], case["G"]
        lead = (B,) if kind == "scan_step" else (B, case["T"])
        s["x"] = rand(*lead, C).to(dt)
        s["z"] = rand(*lead, C).to(dt) if case["z"] else None
        # steps from 1e-3 to 1e-1 around each channel's bias, decays of 1 to N a unit of step
        step = torch.exp(uniform(C) * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["dt"] = (0.5 * rand(*lead, C)).to(torch.float32 if case.get("dt32") else dt)
        s["A"] = -torch.arange(1, N + 1, device="cuda") * torch.exp(0.1 * rand(C, N))
        s["Bm"], s["Cm"] = rand(*lead, G, N).to(dt), rand(*lead, G, N).to(dt)
        s["D"] = 1.0 + 0.1 * rand(C)
        s["h0"] = rand(B, C, N) if case.get("h0", True) else None
    s["starts"] = None
    if case.get("starts"):     # sequences of some hundred tokens
        s["starts"] = uniform(B, case["T"]) < 1.0 / min(300, case["T"])
        s["starts"][:, 0] = False
    if kind == "conv_train":
        s["dy"], s["dstate"] = rand(B, case["T"], C).to(dt), rand(B, case["W"] - 1, C).to(dt)
        _grads_wanted(s["x"], s["w"], s["bias"], s["state"])
    elif kind == "scan_train":
        s["dy"], s["dh"] = rand(B, case["T"], C).to(dt), rand(B, C, case["N"])
        _grads_wanted(*(s[n] for n in _SCAN_LEAVES))
    return s


_SCAN_LEAVES = ("x", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "h0")


# ---------------------------------------------------------------- plain forms, float32

def _f(t):
    return None if t is None else t.float()


def _taps(s):
    """x at the W tokens up to each token, oldest first, (B, T, C, W), zero before a start."""
    x, W = s["x"].float(), s["case"]["W"]
    before = torch.zeros_like(x[:, :1]).expand(-1, W - 1, -1) if s["state"] is None \
        else s["state"].float()
    taps = torch.cat([before, x], 1).unfold(1, W, 1)
    return taps if s["starts"] is None else taps * _reach(s)


def _reach(s):
    """1 where a token's tap (oldest first) is of its own sequence, (B, T, 1, W)."""
    W = s["case"]["W"]
    past = torch.nn.functional.pad(s["starts"].float().cumsum(1), (W - 1, 0))
    seq = past.unfold(1, W, 1)
    return (seq == seq[..., -1:]).float()[:, :, None]


def _plain_conv(s, train):
    w, b, T, W = s["w"].float(), _f(s["bias"]), s["case"]["T"], s["case"]["W"]
    taps = _taps(s)
    pre = (taps * w).sum(-1)
    pre = pre if b is None else pre + b
    gate = torch.sigmoid(pre)
    res = {"y": (pre * gate).to(s["x"].dtype)}
    # the last W - 1 inputs, those before the last start as zeros
    res["state"] = _last_inputs(s).to(s["x"].dtype)
    if not train:
        return res
    dpre = s["dy"].float() * gate * (1.0 + pre * (1.0 - gate))
    res["dw"] = (dpre[..., None] * taps).sum((0, 1))
    if b is not None:
        res["dbias"] = dpre.sum((0, 1))
    back = dpre[..., None] * w                  # to the tap W - 1 - j tokens ago
    if s["starts"] is not None:
        back = back * _reach(s)
    pad = torch.nn.functional.pad
    parts = [pad(back[..., j], (0, 0, j, W - 1 - j)) for j in range(W)]
    dx = torch.stack(parts).sum(0)              # of state and x
    last = s["dstate"].float()
    if s["starts"] is not None:
        last = last * _kept_inputs(s)
    dx = dx + pad(last, (0, 0, T, 0))
    res["dx"] = dx[:, W - 1:].to(s["x"].dtype)
    if s["state"] is not None:
        res["dstate"] = dx[:, :W - 1].to(s["x"].dtype)
    return res


def _kept_inputs(s):
    """1 where the last W - 1 inputs are of the last token's sequence, (B, W - 1, 1)."""
    seq = torch.nn.functional.pad(s["starts"].float().cumsum(1), (s["case"]["W"] - 1, 0))
    return (seq[:, -(s["case"]["W"] - 1):] == seq[:, -1:]).float()[..., None]


def _last_inputs(s):
    W = s["case"]["W"]
    state = torch.zeros((s["x"].shape[0], W - 1, s["x"].shape[2]), device="cuda") \
        if s["state"] is None else s["state"].float()
    last = torch.cat([state, s["x"].float()], 1)[:, -(W - 1):]
    return last if s["starts"] is None else last * _kept_inputs(s)


def _plain_conv_step(s):
    taps = torch.cat([s["state"], s["x"][:, None]], 1)
    pre = (taps.float() * s["w"].float().t()).sum(1)
    pre = pre if s["bias"] is None else pre + s["bias"].float()
    return {"y": (pre * torch.sigmoid(pre)).to(s["x"].dtype), "state": taps[:, 1:].contiguous()}


def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along the second axis from zero, by doubling."""
    d = 1
    while d < u.shape[1]:
        u = torch.cat([u[:, :d], u[:, d:] + a[:, d:] * u[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return u


def _softplus(v):
    return v.clamp_min(0.0) + torch.log1p(torch.exp(-v.abs()))


def _by_channel(m, C):
    """(..., G, N) for each channel: (..., C, N)."""
    return m.float().repeat_interleave(C // m.shape[-2], -2)


def _by_group(t, G):
    """(..., C, N) summed over each group's channels: (..., G, N)."""
    return t.unflatten(-2, (G, -1)).sum(-2)


def _plain_ssm(s, train):
    C, G = s["case"]["C"], s["case"]["G"]
    x, A, z = s["x"].float(), s["A"].float(), _f(s["z"])
    raw = s["dt"].float() + s["dt_bias"]
    d = _softplus(raw)
    Bc, Cc = _by_channel(s["Bm"], C), _by_channel(s["Cm"], C)
    a = torch.exp(d[..., None] * A)
    if s["starts"] is not None:
        a = a * (~s["starts"])[..., None, None]
    u = (d * x)[..., None] * Bc
    if s["h0"] is not None:
        u = torch.cat([u[:, :1] + a[:, :1] * s["h0"][:, None], u[:, 1:]], 1)
    h = _scan(a, u)
    y = (h * Cc).sum(-1) + s["D"] * x
    gate = None if z is None else torch.sigmoid(z)
    res = {"out": (y if z is None else y * z * gate).to(s["x"].dtype), "h_final": h[:, -1].clone()}
    if not train:
        return res
    dout = s["dy"].float()
    dy = dout
    if z is not None:
        dy = dout * z * gate
        res["dz"] = (dout * y * gate * (1.0 + z * (1.0 - gate))).to(s["z"].dtype)
    e = dy[..., None] * Cc
    e = torch.cat([e[:, :-1], e[:, -1:] + s["dh"][:, None]], 1)
    ahead = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _scan(ahead.flip(1), e.flip(1)).flip(1)
    first = torch.zeros_like(h[:, :1]) if s["h0"] is None else s["h0"][:, None]
    through = dh * a * torch.cat([first, h[:, :-1]], 1)
    dB = (dh * Bc).sum(-1)
    res["dx"] = (d * dB + s["D"] * dy).to(s["x"].dtype)
    draw_ = ((through * A).sum(-1) + x * dB) * torch.sigmoid(raw)
    res["ddt"] = draw_.to(s["dt"].dtype)
    res["dA"] = (through * d[..., None]).sum((0, 1))
    res["dBm"] = _by_group(dh * (d * x)[..., None], G).to(s["Bm"].dtype)
    res["dCm"] = _by_group(h * dy[..., None], G).to(s["Cm"].dtype)
    res["dD"] = (dy * x).sum((0, 1))
    res["ddt_bias"] = draw_.sum((0, 1))
    if s["h0"] is not None:
        res["dh0"] = a[:, 0] * dh[:, 0]
    return res


def _plain_ssm_step(s):
    C, x = s["case"]["C"], s["x"].float()
    d = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(d[..., None] * s["A"]) * s["h0"] \
        + (d * x)[..., None] * _by_channel(s["Bm"], C)
    y = (h * _by_channel(s["Cm"], C)).sum(-1) + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z * torch.sigmoid(z)
    return {"out": y.to(s["x"].dtype), "state": h}


def _pow2(top):
    """The smallest power of two s with top <= 448 s; 448 = 0.875 2^9."""
    part, power = torch.frexp(top)
    power = (power - 9 + (part > 0.875)).clamp_min(-126)
    return torch.ldexp(torch.ones_like(top), power)


def _held(t, rows):
    """What t (M, K) stands for in 8 bits, in blocks of 128 along K and of `rows` rows."""
    M, K = t.shape
    p = torch.nn.functional.pad(t, (0, -K % 128, 0, -M % rows))
    p = p.view(-1, rows, p.shape[1] // 128, 128)
    scale = _pow2(p.abs().amax((1, 3), keepdim=True))
    q = (p / scale).to(torch.float8_e4m3fn).float() * scale
    return q.view(-1, q.shape[2] * 128)[:M, :K]


def _plain_product(s):
    wide = s["sw"].repeat_interleave(128, 0).repeat_interleave(128, 1)
    w = s["w"].float() * wide[:s["w"].shape[0], :s["w"].shape[1]]
    y = _held(s["x"].float(), 1) @ w.t()
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _plain_linear(s):
    x, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
    wq = _held(w, 128)
    y = _held(x, 1) @ wq.t()
    res = {"y": (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype),
           "dx": (_held(dy, 1) @ wq).to(s["x"].dtype),
           "dw": (_held(dy.t(), 1) @ _held(x.t(), 1).t()).to(s["w"].dtype)}
    if s["bias"] is not None:
        res["dbias"] = dy.sum(0)
    return res


def _plain(s):
    kind = s["case"]["kind"]
    with torch.no_grad():
        if kind == "conv_step":
            return _plain_conv_step(s)
        if kind.startswith("conv"):
            return _plain_conv(s, kind == "conv_train")
        if kind == "scan_step":
            return _plain_ssm_step(s)
        if kind.startswith("scan"):
            return _plain_ssm(s, kind == "scan_train")
        return _plain_product(s) if kind == "product" else _plain_linear(s)


# ---------------------------------------------------------------- the package's operators

def _grads(outputs, cotangents, s, names):
    names = [n for n in names if s[n] is not None]
    grads = torch.autograd.grad(outputs, [s[n] for n in names], cotangents)
    return {"d" + n: t for n, t in zip(names, grads)}


def _own(s):
    gp, kind = _gp(), s["case"]["kind"]
    if kind == "conv_step":
        y, state = gp.gdn2_short_conv_step(s["x"], s["w"], bias=s["bias"], state=s["state"])
        return {"y": y, "state": state}
    if kind.startswith("conv"):
        y, state = gp.gdn2_short_conv(s["x"], s["w"], bias=s["bias"], state=s["state"],
                                      starts=s["starts"])
        res = {"y": y, "state": state}
        if kind == "conv_train":
            res.update(_grads((y, state), (s["dy"], s["dstate"]), s, ("x", "w", "bias", "state")))
        return res
    if kind == "scan_step":
        out, state = gp.gdn2_selective_scan_step(
            s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
            dt_softplus=True, state=s["h0"])
        return {"out": out, "state": state}
    if kind.startswith("scan"):
        out, h = gp.gdn2_selective_scan(
            s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
            dt_softplus=True, h0=s["h0"], starts=s["starts"])
        res = {"out": out, "h_final": h}
        if kind == "scan_train":
            res.update(_grads((out, h), (s["dy"], s["dh"]), s, _SCAN_LEAVES))
        return res
    if kind == "product":
        q, scale = gp.gdn2_quantize_fp8(s["x"])
        return gp.gdn2_fp8_matmul(q, scale, s["w"], s["sw"], bias=s["bias"],
                                  out_dtype=s["x"].dtype)
    y = gp.gdn2_fp8_linear(s["x"], s["w"], bias=s["bias"])
    return {"y": y, **_grads((y,), (s["dy"],), s, ("x", "w", "bias"))}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each input read once, each output written once; the operations of the definition."""
    e, kind = (2 if case["dtype"] == "bf16" else 4), case["kind"]
    if kind == "product":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": e * M * K + N * K + N * K // 4096 + e * M * N, "flops": 2 * M * N * K}
    if kind == "linear_train":   # x, w, dy read; y, dx, dw written
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": 2 * e * (M * K + N * K + M * N), "flops": 6 * M * N * K}
    B, C, T = case["B"], case["C"], case.get("T", 1)
    n = B * T * C
    if kind.startswith("conv"):
        W = case["W"]
        bytes_, flops = 2 * n * e + 2 * B * (W - 1) * C * e + 4 * C * W, n * (2 * W + 4)
        if kind == "conv_train":   # x and dy read, dx written
            bytes_, flops = bytes_ + 3 * n * e + 4 * C * W, flops + n * (4 * W + 8)
        return {"bytes": bytes_, "flops": flops}
    N, G, ed = case["N"], case["G"], 4 if case.get("dt32") else e
    ins = n * (e + ed + (e if case["z"] else 0)) + 2 * B * T * G * N * e
    state = 4 * B * C * N * (2 if case.get("h0", True) else 1)
    bytes_, flops = ins + n * e + state + 4 * C * N, n * (7 * N + 12)
    if kind == "scan_train":       # dout and the inputs again; a gradient of each input
        bytes_, flops = bytes_ + n * e + 2 * ins + state + 8 * C * N, flops + n * (18 * N + 20)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_conv(s, train):
    x, w, W = s["x"].double(), s["w"].double(), s["case"]["W"]
    B, T, C = x.shape
    before = torch.zeros((B, W - 1, C), dtype=torch.float64, device="cuda") \
        if s["state"] is None else s["state"].double()
    line = torch.cat([before, x], 1)               # position p holds token p - (W - 1)
    number = torch.zeros((B, T + W - 1), dtype=torch.long, device="cuda")
    if s["starts"] is not None:
        number[:, W - 1:] = s["starts"].long().cumsum(1)
    same = [(number[:, k:k + T] == number[:, W - 1:])[..., None] for k in range(W)]
    pre = torch.zeros_like(x) if s["bias"] is None else s["bias"].double().expand_as(x).clone()
    for k in range(W):
        pre += torch.where(same[k], line[:, k:k + T], 0.0) * w[:, k]
    kept = (number[:, T:] == number[:, -1:])[..., None]
    res = {"y": pre / (1.0 + torch.exp(-pre)), "state": torch.where(kept, line[:, T:], 0.0)}
    if not train:
        return res
    sig = 1.0 / (1.0 + torch.exp(-pre))
    dpre = s["dy"].double() * (sig + pre * sig * (1.0 - sig))
    dline = torch.zeros_like(line)
    dw = torch.zeros_like(w)
    for k in range(W):
        part = torch.where(same[k], dpre, 0.0)
        dline[:, k:k + T] += part * w[:, k]
        dw[:, k] = (part * line[:, k:k + T]).sum((0, 1))
    dline[:, T:] += torch.where(kept, s["dstate"].double(), 0.0)
    res.update(dw=dw, dx=dline[:, W - 1:])
    if s["bias"] is not None:
        res["dbias"] = dpre.sum((0, 1))
    if s["state"] is not None:
        res["dstate"] = dline[:, :W - 1]
    return res


def _exact_ssm(s, train):
    B, T, C = s["x"].shape
    G, N = s["Bm"].shape[2:]
    x, A = s["x"].double(), s["A"].double()
    raw = s["dt"].double() + s["dt_bias"].double()
    d = torch.logaddexp(raw, torch.zeros_like(raw))
    at = lambda m, t: m[:, t].double()[:, :, None].expand(B, G, C // G, N).reshape(B, C, N)
    h = torch.zeros((B, C, N), dtype=torch.float64, device="cuda") if s["h0"] is None \
        else s["h0"].double().clone()
    starts = [False] * T if s["starts"] is None else s["starts"].any(0).tolist()
    y, before = torch.empty_like(x), []

    def decay(t):
        a = torch.exp(d[:, t, :, None] * A)
        return a * (~s["starts"][:, t]).double()[:, None, None] if starts[t] else a

    for t in range(T):
        if train:
            before.append(h)
        h = decay(t) * h + (d[:, t] * x[:, t])[..., None] * at(s["Bm"], t)
        y[:, t] = (h * at(s["Cm"], t)).sum(-1)
    y += s["D"].double() * x
    z = None if s["z"] is None else s["z"].double()
    sig = None if z is None else torch.sigmoid(z)
    res = {"out": y if z is None else y * z * sig, "h_final": h}
    if not train:
        return res
    dout = s["dy"].double()
    dy = dout if z is None else dout * z * sig
    if z is not None:
        res["dz"] = dout * y * sig * (1.0 + z * (1.0 - sig))
    e, dA = s["dh"].double().clone(), torch.zeros_like(A)
    dx, dd = s["D"].double() * dy, torch.empty_like(x)
    dB = torch.empty((B, T, G, N), dtype=torch.float64, device="cuda")
    dC = torch.empty_like(dB)
    for t in reversed(range(T)):
        a, Bt = decay(t), at(s["Bm"], t)
        now = a * before[t] + (d[:, t] * x[:, t])[..., None] * Bt
        dC[:, t] = (now * dy[:, t, :, None]).view(B, G, C // G, N).sum(2)
        e = e + dy[:, t, :, None] * at(s["Cm"], t)
        dB[:, t] = (e * (d[:, t] * x[:, t])[..., None]).view(B, G, C // G, N).sum(2)
        inner = (e * Bt).sum(-1)
        e_a = e * a
        back = e_a * before[t]
        dA += (back * d[:, t, :, None]).sum(0)
        dd[:, t] = (back * A).sum(-1) + x[:, t] * inner
        dx[:, t] += d[:, t] * inner
        e = e_a
    dd = dd * torch.sigmoid(raw)
    res.update(dx=dx, ddt=dd, dA=dA, dBm=dB, dCm=dC, dD=(dy * x).sum((0, 1)),
               ddt_bias=dd.sum((0, 1)))
    if s["h0"] is not None:
        res["dh0"] = e
    return res


def _stands_for(t, down, along):
    """The values of t (64 bits) in e4m3 with a power of two for each down x along block."""
    out = torch.empty_like(t)
    pad = torch.zeros((-(-t.shape[0] // down) * down, -(-t.shape[1] // along) * along),
                      dtype=torch.float64, device="cuda")
    pad[:t.shape[0], :t.shape[1]] = t
    cells = pad.reshape(pad.shape[0] // down, down, pad.shape[1] // along, along)
    top = cells.abs().amax(3).amax(1)
    scale = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp_min(-126.0))[:, None, :, None]
    v = cells / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    out.copy_((torch.round(v / step) * step * scale).reshape(pad.shape)[:t.shape[0], :t.shape[1]])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "conv_step":
            taps = torch.cat([s["state"], s["x"][:, None]], 1).double()
            pre = torch.zeros_like(taps[:, 0]) if s["bias"] is None else s["bias"].double()
            for k in range(case["W"]):
                pre = pre + taps[:, k] * s["w"][:, k].double()
            return {"y": pre / (1.0 + torch.exp(-pre)), "state": taps[:, 1:]}
        if kind.startswith("conv"):
            return _exact_conv(s, kind == "conv_train")
        if kind == "scan_step":
            one = dict(s, starts=None, **{n: None if s[n] is None else s[n][:, None]
                                          for n in ("x", "dt", "z", "Bm", "Cm")})
            res = _exact_ssm(one, False)
            return {"out": res["out"][:, 0], "state": res["h_final"]}
        if kind.startswith("scan"):
            return _exact_ssm(s, kind == "scan_train")
        x = s["x"].double()
        bias = 0.0 if s["bias"] is None else s["bias"].double()
        if kind == "product":
            w = s["w"].double()
            n, k = (torch.arange(m, device="cuda") // 128 for m in w.shape)
            w = w * s["sw"].double()[n][:, k]
            return _stands_for(x, 1, 128) @ w.t() + bias
        w, dy = s["w"].double(), s["dy"].double()
        wq = _stands_for(w, 128, 128)
        res = {"y": _stands_for(x, 1, 128) @ wq.t() + bias, "dx": _stands_for(dy, 1, 128) @ wq,
               "dw": _stands_for(dy, 128, 1).t() @ _stands_for(x, 128, 1)}
        if s["bias"] is not None:
            res["dbias"] = dy.sum(0)
        return res
