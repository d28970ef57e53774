"""Performance cases of the operators around the GDN-2 mixer in a recurrent block.

Three families, each called as a program that trains or serves such a block calls it:

* ``scan``, ``scan_train``, ``step`` -- the gated linear recurrence
  h_t = e^{g_t} h_{t-1} + b_t x_t, elementwise over the channels: forward, forward and
  backward, one decoding token;
* ``norm8``, ``norm_train`` -- RMS norm of x + residual: with an output in 8 bits and a
  scale for each row, and in the input's type with its backward;
* ``product`` -- matrix product in 8-bit integers with a scale for each token (row of the
  activations) and each channel (row of the weight).

Definitions.  h = x + residual is returned in the residual's type, and the norm is that of h
as returned: y = h w / sqrt(mean(h^2) + eps).  In 8 bits a row is q = round(127 t / max|t|),
ties to even, with t = h w, and stands for q max|t| / (127 sqrt(mean(h^2) + eps)).

Where ``own`` is false the operators run in their plain form, elementary torch operations in
float32; where it is true the package's entry points are called.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gp():
    path = os.path.join(os.getcwd(), "gdn2-jax-kernel_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gdn2_package
    return gdn2_package


def listed():
    return [
        # one decoding token of 32 sequences, 6 heads of 128 channels: launch and latency
        {"name": "step_b32", "kind": "step", "B": 32, "C": 768, "dtype": "bf16"},
        # one prompt of an odd length continued from a state: few channels, a long axis
        {"name": "scan_prompt_bf16", "kind": "scan", "B": 1, "T": 4001, "C": 768,
         "dtype": "bf16", "gate": True, "h0": True},
        # prefill at the size of the package's headline forward
        {"name": "scan_b8_bf16", "kind": "scan", "B": 8, "T": 8192, "C": 768,
         "dtype": "bf16", "gate": True, "h0": False},
        # one long context of 8 heads of 128 channels, float32, no input gate
        {"name": "scan_long_f32", "kind": "scan", "B": 1, "T": 131072, "C": 1024,
         "dtype": "f32", "gate": False, "h0": False},
        # the training step at the size of the package's headline forward
        {"name": "scan_train_bf16", "kind": "scan_train", "B": 8, "T": 8192, "C": 768,
         "dtype": "bf16", "gate": True, "h0": True},
        # a decoding step's norm: 32 rows
        {"name": "norm8_decode", "kind": "norm8", "M": 32, "C": 768, "dtype": "bf16",
         "residual": True},
        # a prefill's norm, 8 x 8192 tokens
        {"name": "norm8_prefill", "kind": "norm8", "M": 65536, "C": 768, "dtype": "bf16",
         "residual": True},
        # the norm of a training step with a wide residual stream
        {"name": "norm_train_bf16", "kind": "norm_train", "M": 16384, "C": 4096,
         "dtype": "bf16", "residual": True},
        # the six projections of one decoding step of 32 sequences: the weight is read once
        {"name": "product_decode", "kind": "product", "M": 32, "K": 768, "N": 4608,
         "dtype": "bf16", "bias": False},
        # a middling batch through a wide layer
        {"name": "product_mid", "kind": "product", "M": 512, "K": 4096, "N": 4096,
         "dtype": "bf16", "bias": False},
        # the six projections of a prefill, 8 x 8192 tokens
        {"name": "product_prefill", "kind": "product", "M": 65536, "K": 768, "N": 4608,
         "dtype": "bf16", "bias": False},
        # nothing a multiple of anything, a bias, float32 results
        {"name": "product_odd_f32", "kind": "product", "M": 1001, "K": 1003, "N": 777,
         "dtype": "f32", "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width over [lo, hi]: half of them heads of 64 or 128 channels, half any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.5 else min(hi, max(64, n // 64 * 64))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "scan_train", "scan_train", "norm8", "norm8",
                       "norm_train", "norm_train", "product", "product", "product"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "step":
        return {"kind": kind, "B": _log(rng, 1, 512), "C": _width(rng, 64, 8192), "dtype": dtype}
    if kind in ("scan", "scan_train"):
        most = 131072 * 1024 if kind == "scan" else 8 * 8192 * 768
        if dtype == "f32":
            most //= 2
        C, B = _width(rng, 64, 4096), _log(rng, 1, 16)
        T = max(1, min(131072, most // (B * C)))
        return {"kind": kind, "B": B, "T": _log(rng, 1, T), "C": C, "dtype": dtype,
                "gate": rng.random() < 0.7, "h0": rng.random() < 0.5}
    if kind in ("norm8", "norm_train"):
        C = _width(rng, 64, 8192)
        most = 65536 * 768 // (2 if dtype == "f32" else 1)
        return {"kind": kind, "M": _log(rng, 1, min(65536, most // C)), "C": C, "dtype": dtype,
                "residual": rng.random() < 0.75}
    K, N = _width(rng, 64, 8192), _width(rng, 64, 8192)
    M = _log(rng, 1, min(65536, 65536 * 768 * 4608 // (K * N), 65536 * 4608 // (2 * N)))
    return {"kind": kind, "M": M, "K": K, "N": N, "dtype": dtype, "bias": rng.random() < 0.5}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows8(t):
    """Rows of t in 8 bits and their scales.  Rows start at multiples of 16 bytes, as the
    package's quantiser lays them out."""
    m = t.abs().amax(-1)
    ld = -(-t.shape[1] // 16) * 16
    q = torch.zeros((t.shape[0], ld), dtype=torch.int8, device=t.device)[:, :t.shape[1]]
    q.copy_(torch.round(t * (127.0 / m)[:, None]).to(torch.int8))
    return q, m / 127.0


def prepare(case, seed):
    gen, kind, dt = _generator(seed), case["kind"], _DT[case["dtype"]]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    s = {"case": case}
    if kind in ("step", "scan", "scan_train"):
        shape = (case["B"], case["C"]) if kind == "step" else (case["B"], case["T"], case["C"])
        x, b = rand(*shape).to(dt), torch.sigmoid(rand(*shape)).to(dt)
        # decays from a few tokens to some hundreds, another for each channel
        g = -torch.nn.functional.softplus(rand(*shape))
        g *= torch.exp(-4.0 * torch.rand(case["C"], generator=gen, device="cuda"))
        if case.get("gate", True) is False:
            b = None
        h0 = rand(case["B"], case["C"]) if case.get("h0", True) else None
        s.update(x=x, g=g, b=b, h0=h0)
        if kind == "scan_train":
            s.update(dout=rand(*shape).to(dt), dh=rand(case["B"], case["C"]))
            for t in (x, g, b, h0):
                if t is not None:
                    t.requires_grad_()
    elif kind in ("norm8", "norm_train"):
        shape = (case["M"], case["C"])
        s["x"] = rand(*shape).to(dt)
        s["r"] = (4.0 * rand(*shape)).to(dt) if case["residual"] else None
        s["w"] = 1.0 + 0.2 * rand(case["C"])
        if kind == "norm_train":
            s.update(dy=rand(*shape).to(dt), dh=rand(*shape).to(dt))
            for t in (s["x"], s["r"], s["w"]):
                if t is not None:
                    t.requires_grad_()
    else:
        s["x"], s["sx"] = _rows8(rand(case["M"], case["K"]))
        s["w"], s["sw"] = _rows8(rand(case["N"], case["K"]) * case["K"] ** -0.5)
        s["bias"] = rand(case["N"]) if case["bias"] else None
    return s


# ---------------------------------------------------------------- plain forms, float32

def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along the second axis from zero, by doubling."""
    d = 1
    while d < u.shape[1]:
        u = torch.cat([u[:, :d], u[:, d:] + a[:, d:] * u[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return u


def _plain_scan(s, train):
    x, a = s["x"].float(), torch.exp(s["g"].float())
    b = None if s["b"] is None else s["b"].float()
    u = x if b is None else b * x
    if s["h0"] is not None:
        u = torch.cat([u[:, :1] + a[:, :1] * s["h0"][:, None], u[:, 1:]], 1)
    h = _scan(a, u)
    res = {"out": h.to(s["x"].dtype), "h_final": h[:, -1].clone()}
    if not train:
        return res
    d = s["dout"].float()
    d = torch.cat([d[:, :-1], d[:, -1:] + s["dh"][:, None]], 1)
    ahead = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _scan(ahead.flip(1), d.flip(1)).flip(1)
    first = torch.zeros_like(h[:, :1]) if s["h0"] is None else s["h0"][:, None]
    res["dg"] = a * torch.cat([first, h[:, :-1]], 1) * dh
    res["dx"] = (dh if b is None else b * dh).to(s["x"].dtype)
    if b is not None:
        res["db"] = (x * dh).to(s["b"].dtype)
    if s["h0"] is not None:
        res["dh0"] = a[:, 0] * dh[:, 0]
    return res


def _plain_step(s):
    h = torch.exp(s["g"].float()) * s["h0"] + s["b"].float() * s["x"].float()
    return {"out": h.to(s["x"].dtype), "state": h}


def _plain_norm(s, train):
    h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["r"].dtype)
    f, w = h.float(), s["w"].float()
    rstd = 1.0 / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS)
    if not train:
        t = f * w
        m = t.abs().amax(-1, keepdim=True)
        y = torch.round(t * (127.0 / m)) * (m * rstd / 127.0)
        return {"y": y.to(s["x"].dtype), "h": h}
    n, dy = f * rstd, s["dy"].float()
    dn = dy * w
    dx = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    res = {"y": (n * w).to(s["x"].dtype), "dw": (dy * n).sum(0)}
    if s["r"] is not None:
        dx = dx + s["dh"].float()
        res.update(h=h, dr=dx.to(s["r"].dtype))
    return {**res, "dx": dx.to(s["x"].dtype)}


def _plain_product(s):
    y = (s["x"].float() @ s["w"].float().t()) * s["sx"][:, None] * s["sw"]
    return (y if s["bias"] is None else y + s["bias"]).to(_DT[s["case"]["dtype"]])


def _plain(s):
    kind = s["case"]["kind"]
    with torch.no_grad():
        if kind == "step":
            return _plain_step(s)
        if kind in ("scan", "scan_train"):
            return _plain_scan(s, kind == "scan_train")
        if kind in ("norm8", "norm_train"):
            return _plain_norm(s, kind == "norm_train")
        return _plain_product(s)


# ---------------------------------------------------------------- the package's operators

def _own(s):
    gp, kind = _gp(), s["case"]["kind"]
    if kind == "step":
        out, state = gp.gdn2_gated_scan_step(s["x"], s["g"], s["b"], state=s["h0"])
        return {"out": out, "state": state}
    if kind in ("scan", "scan_train"):
        out, h_final = gp.gdn2_gated_scan(s["x"], s["g"], s["b"], h0=s["h0"])
        res = {"out": out, "h_final": h_final}
        if kind == "scan_train":
            names = [n for n in ("x", "g", "b", "h0") if s[n] is not None]
            grads = torch.autograd.grad((out, h_final), [s[n] for n in names],
                                        (s["dout"], s["dh"]))
            res.update(("d" + n, t) for n, t in zip(names, grads))
        return res
    if kind == "norm8":
        q, scale, h = gp.gdn2_rms_norm_int8(s["x"], s["w"], residual=s["r"], eps=EPS)
        return {"y": gp.gdn2_dequantize_int8(q, scale, dtype=s["x"].dtype), "h": h}
    if kind == "norm_train":
        y, h = gp.gdn2_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
        if s["r"] is None:   # h is x itself
            dx, dw = torch.autograd.grad(y, [s["x"], s["w"]], s["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        dx, dw, dr = torch.autograd.grad((y, h), [s["x"], s["w"], s["r"]], (s["dy"], s["dh"]))
        return {"y": y, "h": h, "dx": dx, "dw": dw, "dr": dr}
    return gp.gdn2_int8_matmul(s["x"], s["sx"], s["w"], s["sw"], bias=s["bias"],
                               out_dtype=_DT[s["case"]["dtype"]])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each input read once, each output written once; the operations of the definition."""
    e = 2 if case["dtype"] == "bf16" else 4
    kind = case["kind"]
    if kind == "step":
        n = case["B"] * case["C"]
        return {"bytes": n * (2 * e + 4 + 4 + e + 4), "flops": 4 * n}
    if kind in ("scan", "scan_train"):
        n, c = case["B"] * case["T"] * case["C"], case["B"] * case["C"] * 4
        gate = e if case["gate"] else 0
        bytes_, flops = n * (e + 4 + gate + e) + c * (2 if case["h0"] else 1), 4 * n
        if kind == "scan_train":   # dout and the inputs again; dx, dg, db
            bytes_ += n * (e + (e + 4 + gate) + (e + 4 + gate)) + c * (2 if case["h0"] else 1)
            flops += 8 * n
        return {"bytes": bytes_, "flops": flops}
    if kind in ("norm8", "norm_train"):
        n, r = case["M"] * case["C"], e if case["residual"] else 0
        if kind == "norm8":
            return {"bytes": n * (e + r + r + 1) + 4 * (case["M"] + case["C"]), "flops": 6 * n}
        # y (and h) written; then h, dy (and dh) read and one gradient of x and residual written
        return {"bytes": n * (e + r + r + e + 2 * e + r + e) + 8 * case["C"], "flops": 16 * n}
    M, K, N = case["M"], case["K"], case["N"]
    return {"bytes": M * K + N * K + 4 * (M + N) + e * M * N, "flops": 2 * M * N * K}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_scan(s, train):
    x, a = s["x"].double(), s["g"].double().exp()
    b = torch.ones((), device="cuda", dtype=torch.float64).expand_as(x) if s["b"] is None \
        else s["b"].double()
    T = x.shape[1]
    h = torch.zeros_like(x[:, 0]) if s["h0"] is None else s["h0"].double().clone()
    start, out = h.clone(), torch.empty_like(x)
    u = b * x
    for t in range(T):
        h = torch.addcmul(u[:, t], a[:, t], h)
        out[:, t] = h
    res = {"out": out, "h_final": h}
    if not train:
        return res
    dout, dh = s["dout"].double(), torch.empty_like(x)
    e = s["dh"].double()
    for t in reversed(range(T)):
        d = dout[:, t] + e
        dh[:, t] = d
        e = a[:, t] * d
    res["dx"] = b * dh
    if s["b"] is not None:
        res["db"] = x * dh
    if s["h0"] is not None:
        res["dh0"] = e
    before = torch.roll(out, 1, 1)
    before[:, 0] = start
    res["dg"] = dh * before * a
    return res


def _exact_norm(s, train):
    if s["r"] is None:
        h = s["x"]
    else:   # the sum of two floats is exact in 64 bits: one rounding to the residual's type
        h = (s["x"].double() + s["r"].double()).to(s["r"].dtype)
    v, w = h.double(), s["w"].double()
    size = torch.sqrt(v.square().mean(-1) + EPS)[:, None]
    if not train:
        t = v * w
        top = t.abs().max(-1, keepdim=True).values
        return {"y": torch.round(127.0 * t / top) * top / 127.0 / size, "h": v}
    C = v.shape[1]
    dy = s["dy"].double()
    through = (dy * w * v).sum(-1, keepdim=True)
    dx = dy * w / size - v * through / (C * size ** 3)
    res = {"y": v / size * w, "dw": (dy * v / size).sum(0)}
    if s["r"] is not None:
        dx += s["dh"].double()
        res.update(h=v, dr=dx)
    return {**res, "dx": dx}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "step":
            h = s["g"].double().exp() * s["h0"].double() + s["b"].double() * s["x"].double()
            return {"out": h, "state": h}
        if kind in ("scan", "scan_train"):
            return _exact_scan(s, kind == "scan_train")
        if kind in ("norm8", "norm_train"):
            return _exact_norm(s, kind == "norm_train")
        y = s["sx"].double()[:, None] * s["sw"].double() * (s["x"].double()
                                                           @ s["w"].double().t())
        return y if s["bias"] is None else y + s["bias"].double()
