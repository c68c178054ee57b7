"""What is measured of the operators that run a transformer's feed-forward block on packed int4 weights: the
root-mean-square norm with the residual's addition (16-bit output, or e4m3 with scales), the matrix product over
pack-quantized int4 weights with bias, activation and residual, and the gated product of two such matrices; each with
its backward pass (the int4 weights are frozen, so gradients go to inputs, biases and norm gains).

`own` chooses the side: the plain form (elementary torch operations in fp32, one rounding at the end) or the
framework's kernels.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
F8_MAX = 448.0            # largest finite e4m3 value
AMAX_FLOOR = 1e-12        # a group whose largest magnitude is below this is scaled as if it were this

_ops = None


def _forge_ops():
    global _ops
    if _ops is None:
        path = os.path.join(os.getcwd(), "4bit-forge_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from forge import ops
        _ops = ops
    return _ops


def listed():
    return [
        # the norm in front of a decode step's feed-forward block, sixteen sequences, DeepSeek-V3 width
        {"name": "norm decode 16x7168", "op": "norm", "T": 16, "C": 7168, "dtype": "bf16", "residual": True, "group": 0},
        # a long prompt's norm whose output leaves in 8 bits with a scale per 128 channels
        {"name": "norm prompt e4m3 8192x7168", "op": "norm", "T": 8192, "C": 7168, "dtype": "bf16", "residual": True,
         "group": 128},
        # a norm's gain being tuned on a ragged calibration batch, Qwen3-30B-A3B width: forward and backward
        {"name": "norm train 5003x2048", "op": "norm_train", "T": 5003, "C": 2048, "dtype": "bf16", "residual": True},
        # one token through the down projection of a shared expert, added to the residual stream
        {"name": "down 1 token 2048-7168", "op": "linear", "T": 1, "C": 2048, "R": 7168, "gs": 128, "dtype": "bf16",
         "bias": False, "act": "none", "residual": True},
        # a decode batch of 24 sequences through a wide input projection
        {"name": "linear 24 tokens 7168-2048", "op": "linear", "T": 24, "C": 7168, "R": 2048, "gs": 128, "dtype": "bf16",
         "bias": True, "act": "none", "residual": False},
        # odd sizes, the smallest group, every part of the epilogue
        {"name": "linear odd 333x776-1001 gelu", "op": "linear", "T": 333, "C": 776, "R": 1001, "gs": 32, "dtype": "fp16",
         "bias": True, "act": "gelu", "residual": True},
        # a prompt through the down projection, added to the residual stream
        {"name": "down prompt 4096 2048-7168", "op": "linear", "T": 4096, "C": 2048, "R": 7168, "gs": 128, "dtype": "bf16",
         "bias": False, "act": "none", "residual": True},
        # tuning through a frozen projection: forward, gradients of the input and the bias
        {"name": "linear train 2048 2048-2048", "op": "linear_train", "T": 2048, "C": 2048, "R": 2048, "gs": 64,
         "dtype": "bf16", "act": "gelu"},
        # one token through gate and up of a shared expert (DeepSeek-V3)
        {"name": "gated 1 token 7168-2048", "op": "gated", "T": 1, "C": 7168, "R": 2048, "gs": 128, "dtype": "bf16",
         "act": "silu"},
        # a decode batch of 64 sequences through one Qwen3-30B-A3B expert
        {"name": "gated 64 tokens 2048-768", "op": "gated", "T": 64, "C": 2048, "R": 768, "gs": 128, "dtype": "fp16",
         "act": "silu"},
        # a long prompt through gate and up of a shared expert (DeepSeek-V3)
        {"name": "gated prompt 8192 7168-2048", "op": "gated", "T": 8192, "C": 7168, "R": 2048, "gs": 128, "dtype": "bf16",
         "act": "silu"},
        # a tuning step through the same: forward, gradient of the input
        {"name": "gated train 4096 7168-2048", "op": "gated_train", "T": 4096, "C": 7168, "R": 2048, "gs": 128,
         "dtype": "bf16", "act": "silu"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_train", "linear", "linear", "linear_train", "gated", "gated", "gated_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    T = _log_int(rng, 1, 8192)
    if op in ("norm", "norm_train"):
        case = {"op": op, "T": T, "C": _log_int(rng, 64, 8192), "dtype": dtype, "residual": rng.random() < 0.7}
        if op == "norm":
            case["group"] = rng.choice([0, 128])
        return case
    C, R = 8 * _log_int(rng, 8, 7168 // 8), _log_int(rng, 16, 7168)
    # a drawn case costs no more than the largest listed one: 2 matrices x 8192 x 7168 x 2048
    most = 2 * 8192 * 7168 * 2048
    per = C * R * {"linear": 1, "linear_train": 2, "gated": 2, "gated_train": 4}[op]
    T = max(1, min(T, most // per))
    case = {"op": op, "T": T, "C": C, "R": R, "gs": rng.choice([32, 64, 128, 128]), "dtype": dtype}
    if op == "linear":
        case.update(bias=rng.random() < 0.5, act=rng.choice(["none", "none", "relu", "silu", "gelu"]),
                    residual=rng.random() < 0.5)
    elif op == "linear_train":
        case.update(act=rng.choice(["relu", "silu", "gelu"]))
    else:
        case.update(act=rng.choice(["silu", "silu", "gelu"]))
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _activations(T, C, dt, g):
    """Hidden states: normal entries, per-channel spread of a trained network's activations."""
    dev = g.device
    ch = torch.exp(0.5 * torch.randn(C, generator=g, device=dev))
    return (torch.randn(T, C, generator=g, device=dev) * ch).to(dt)


def _int4_weight(R, C, gs, g):
    """A quantised matrix in the pack-quantized layout: eight codes of a row per int32 word, value (code - 8) * scale."""
    dev = g.device
    codes = (torch.randn(R, C, generator=g, device=dev) * 2.7 + 8.0).round_().clamp_(0, 15).to(torch.int32)
    shifts = torch.arange(0, 32, 4, device=dev, dtype=torch.int32)
    packed = (codes.view(R, C // 8, 8) << shifts).sum(-1, dtype=torch.int32)
    G = (C + gs - 1) // gs
    scales = (0.5 + torch.rand(R, G, generator=g, device=dev)) * (0.37 / math.sqrt(C))
    return packed.contiguous(), scales.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, T, C, op = DTYPES[case["dtype"]], case["T"], case["C"], case["op"]
    st = {"case": dict(case), "x": _activations(T, C, dt, g)}
    if op in ("norm", "norm_train"):
        st["weight"] = (1.0 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(dt)
        st["res"] = (4.0 * torch.randn(T, C, generator=g, device="cuda")).to(dt) if case["residual"] else None
        if op == "norm_train":
            st["dy"] = torch.randn(T, C, generator=g, device="cuda").to(dt)
            st["dres"] = torch.randn(T, C, generator=g, device="cuda").to(dt) if case["residual"] else None
        return st
    R, gs = case["R"], case["gs"]
    st["w"], st["s"] = _int4_weight(R, C, gs, g)
    if op.startswith("gated"):
        st["w2"], st["s2"] = _int4_weight(R, C, gs, g)
    if case.get("bias") or op == "linear_train":
        st["bias"] = (0.3 * torch.randn(R, generator=g, device="cuda")).to(dt)
    if case.get("residual"):
        st["res"] = (2.0 * torch.randn(T, R, generator=g, device="cuda")).to(dt)
    if op.endswith("train"):
        st["dy"] = torch.randn(T, R, generator=g, device="cuda").to(dt)
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _dense(packed, scales, gs, dtype=torch.float32):
    R, C = packed.shape[0], packed.shape[1] * 8
    shifts = torch.arange(0, 32, 4, device=packed.device, dtype=torch.int32)
    codes = ((packed.unsqueeze(-1) >> shifts) & 15).view(R, C).to(dtype) - 8
    return codes * scales.to(dtype).repeat_interleave(gs, dim=1)[:, :C]


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _dact(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


EPS = 1e-6


def _plain(st):
    c = st["case"]
    op, dt = c["op"], st["x"].dtype
    x = st["x"].float()
    if op in ("norm", "norm_train"):
        h = x if st["res"] is None else x + st["res"].float()
        w = st["weight"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * w
        r = h.to(dt)
        if op == "norm":
            if c["group"] == 0:
                out = {"y": y.to(dt)}
            else:
                T, C, gq = c["T"], c["C"], c["group"]
                pad = (-C) % gq
                yg = torch.cat([y, y.new_zeros(T, pad)], 1).view(T, -1, gq)
                scale = yg.abs().amax(2).clamp_min(AMAX_FLOOR) / F8_MAX
                q = (yg / scale.unsqueeze(2)).to(torch.float8_e4m3fn)
                out = {"q": q.view(T, C + pad)[:, :C].contiguous(), "scales": scale}
            if st["res"] is not None:
                out["residual"] = r
            return out
        rf, dy = r.float(), st["dy"].float()
        rstd = torch.rsqrt((rf * rf).mean(1, keepdim=True) + EPS)
        xh = rf * rstd
        dyw = dy * w
        dx = rstd * (dyw - xh * (dyw * xh).mean(1, keepdim=True))
        if st["dres"] is not None:
            dx = dx + st["dres"].float()
        return {"y": y.to(dt), "dx": dx.to(dt), "dweight": (dy * xh).sum(0).to(dt)}
    W = _dense(st["w"], st["s"], c["gs"])
    z = x @ W.t()
    if op in ("linear", "linear_train"):
        if "bias" in st:
            z = z + st["bias"].float()
        y = _act(z, c["act"])
        if op == "linear":
            if "res" in st:
                y = y + st["res"].float()
            return {"y": y.to(dt)}
        dz = st["dy"].float() * _dact(z.to(dt).float(), c["act"])
        return {"y": y.to(dt), "dx": (dz @ W).to(dt), "dbias": dz.sum(0).to(dt)}
    U = _dense(st["w2"], st["s2"], c["gs"])
    u = x @ U.t()
    h = (_act(z, c["act"]) * u).to(dt)
    if op == "gated":
        return {"y": h}
    zr, ur, dy = z.to(dt).float(), u.to(dt).float(), st["dy"].float()
    dx = (dy * ur * _dact(zr, c["act"])) @ W + (dy * _act(zr, c["act"])) @ U
    return {"y": h, "dx": dx.to(dt)}


# ---- the framework's operators ----------------------------------------------------------------------------------------

def _kernels(st):
    ops, c = _forge_ops(), st["case"]
    op, x = c["op"], st["x"]
    if op == "norm":
        if c["group"] == 0:
            if st["res"] is None:
                return {"y": ops.rmsnorm(x, st["weight"], EPS)}
            y, r = ops.rmsnorm(x, st["weight"], EPS, residual=st["res"])
            return {"y": y, "residual": r}
        if st["res"] is None:
            q, s = ops.rmsnorm(x, st["weight"], EPS, quant_group=c["group"])
            return {"q": q, "scales": s}
        q, s, r = ops.rmsnorm(x, st["weight"], EPS, residual=st["res"], quant_group=c["group"])
        return {"q": q, "scales": s, "residual": r}
    if op == "norm_train":
        y, r = (ops.rmsnorm(x, st["weight"], EPS), x) if st["res"] is None else \
            ops.rmsnorm(x, st["weight"], EPS, residual=st["res"])
        dx, dw = ops.rmsnorm_backward(st["dy"], r, st["weight"], EPS, dresidual=st["dres"])
        return {"y": y, "dx": dx, "dweight": dw}
    if op == "linear":
        return {"y": ops.int4_linear(x, st["w"], st["s"], c["gs"], bias=st.get("bias"), act=c["act"],
                                     residual=st.get("res"))}
    if op == "linear_train":
        y, z = ops.int4_linear(x, st["w"], st["s"], c["gs"], bias=st["bias"], act=c["act"], want_preact=True)
        dx, db = ops.int4_linear_backward(st["dy"], st["w"], st["s"], c["gs"], preact=z, act=c["act"], want_dbias=True)
        return {"y": y, "dx": dx, "dbias": db}
    if op == "gated":
        return {"y": ops.int4_gated(x, st["w"], st["s"], st["w2"], st["s2"], c["gs"], act=c["act"])}
    h, g, u = ops.int4_gated(x, st["w"], st["s"], st["w2"], st["s2"], c["gs"], act=c["act"], want_preact=True)
    dx = ops.int4_gated_backward(st["dy"], g, u, st["w"], st["s"], st["w2"], st["s2"], c["gs"], act=c["act"])
    return {"y": h, "dx": dx}


def run(state):
    return _kernels(state) if own else _plain(state)


def work(case):
    """Bytes: every input once, every output once.  Flops: 2 per multiply-add of the products; ~8 per element of a norm.
    The saved pre-activations of a training step are an intermediate and not counted."""
    T, C, op = case["T"], case["C"], case["op"]
    if op in ("norm", "norm_train"):
        res = 2 if case["residual"] else 0                        # read the branch, write the stream
        n = T * C
        if op == "norm":
            out = n * (1 if case["group"] else 2) + (4 * T * -(-C // 128) if case["group"] else 0)
            return {"bytes": 2 * n + 2 * n * res + out + 2 * C, "flops": 6 * n}
        # forward x (+ branch) in, y out; backward dy (+ its residual gradient) in, dx out
        return {"bytes": 2 * n * (4 + res) + 2 * C + 2 * C, "flops": 18 * n}
    R, gs = case["R"], case["gs"]
    mats = 2 if op.startswith("gated") else 1
    weights = mats * (R * C // 2 + 4 * R * -(-C // gs))
    b = weights + 2 * T * C + 2 * T * R
    f = 2 * T * C * R * mats
    if case.get("bias") or op == "linear_train":
        b += 2 * R
    if case.get("residual"):
        b += 2 * T * R
    if op.endswith("train"):
        b += 2 * T * R + 2 * T * C + (2 * R if op == "linear_train" else 0)
        f *= 2
    return {"bytes": b, "flops": f}


# ---- 64-bit values, from the definitions -------------------------------------------------------------------------------

def _sigma(z):
    return torch.sigmoid(z)


def _phi64(z, act):
    """(activation, its derivative)"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.relu(z), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if act == "silu":
        s = _sigma(z)
        return z * s, s + z * s * (1.0 - s)
    cdf = torch.special.ndtr(z)
    pdf = torch.exp(-z * z / 2.0) * (1.0 / math.sqrt(2.0 * math.pi))
    return z * cdf, cdf + z * pdf


def _weights64(packed, scales, gs):
    R, words = packed.shape
    W = torch.empty(R, words, 8, dtype=torch.float64, device=packed.device)
    for i in range(8):
        W[:, :, i] = torch.bitwise_and(torch.bitwise_right_shift(packed, 4 * i), 15).double().sub_(8.0)
    W = W.view(R, words * 8)
    for j in range(scales.shape[1]):
        W[:, j * gs:(j + 1) * gs] *= scales[:, j:j + 1].double()
    return W


def exact(case, seed):
    st = prepare(case, seed)
    op, x = case["op"], st["x"].double()
    if op in ("norm", "norm_train"):
        h = x if st["res"] is None else torch.add(x, st["res"].double())
        gain = st["weight"].double()
        inv = 1.0 / torch.sqrt(h.square().mean(dim=1) + EPS)
        y = torch.einsum("tc,t,c->tc", h, inv, gain)
        if op == "norm":
            out = {"y": y}
            if case["group"]:
                T, C, n = case["T"], case["C"], case["group"]
                G = -(-C // n)
                q, sc = torch.empty_like(y), torch.empty(T, G, dtype=torch.float64, device=y.device)
                for j in range(G):
                    part = y[:, j * n:(j + 1) * n]
                    sc[:, j] = torch.clamp(part.abs().max(dim=1).values, min=AMAX_FLOOR) / F8_MAX
                    q[:, j * n:(j + 1) * n] = part / sc[:, j:j + 1]
                out = {"q": q, "scales": sc}
            if st["res"] is not None:
                out["residual"] = h
            return out
        # the backward pass is taken at the stored stream, which the forward rounds to its type
        r = h.to(st["x"].dtype).double()
        inv = 1.0 / torch.sqrt(r.square().mean(dim=1, keepdim=True) + EPS)
        n = r * inv
        up = st["dy"].double()
        t = up * gain
        dx = inv * t - n * inv * (t * n).sum(dim=1, keepdim=True) / case["C"]
        if st["dres"] is not None:
            dx = dx + st["dres"].double()
        return {"y": y, "dx": dx, "dweight": torch.einsum("tc,tc->c", up, n)}
    W = _weights64(st["w"], st["s"], case["gs"])
    z = torch.matmul(x, W.transpose(0, 1))
    if op in ("linear", "linear_train"):
        if "bias" in st:
            z = z + st["bias"].double()
        y, _ = _phi64(z, case["act"])
        if op == "linear":
            return {"y": y + st["res"].double() if "res" in st else y}
        # the backward pass is taken at the stored pre-activation, which the forward rounds to its type
        _, d = _phi64(z.to(st["x"].dtype).double(), case["act"])
        dz = st["dy"].double() * d
        return {"y": y, "dx": torch.matmul(dz, W), "dbias": dz.sum(dim=0)}
    U = _weights64(st["w2"], st["s2"], case["gs"])
    u = torch.matmul(x, U.transpose(0, 1))
    a, _ = _phi64(z, case["act"])
    if op == "gated":
        return {"y": a * u}
    dt = st["x"].dtype
    ar, dr = _phi64(z.to(dt).double(), case["act"])
    dy = st["dy"].double()
    dx = torch.matmul(dy * u.to(dt).double() * dr, W) + torch.matmul(dy * ar, U)
    return {"y": a * u, "dx": dx}
