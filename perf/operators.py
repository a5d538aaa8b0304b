"""Performance cases of the layers that read a grid's features: the matrix
product with bias, activation and residual in its epilogue (`ash.linear`) and
the root-mean-square norm with the residual's addition and an output in 8 bits
(`ash.rms_norm`), as a decoder of interpolated features chains them.

Kinds of work (the "op" of a case):

  linear    activation(x W^T + b) + residual, without gradients
  train     the same with the gradients of every operand
  second    the gradient with respect to the features, as an eikonal loss takes
            it, and its own gradients
  linear8   the product of 8-bit rows with 8-bit weights, both with a scale a row
  norm      rms_norm(x + residual) * weight with the sum, and all gradients
  norm8     the same without gradients, rounded to 8 bits with a scale a row

`own` says whose work is measured: the package's operators, or the same
formulas written out in elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = torch.device("cuda")
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
EPS = 1e-6


def _ash():
    path = os.path.join(os.getcwd(), "torch-ash_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ash

    return ash


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one position through a layer of a served decoder: the latency of a call
        {"name": "linear_one_row", "op": "linear", "type": "bf16", "rows": 1, "k": 1024, "m": 1024,
         "act": "gelu", "scale": 1.0, "residual": True},
        # samples of a batch of rays into a sine network: 16 channels of the
        # grid and the position itself, an odd width
        {"name": "linear_samples", "op": "linear", "type": "fp32", "rows": 262_144, "k": 19, "m": 64,
         "act": "sine", "scale": 30.0, "residual": False},
        # a hidden layer of a surface decoder in training, the usual width
        {"name": "train_narrow", "op": "train", "type": "fp32", "rows": 524_288, "k": 64, "m": 64,
         "act": "softplus", "scale": 100.0, "residual": False},
        # odd sizes throughout: ragged batches, concatenated features
        {"name": "train_odd", "op": "train", "type": "fp16", "rows": 10_007, "k": 131, "m": 257,
         "act": "silu", "scale": 1.0, "residual": True},
        # the wide layers of a large decoder, a residual block
        {"name": "train_wide", "op": "train", "type": "bf16", "rows": 65_536, "k": 1024, "m": 1024,
         "act": "gelu", "scale": 1.0, "residual": True},
        # the eikonal share of a training step of a surface decoder
        {"name": "second_narrow", "op": "second", "type": "fp32", "rows": 131_072, "k": 64, "m": 64,
         "act": "softplus", "scale": 100.0, "residual": False},
        # a few positions of a served decoder with 8-bit weights
        {"name": "linear8_few_rows", "op": "linear8", "type": "bf16", "rows": 16, "k": 2048, "m": 2048,
         "act": "none", "scale": 1.0, "residual": True},
        # a volume of positions through a wide layer, exported in one go
        {"name": "linear8_large", "op": "linear8", "type": "bf16", "rows": 16_384, "k": 4096, "m": 4096,
         "act": "silu", "scale": 1.0, "residual": False},
        # a small batch of odd width in training: launches count
        {"name": "norm_small", "op": "norm", "type": "fp32", "rows": 777, "k": 67, "residual": True},
        # the norm before a wide residual block, in training
        {"name": "norm_wide", "op": "norm", "type": "bf16", "rows": 65_536, "k": 1024, "residual": True},
        # one position before an 8-bit layer
        {"name": "norm8_one_row", "op": "norm8", "type": "bf16", "rows": 1, "k": 1024, "residual": True},
        # an exported volume of positions before an 8-bit layer
        {"name": "norm8_volume", "op": "norm8", "type": "bf16", "rows": 262_144, "k": 256, "residual": True},
    ]


def draw(rng):
    """Rows from one to half a million, widths from three to four thousand, up
    to the cost of the largest listed case of the same kind."""
    def log_uniform(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["linear", "linear", "train", "train", "second", "linear8", "linear8", "norm", "norm8"])
    case = {"op": op, "type": rng.choice(["fp32", "bf16", "fp16"]), "rows": log_uniform(1, 524_288)}
    if op in ("norm", "norm8"):
        case["k"] = log_uniform(3, 4096)
        case["rows"] = max(1, min(case["rows"], 65_536 * 1024 // case["k"]))
        case["residual"] = rng.random() < 0.7
        return case
    case["k"], case["m"] = log_uniform(3, 4096), log_uniform(1, 4096)
    if rng.random() < 0.5:   # whole multiples, as most networks have them
        case["k"], case["m"] = -(-case["k"] // 16) * 16, -(-case["m"] // 16) * 16
    products = {"linear": 65_536 * 1024 * 1024, "linear8": 16_384 * 4096 * 4096,
                "train": 16_384 * 1024 * 1024, "second": 4_096 * 1024 * 1024}[op]
    case["rows"] = max(1, min(case["rows"], products // (case["k"] * case["m"]),
                              524_288 * 128 // (case["k"] + case["m"])))
    case["act"] = rng.choice(["none", "relu", "silu", "gelu", "softplus", "sine"])
    if op == "second" and case["act"] in ("none", "relu"):
        case["act"] = "silu"
    if case["act"] == "softplus":
        case["scale"] = rng.choice([1.0, 10.0, 100.0])
    else:
        case["scale"] = rng.choice([1.0, 30.0]) if case["act"] == "sine" else 1.0
    case["residual"] = op != "second" and rng.random() < 0.5
    return case


# ----------------------------------------------------------------- the inputs
def prepare(case, seed):
    """Features of unit size, as a norm or a trained grid leaves them; weights
    at the scale that keeps them so (of a sine network: such that the argument
    of the sine does); gradients of unit size."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, dtype, n, k = case["op"], TYPES[case["type"]], case["rows"], case["k"]
    learns = op in ("train", "second", "norm")

    def normal(*shape, size=1.0):
        return torch.empty(shape, device=DEV).normal_(0.0, size, generator=g)

    def leaf(t):
        t = t.to(dtype)
        return t.requires_grad_() if learns else t

    s = {"case": case}
    if op in ("norm", "norm8"):
        s["x"] = leaf(normal(n, k) * (1.0 + normal(n, 1, size=0.3).abs()))
        s["w"] = leaf(1.0 + normal(k, size=0.1))
        s["residual"] = leaf(normal(n, k)) if case["residual"] else None
        if learns:
            s["gy"] = normal(n, k).to(dtype)
            s["gs"] = normal(n, k).to(dtype) if case["residual"] else None
        return s
    m = case["m"]
    size = 1.0 / math.sqrt(k)
    if case["act"] == "sine":
        size *= math.sqrt(2.0) / case["scale"]
    x, w = normal(n, k), normal(m, k, size=size)
    if op == "linear8":
        s["x"], s["x_scale"] = _rounded_rows(x)
        s["w"], s["w_scale"] = _rounded_rows(w)
    else:
        s["x"], s["w"] = leaf(x), leaf(w)
    s["b"] = leaf(normal(m, size=size))
    s["residual"] = leaf(normal(n, m)) if case["residual"] else None
    if learns:
        s["gy"] = normal(n, m).to(dtype)
    if op == "second":
        s["gy"].requires_grad_()
        s["u"] = normal(n, k).to(dtype)
    return s


def _rounded_rows(v):
    """(e4m3 values, scale a row) such that values * scale stand for `v`."""
    scale = v.abs().amax(1) / E4M3_MAX
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (v / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3), scale


# ------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ash, c = _ash(), s["case"]
    op = c["op"]
    if op == "norm":
        grad = torch.autograd.grad
        if s["residual"] is None:
            y = ash.rms_norm(s["x"], s["w"], eps=EPS)
            gx, gw = grad(y, [s["x"], s["w"]], s["gy"])
            return {"y": y, "gx": gx, "gw": gw}
        y, total = ash.rms_norm(s["x"], s["w"], residual=s["residual"], eps=EPS)
        gx, gr, gw = grad([y, total], [s["x"], s["residual"], s["w"]], [s["gy"], s["gs"]])
        return {"y": y, "sum": total, "gx": gx, "gr": gr, "gw": gw}
    if op == "norm8":
        if s["residual"] is None:
            y = ash.rms_norm(s["x"], s["w"], eps=EPS, quantize=True)
            return {"y": y.data, "scale": y.scales}
        y, total = ash.rms_norm(s["x"], s["w"], residual=s["residual"], eps=EPS, quantize=True)
        return {"y": y.data, "scale": y.scales, "sum": total}
    if op == "linear8":
        return ash.linear(ash.QuantizedRows(s["x"], s["x_scale"]), ash.QuantizedRows(s["w"], s["w_scale"]),
                          s["b"], activation=c["act"], scale=c["scale"], residual=s["residual"])
    y = ash.linear(s["x"], s["w"], s["b"], activation=c["act"], scale=c["scale"], residual=s["residual"])
    if op == "linear":
        return y
    grad = torch.autograd.grad
    if op == "train":
        leaves = [t for t in (s["x"], s["w"], s["b"], s["residual"]) if t is not None]
        return {"y": y, "grads": grad(y, leaves, s["gy"])}
    gx, = grad(y, s["x"], s["gy"], create_graph=True)
    return {"y": y, "gx": gx, "grads": grad(gx, [s["gy"], s["x"], s["w"], s["b"]], s["u"])}


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    op, dtype = c["op"], TYPES[c["type"]]
    x = s["x"].float()
    if op in ("norm", "norm8"):
        if s["residual"] is not None:
            x = x + s["residual"].float()
        w = s["w"].float()
        r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
        y = x * r * w
        if op == "norm8":
            values, scale = _rounded_rows(y)
            out = {"y": values, "scale": scale}
            if s["residual"] is not None:
                out["sum"] = x.to(dtype)
            return out
        gy = s["gy"].float()
        t = gy * w
        gx = r * t - x * (r * r * r * (t * x).mean(1, keepdim=True))
        out = {"y": y.to(dtype), "gw": (gy * x * r).sum(0).to(dtype)}
        if s["residual"] is not None:
            gx = (gx + s["gs"].float()).to(dtype)
            return {**out, "sum": x.to(dtype), "gx": gx, "gr": gx}
        return {**out, "gx": gx.to(dtype)}
    w, b = s["w"].float(), s["b"].float()
    z = x @ w.t()
    if op == "linear8":
        z = z * s["x_scale"][:, None] * s["w_scale"]
    z = z + b
    y = _act(z, c)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(dtype)
    if op in ("linear", "linear8"):
        return y
    gy = s["gy"].float()
    d = _act_1(z, c)
    gz = gy * d
    gx = gz @ w
    if op == "train":
        grads = [gx.to(dtype), (gz.t() @ x).to(dtype), gz.sum(0).to(dtype)]
        if s["residual"] is not None:
            grads.append(s["gy"])
        return {"y": y, "grads": grads}
    # of <u, gx>: t is its derivative by gz, q by z
    u = s["u"].float()
    t = u @ w.t()
    q = t * gy * _act_2(z, c)
    grads = [t * d, q @ w, gz.t() @ u + q.t() @ x, q.sum(0)]
    return {"y": y, "gx": gx.to(dtype), "grads": [v.to(dtype) for v in grads]}


def _act(z, c):
    a = c["scale"]
    if c["act"] == "relu":
        return z.clamp(min=0)
    if c["act"] == "silu":
        return z * torch.sigmoid(z)
    if c["act"] == "gelu":
        return z * (0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))))
    if c["act"] == "softplus":   # log(1 + exp(a z)) / a, without overflow
        return (z.clamp(min=0) * a + torch.log1p(torch.exp(-(z * a).abs()))) / a
    return torch.sin(a * z) if c["act"] == "sine" else z


def _act_1(z, c):
    a = c["scale"]
    if c["act"] == "relu":
        return (z > 0).to(z.dtype)
    if c["act"] == "silu":
        p = torch.sigmoid(z)
        return p * (1.0 + z * (1.0 - p))
    if c["act"] == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if c["act"] == "softplus":
        return torch.sigmoid(a * z)
    return a * torch.cos(a * z) if c["act"] == "sine" else torch.ones_like(z)


def _act_2(z, c):
    a = c["scale"]
    if c["act"] == "silu":
        p = torch.sigmoid(z)
        return p * (1.0 - p) * (2.0 + z * (1.0 - 2.0 * p))
    if c["act"] == "gelu":
        return (2.0 - z * z) * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if c["act"] == "softplus":
        return a * torch.sigmoid(a * z) * torch.sigmoid(-a * z)
    return -a * a * torch.sin(a * z)


# ------------------------------------------------------------------- the work
def work(case):
    """Every operand read once, every output written once; a product is two
    operations a term, first order has three of them, second order seven (its
    own forward and gradient among them)."""
    op, n, k = case["op"], case["rows"], case["k"]
    e = 4 if case["type"] == "fp32" else 2
    if op == "norm":     # forward: x (residual) w -> y (sum); backward: gy (gs) sum w -> gx gw
        planes = 3 if not case["residual"] else 4
        return {"bytes": e * (n * k * (planes + planes) + 3 * k), "flops": 20 * n * k}
    if op == "norm8":
        planes = 1 if not case["residual"] else 3
        return {"bytes": n * k * (e * planes + 1) + e * k + 4 * n, "flops": 10 * n * k}
    m, res = case["m"], n * case["m"] * bool(case["residual"])
    if op == "linear8":
        return {"bytes": n * k + m * k + 4 * (n + m) + e * (m + n * m + res), "flops": 2 * n * k * m}
    forward = n * k + m * k + m + n * m + res
    if op == "linear":
        return {"bytes": e * forward, "flops": 2 * n * k * m}
    first = n * m + n * k + m * k + m          # gy -> gx gw gb
    if op == "train":
        return {"bytes": e * (forward + first), "flops": 6 * n * k * m}
    second = 2 * (n * k) + n * m + m * k + m   # u -> ggy gx gw gb
    return {"bytes": e * (forward + n * m + n * k + second), "flops": 14 * n * k * m}


# -------------------------------------------------- the definition in 64 bits
@torch.no_grad()
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    for name, v in s.items():
        if torch.is_tensor(v):
            s[name] = v.detach().double()
    if op in ("norm", "norm8"):
        v = s["x"] if s["residual"] is None else s["x"] + s["residual"]
        inverse = (v.square().sum(1) / v.shape[1] + EPS) ** -0.5
        unit = v * inverse[:, None]
        y = unit * s["w"][None, :]
        if op == "norm8":
            scale = y.abs().max(1).values / E4M3_MAX
            out = {"y": y / scale[:, None], "scale": scale}
        else:
            up = s["gy"] * s["w"][None, :]
            along = (up * unit).sum(1) / v.shape[1]
            gx = (up - unit * along[:, None]) * inverse[:, None]
            out = {"y": y, "gw": (s["gy"] * unit).sum(0)}
            if s["residual"] is not None:
                gx = out["gr"] = gx + s["gs"]
            out["gx"] = gx
        if s["residual"] is not None:
            out["sum"] = v
        return out
    x, w = s["x"], s["w"]
    if op == "linear8":
        x, w = x * s["x_scale"][:, None], w * s["w_scale"][:, None]
    z = torch.addmm(s["b"], x, w.T)
    f, f1, f2 = _exact_act(z, case)
    y = f if s["residual"] is None else f + s["residual"]
    if op in ("linear", "linear8"):
        return y
    gz = s["gy"] * f1
    gx = gz.mm(w)
    if op == "train":
        grads = [gx, gz.T.mm(x), gz.sum(0)]
        return {"y": y, "grads": grads + ([s["gy"]] if s["residual"] is not None else [])}
    t = s["u"].mm(w.T)
    q = t * s["gy"] * f2
    return {"y": y, "gx": gx, "grads": [t * f1, q.mm(w), q.T.mm(x) + gz.T.mm(s["u"]), q.sum(0)]}


def _exact_act(z, case):
    """The activation and its first two derivatives."""
    a, name = case["scale"], case["act"]
    one, zero = torch.ones_like(z), torch.zeros_like(z)
    if name == "relu":
        return torch.maximum(z, zero), torch.where(z > 0, one, zero), zero
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        dp = p * (1.0 - p)
        return z * p, p + z * dp, 2.0 * dp + z * dp * (1.0 - 2.0 * p)
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / 2.0**0.5)
        pdf = torch.exp(-z.square() / 2.0) / (2.0 * math.pi) ** 0.5
        return z * cdf, cdf + z * pdf, 2.0 * pdf - z.square() * pdf
    if name == "softplus":
        p = 1.0 / (1.0 + torch.exp(-a * z))
        return torch.logaddexp(a * z, zero) / a, p, a * p * (1.0 - p)
    if name == "sine":
        return (a * z).sin(), a * (a * z).cos(), -(a**2) * (a * z).sin()
    return z, one, zero
