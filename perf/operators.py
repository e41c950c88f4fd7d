"""The dense operators of residual blocks over node or token features, as measurable cases: the norm with the residual's addition (training, and
with an output in 8 bits for serving), the product with bias, activation and residual in its epilogue (training, a few rows, operands in 8
bits), and the orthogonalised update of weight matrices.

`run` computes them in elementary operations in 32 bits where `own` is false, and calls the package's operators where it is true."""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EIGHT = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def listed():
    return [
        # the norm of a citation graph's hidden features in a training step: launches and host work count
        dict(name="norm_train_cora", kind="norm", rows=2708, cols=128, type="fp32", residual=True),
        # a training step over a long batch of tokens, or over wide features of many nodes
        dict(name="norm_train_tokens", kind="norm", rows=16384, cols=4096, type="bf16", residual=True),
        # one token of a served model
        dict(name="norm_q8_token", kind="norm_q8", rows=1, cols=4096, type="bf16", eight="int8", residual=True),
        # inference over all nodes of the largest input graph, 602 features: rows that start at odd multiples of four bytes
        dict(name="norm_q8_reddit", kind="norm_q8", rows=232965, cols=602, type="fp16", eight="e4m3", residual=True),
        # a layer over a citation graph's nodes, in the type that the package's drivers train in
        dict(name="linear_train_arxiv", kind="linear", rows=169343, k=128, n=256, type="fp32", activation="gelu", bias=True, residual=True, grad=True),
        # the widening product of a block over a batch of tokens
        dict(name="linear_train_tokens", kind="linear", rows=8192, k=4096, n=8192, type="bf16", activation="silu", bias=True, residual=False, grad=True),
        # odd sizes on every side: rows of 16-bit values that start anywhere
        dict(name="linear_train_odd", kind="linear", rows=5003, k=602, n=1433, type="fp16", activation="relu", bias=True, residual=True, grad=True),
        # one token of a served model
        dict(name="linear_token", kind="linear", rows=1, k=4096, n=8192, type="bf16", activation="gelu", bias=True, residual=True, grad=False),
        # sixteen sequences decoded together, weights in 8 bits
        dict(name="q8_decode", kind="linear_q8", rows=16, k=8192, n=4096, type="bf16", eight="int8", activation=None, bias=True, residual=True),
        # a long prompt, weights in 8 bits
        dict(name="q8_prompt", kind="linear_q8", rows=8192, k=4096, n=8192, type="bf16", eight="e4m3", activation="silu", bias=True, residual=False),
        # the update of four of the drivers' hidden layers
        dict(name="orth_layers", kind="orth", batch=4, m=256, n=128, type="fp32"),
        # the update of one wide weight matrix
        dict(name="orth_wide", kind="orth", batch=1, m=2048, n=8192, type="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: as often a multiple of 64 (or of 8) as an odd one."""
    v = _log(rng, lo, hi)
    unit = rng.choice([64, 8, 1])
    return max(lo, v // unit * unit)


def draw(rng):
    """One more case: sizes spread over their logarithm and cut so that none costs more than the largest listed one of its kind."""
    kind = rng.choice(["norm", "norm_q8", "linear", "serve", "linear_q8", "orth"])
    kept = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if kind in ("norm", "norm_q8"):
        cols = _size(rng, 16, 8192)
        rows = min(_log(rng, 1, 240000), (1 << 26) // cols)
        c = dict(kind=kind, rows=rows, cols=cols, type=kept, residual=rng.random() < 0.7)
        if kind == "norm_q8":
            c.update(eight=rng.choice(sorted(EIGHT)), type=rng.choice(["bf16", "fp16"]))
        return c
    activation = rng.choice([None, "relu", "gelu", "silu"])
    if kind == "orth":
        m, n = _size(rng, 16, 4096), _size(rng, 16, 8192)
        small, wide = min(m, n), max(m, n)
        one = 4 * small * small * wide + 2 * small ** 3
        batch = max(1, min(_log(rng, 1, 12), int(1.5e11 // one)))
        return dict(kind="orth", batch=batch, m=m, n=n, type=kept)
    k, n = _size(rng, 16, 8192), _size(rng, 16, 8192)
    most = max(1, int(2.7e11 // (k * n)))
    if kind == "linear":
        return dict(kind="linear", rows=min(_log(rng, 16, 170000), most // (2 if kept == "fp32" else 1), (1 << 27) // max(k, n)), k=k, n=n, type=kept, activation=activation,
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5, grad=True)
    if kind == "serve":
        return dict(kind="linear", rows=_log(rng, 1, 512), k=k, n=n, type=kept, activation=activation, bias=rng.random() < 0.7,
                    residual=rng.random() < 0.5, grad=False)
    return dict(kind="linear_q8", rows=min(_log(rng, 1, 8192), most), k=k, n=n, type=rng.choice(["bf16", "fp16"]), eight=rng.choice(sorted(EIGHT)),
                activation=activation, bias=rng.random() < 0.7, residual=rng.random() < 0.5)


def _eight(v, kind):
    """Rows of v in 8 bits and a scale for each, as a program lays out its weights once."""
    dtype, top = EIGHT[kind]
    a = v.abs().amax(-1)
    q = v * torch.where(a > 0, top / a, 0).unsqueeze(-1)
    return (torch.round(q) if kind == "int8" else q).to(dtype), a / top


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, std, generator=g).to(t)

    s = {"case": dict(case)}
    kind = case["kind"]
    if kind in ("norm", "norm_q8"):
        rows, cols = case["rows"], case["cols"]
        # features of which a few are larger, as in trained models
        s["x"] = normal(rows, cols) * torch.exp(normal(cols, std=0.5))
        s["weight"] = normal(cols, std=0.2, mean=1.0)
        s["residual"] = normal(rows, cols) if case["residual"] else None
        if kind == "norm":
            s["gy"], s["gh"] = normal(rows, cols, std=0.1), normal(rows, cols, std=0.1)
            for name in ("x", "weight", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = normal(rows, k)
        s["weight"] = normal(n, k, std=k ** -0.5)
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        s["residual"] = normal(rows, n) if case["residual"] else None
        if case["grad"]:
            s["gy"] = normal(rows, n, std=1.0 / 64)
            for name in ("x", "weight", "bias", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif kind == "linear_q8":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["q"], s["scale"] = _eight(normal(rows, k).float(), case["eight"])
        s["weight_q"], s["weight_scale"] = _eight(normal(n, k, std=k ** -0.5).float(), case["eight"])
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        s["residual"] = normal(rows, n) if case["residual"] else None
    else:
        batch, m, n = case["batch"], case["m"], case["n"]
        # a momentum of gradients: a few strong directions over noise
        rank = max(1, min(m, n) // 8)
        left, right = normal(batch, m, rank).float(), normal(batch, rank, n).float()
        s["g"] = (torch.matmul(left, right) * rank ** -0.5 + 0.5 * normal(batch, m, n).float()).to(t)
    return s


def _act(z, name):
    if name is None:
        return z
    if name == "relu":
        return torch.where(z > 0, z, 0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _wide(t):
    return None if t is None else t.detach().float()


def _plain_norm(s, case):
    t = s["x"].dtype
    x, w, r = _wide(s["x"]), _wide(s["weight"]), _wide(s["residual"])
    h = x if r is None else x + r
    scale = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    y = h * scale * w
    out = {} if r is None else {"h": h.to(t)}
    if case["kind"] == "norm_q8":
        _, top = EIGHT[case["eight"]]
        a = y.abs().amax(-1, keepdim=True)
        q = y * torch.where(a > 0, top / a, 0)
        q = torch.round(q) if case["eight"] == "int8" else q.to(torch.float8_e4m3fn)
        out["scale"] = (a / top).squeeze(-1)
        out["values"] = (q.float() * (a / top)).to(t)
        return out
    out["y"] = y.to(t)
    gy = _wide(s["gy"])
    g = gy * w
    dx = scale * g - h * (scale ** 3 * (g * h).mean(-1, keepdim=True))
    if r is not None:
        dx = dx + _wide(s["gh"])
    out["dx"] = dx.to(t)
    out["dw"] = (gy * h * scale).sum(0).to(t)
    return out


def _plain_linear(s, case):
    t = s["x"].dtype
    x, w, b, r = _wide(s["x"]), _wide(s["weight"]), _wide(s["bias"]), _wide(s["residual"])
    z = torch.matmul(x, w.t())
    if b is not None:
        z = z + b
    y = _act(z, case["activation"])
    if r is not None:
        y = y + r
    out = {"y": y.to(t)}
    if case["grad"]:
        dz = _wide(s["gy"])
        if case["activation"]:
            dz = dz * _act_slope(z, case["activation"])
        out["dx"] = torch.matmul(dz, w).to(t)
        out["dw"] = torch.matmul(dz.t(), x).to(t)
        if b is not None:
            out["db"] = dz.sum(0).to(t)
    return out


def _plain_q8(s, case):
    z = torch.matmul(s["q"].float(), s["weight_q"].float().t()) * s["scale"].unsqueeze(-1) * s["weight_scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[case["type"]])


def _plain_orth(g):
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2)
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + 1e-7)
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-1, -2))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    if tall:
        x = x.transpose(-1, -2)
    return x.to(g.dtype).contiguous()


def _own(s, case):
    from ae_mlsys_gnn_amd import operators as ops
    kind = case["kind"]
    if kind == "norm":
        r = s["residual"]
        if r is None:
            y = ops.rms_norm(s["x"], s["weight"], eps=EPS)
            dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["gy"])
            return {"y": y.detach(), "dx": dx, "dw": dw}
        y, h = ops.rms_norm(s["x"], s["weight"], residual=r, eps=EPS)
        dx, dw = torch.autograd.grad((y, h), (s["x"], s["weight"]), (s["gy"], s["gh"]))
        return {"h": h.detach(), "y": y.detach(), "dx": dx, "dw": dw}
    if kind == "norm_q8":
        q, scale, *h = ops.rms_norm_q8(s["x"], s["weight"], residual=s["residual"], eps=EPS, dtype=EIGHT[case["eight"]][0])
        out = {"h": h[0]} if h else {}
        out["scale"] = scale
        out["values"] = torch.mul(q if case["eight"] == "int8" else q.float(), scale.unsqueeze(-1), out=torch.empty_like(s["x"]))
        return out
    if kind == "linear":
        if not case["grad"]:
            return {"y": ops.linear_act(s["x"], s["weight"], s["bias"], residual=s["residual"], activation=case["activation"])}
        y = ops.linear_act(s["x"], s["weight"], s["bias"], residual=s["residual"], activation=case["activation"])
        wanted = [s["x"], s["weight"]] + ([] if s["bias"] is None else [s["bias"]])
        return {"y": y.detach(), **dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, wanted, s["gy"])))}
    if kind == "linear_q8":
        return ops.linear_q8(s["q"], s["scale"], s["weight_q"], s["weight_scale"], s["bias"], residual=s["residual"], activation=case["activation"],
                             dtype=TYPES[case["type"]])
    return ops.orthogonalize(s["g"], steps=STEPS, coefficients=COEFFICIENTS)


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["kind"] in ("norm", "norm_q8"):
        return _plain_norm(state, case)
    if case["kind"] == "linear":
        return _plain_linear(state, case)
    if case["kind"] == "linear_q8":
        return _plain_q8(state, case)
    return _plain_orth(state["g"])


def work(case):
    """Inputs read once, outputs written once; the norms' operations are the multiplications and additions of their formulas."""
    size = 4 if case["type"] == "fp32" else 2
    kind = case["kind"]
    if kind == "norm":
        one = case["rows"] * case["cols"]
        # forward x (+ r) -> y (+ h), backward gy, h (+ gh) -> dx
        return {"bytes": (8 if case["residual"] else 5) * one * size + 3 * case["cols"] * size, "flops": 14.0 * one}
    if kind == "norm_q8":
        # the values that the 8 bits stand for are handed out in the input's type
        one = case["rows"] * case["cols"]
        return {"bytes": ((3 if case["residual"] else 1) * size + 1 + 1 + size) * one + case["cols"] * size + 8 * case["rows"], "flops": 6.0 * one}
    if kind == "orth":
        small, wide = min(case["m"], case["n"]), max(case["m"], case["n"])
        # the two symmetric products have half of their elements to be formed
        return {"bytes": 2.0 * case["batch"] * small * wide * size, "flops": float(case["batch"]) * STEPS * (small * small * wide + small ** 3 + 2 * small * small * wide)}
    m, k, n = case["rows"], case["k"], case["n"]
    edges = n * (1 if case["bias"] else 0) + m * n * (1 if case["residual"] else 0)
    if kind == "linear_q8":
        return {"bytes": m * k + n * k + 4 * (m + n) + size * (edges + m * n), "flops": 2.0 * m * k * n}
    forward = (m * k + n * k + edges + m * n) * size
    if not case["grad"]:
        return {"bytes": forward, "flops": 2.0 * m * k * n}
    # backward: the gradient and what the slope is taken from, x and the weights again, their gradients out
    slope = m * n if case["activation"] else 0
    return {"bytes": forward + (2 * slope + m * n + 2 * m * k + 2 * n * k + (n if case["bias"] else 0)) * size, "flops": 6.0 * m * k * n}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    kind = case["kind"]
    d = {k: v.detach().to(torch.float64) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if kind in ("norm", "norm_q8"):
        h = d["x"] + d["residual"] if "residual" in d else d["x"]
        rms = (h.square().sum(-1) / case["cols"] + EPS).sqrt()
        unit = h / rms[:, None]
        y = unit * d["weight"]
        out = {"h": h} if "residual" in d else {}
        if kind == "norm_q8":
            top = EIGHT[case["eight"]][1]
            scale = torch.linalg.vector_norm(y, ord=math.inf, dim=-1) / top
            v = y / scale[:, None].clamp_min(1e-300)
            v = v.round() if case["eight"] == "int8" else _to_e4m3(v)
            return {**out, "scale": scale, "values": v * scale[:, None]}
        # the gradient of the unit vectors has no part along them
        g = d["gy"] * d["weight"]
        dx = (g - unit * (g * unit).sum(-1, keepdim=True) / case["cols"]) / rms[:, None]
        return {**out, "y": y, "dx": dx + d["gh"] if "residual" in d else dx, "dw": torch.einsum("ij,ij->j", d["gy"], unit)}
    if kind == "orth":
        return torch.stack([_exact_orth(g) for g in d["g"]])
    if kind == "linear_q8":
        x, w = d["q"] * d["scale"][:, None], d["weight_q"] * d["weight_scale"][:, None]
    else:
        x, w = d["x"], d["weight"]
    z = x @ w.t().contiguous()
    if "bias" in d:
        z += d["bias"]
    name = case["activation"]
    # value and slope from the distribution functions
    if name == "relu":
        slope = torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
        y = slope * z
    elif name == "silu":
        p = torch.special.expit(z)
        y, slope = p * z, p + z * p * torch.special.expit(-z)
    elif name == "gelu":
        p = torch.special.ndtr(z)
        y, slope = p * z, p + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, None
    y = y + d["residual"] if "residual" in d else y
    if kind == "linear_q8":
        return y
    out = {"y": y}
    if case["grad"]:
        dz = d["gy"] if slope is None else d["gy"] * slope
        out.update(dx=dz @ w, dw=(x.t().contiguous() @ dz).t())
        if "bias" in d:
            out["db"] = dz.sum(0)
    return out


def _to_e4m3(v):
    """The nearest values with four significant bits, exponents from -6 up, ties to even."""
    exponent = torch.frexp(v)[1].clamp_min(-5).to(v.dtype)
    unit = torch.exp2(exponent - 4)
    return torch.round(v / unit) * unit


def _exact_orth(g):
    """The iteration carried out on the Gram matrix: every step multiplies by a polynomial of it."""
    a, b, c = COEFFICIENTS
    x = g if g.shape[0] <= g.shape[1] else g.t().contiguous()
    x = x / (torch.linalg.matrix_norm(x) + 1e-7)
    gram = x @ x.t().contiguous()
    one = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
    left = one
    for _ in range(STEPS):
        m = a * one + b * gram + c * gram @ gram
        left, gram = m @ left, m @ gram @ m
    x = left @ x
    return (x if g.shape[0] <= g.shape[1] else x.t()).contiguous()
