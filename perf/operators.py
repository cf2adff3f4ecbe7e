"""Timed cases of the transformer-layer operators: the linear layer with its fused epilogue and the
layer norm, each forward and backward.

The synthesiser's text encoder, flow and duration predictor (the part of the model in front of the
decoder) are made of these: projections with bias, activation and residual, and layer norms.
``own = False`` runs the operators in elementary torch operations in 32 bits; ``own = True`` calls
the library.

    linear            y = act(x W^T + b) + r        (pre = x W^T + b kept for the backward pass)
    linear_backward   dpre = dy * act'(pre);  dx = dpre W;  dW = dpre^T x;  db = sum_rows dpre
    layer_norm        y = (x - mean) * rstd * gamma + beta,  rstd = 1 / sqrt(var + eps)
    layer_norm_backward
                      g = dy * gamma;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat));
                      dgamma = sum_rows dy * xhat;  dbeta = sum_rows dy
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
SLOPE = 0.1            # the model's leaky slope
ACTS = ("none", "leaky", "relu", "gelu", "silu")

# the largest products and tensors that draw() makes: those of the largest listed cases
MAX_FORWARD = 16384 * 4096 * 4096
MAX_BACKWARD = 8192 * 1024 * 4096
MAX_NORM = 32768 * 4096


def _linear(name, dtype, rows, n_in, n_out, act="none", residual=False, save=False, pad=0):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "in": n_in, "out": n_out,
            "act": act, "residual": residual, "save": save, "pad": pad}


def _linear_bwd(name, dtype, rows, n_in, n_out, act="none", pad=0):
    return {"name": name, "op": "linear_backward", "dtype": dtype, "rows": rows, "in": n_in,
            "out": n_out, "act": act, "pad": pad}


def _norm(name, dtype, rows, cols, pad=0):
    return {"name": name, "op": "layer_norm", "dtype": dtype, "rows": rows, "cols": cols, "pad": pad}


def _norm_bwd(name, dtype, rows, cols, pad=0):
    return {"name": name, "op": "layer_norm_backward", "dtype": dtype, "rows": rows, "cols": cols,
            "pad": pad}


def listed():
    return [
        # one token through the expanding half of an encoder feed-forward layer: pure latency
        _linear("linear token f32", "f32", 1, 192, 768, act="relu"),
        # four sequences, one new token each, through a contracting projection: the weights' bytes
        _linear("linear tokens bf16", "bf16", 4, 4096, 1024, residual=True),
        # every frame of a 64-request batch through an encoder feed-forward layer, full precision
        _linear("linear batch f32", "f32", 19434, 192, 768, act="relu"),
        # a ragged batch whose input is a column slice of a wider tensor, widths not multiples of 8
        _linear("linear ragged f16", "f16", 601, 193, 515, act="silu", residual=True, pad=194),
        # a training batch at the large end, pre-activation kept for the backward pass
        _linear("linear train bf16", "bf16", 16384, 4096, 4096, act="gelu", save=True),
        # fine-tuning one utterance batch in full precision, contracting projection
        _linear_bwd("linear bwd f32", "f32", 3616, 768, 192),
        # a training step of a wide feed-forward layer
        _linear_bwd("linear bwd bf16", "bf16", 8192, 1024, 4096, act="gelu"),
        # a short ragged batch, odd widths
        _linear_bwd("linear bwd ragged f16", "f16", 601, 193, 515, act="silu"),
        # one token's norm
        _norm("norm token f32", "f32", 1, 192),
        # a training batch's norm: bytes
        _norm("norm train bf16", "bf16", 32768, 4096),
        # every frame of a 64-request batch, encoder width
        _norm_bwd("norm bwd f32", "f32", 19434, 192),
        # a training batch, wide
        _norm_bwd("norm bwd bf16", "bf16", 16384, 4096),
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; half of them whole multiples of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        v = (v + 7) // 8 * 8
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("linear", "linear_backward", "layer_norm", "layer_norm_backward"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    pad = rng.choice((0, 0, 8, 3))
    if op.startswith("layer_norm"):
        cols = _size(rng, 32, 8192)
        rows = min(_size(rng, 1, 32768), MAX_NORM // cols)
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "pad": pad}
    n_in, n_out = _size(rng, 16, 4096), _size(rng, 16, 4096)
    act = rng.choice(ACTS)
    if op == "linear":
        rows = min(_size(rng, 1, 16384), MAX_FORWARD // (n_in * n_out))
        return {"op": op, "dtype": dtype, "rows": rows, "in": n_in, "out": n_out, "act": act,
                "residual": rng.random() < 0.5, "save": rng.random() < 0.3, "pad": pad}
    rows = min(_size(rng, 1, 16384), MAX_BACKWARD // (n_in * n_out))
    return {"op": op, "dtype": dtype, "rows": rows, "in": n_in, "out": n_out, "act": act, "pad": pad}


def _rows(gen, rows, cols, pad, dtype, scale=1.0, shift=0.0):
    """[rows][cols] of N(shift, scale^2), a column slice of [rows][cols + pad]."""
    t = torch.randn(rows, cols + pad, generator=gen, device="cuda") * scale + shift
    return t.to(dtype)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows, pad = DTYPES[case["dtype"]], case["rows"], case["pad"]
    s = dict(case)
    if case["op"].startswith("linear"):
        n_in, n_out = case["in"], case["out"]
        s["x"] = _rows(gen, rows, n_in, pad, dt)
        s["w"] = _rows(gen, n_out, n_in, 0, dt, 1.0 / math.sqrt(n_in))
        s["b"] = _rows(gen, 1, n_out, 0, dt, 0.1)[0]
        if case["op"] == "linear":
            s["r"] = _rows(gen, rows, n_out, 0, dt) if case["residual"] else None
        else:   # what the forward pass of the same layer left behind, and the gradient that arrives
            s["pre"] = (s["x"].float() @ s["w"].float().T + s["b"].float()).to(dt)
            s["dy"] = _rows(gen, rows, n_out, 0, dt)
    else:
        cols = case["cols"]
        s["x"] = _rows(gen, rows, cols, pad, dt, 1.0, 0.25)
        s["gamma"] = _rows(gen, 1, cols, 0, dt, 0.1, 1.0)[0]
        s["beta"] = _rows(gen, 1, cols, 0, dt, 0.1)[0]
        if case["op"] == "layer_norm_backward":
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
            s["dy"] = _rows(gen, rows, cols, 0, dt)
    return s


_library = None


def _ops():
    """The library's operator handle, opened once as a program would."""
    global _library
    if _library is None:
        path = os.path.join(ROOT, "prime-tts_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import pt_b200
        _library = pt_b200.Operators(device=torch.cuda.current_device())
    return _library


def _act(pre, act):
    if act == "leaky":
        return torch.where(pre >= 0, pre, SLOPE * pre)
    if act == "relu":
        return torch.where(pre > 0, pre, torch.zeros_like(pre))
    if act == "gelu":
        return 0.5 * pre * (1.0 + torch.erf(pre * math.sqrt(0.5)))
    if act == "silu":
        return pre / (1.0 + torch.exp(-pre))
    return pre


def _act_grad(pre, act):
    if act == "leaky":
        return torch.where(pre >= 0, torch.ones_like(pre), torch.full_like(pre, SLOPE))
    if act == "relu":
        return (pre > 0).to(pre.dtype)
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(pre * math.sqrt(0.5)))
        return cdf + pre * torch.exp(-0.5 * pre * pre) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-pre))
        return sig * (1.0 + pre * (1.0 - sig))
    return torch.ones_like(pre)


def _plain(s):
    dt = DTYPES[s["dtype"]]
    x = s["x"].float()
    if s["op"] == "linear":
        pre = x @ s["w"].float().T + s["b"].float()
        y = _act(pre, s["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        return {"y": y.to(dt), "pre": pre.to(dt)} if s["save"] else {"y": y.to(dt)}
    if s["op"] == "linear_backward":
        g = s["dy"].float() * _act_grad(s["pre"].float(), s["act"])
        return {"dx": (g @ s["w"].float()).to(dt), "dw": (g.T @ x).to(dt), "db": g.sum(0).to(dt)}
    if s["op"] == "layer_norm":
        mean = x.mean(1)
        c = x - mean[:, None]
        rstd = torch.rsqrt(c.square().mean(1) + EPS)
        y = c * rstd[:, None] * s["gamma"].float() + s["beta"].float()
        return {"y": y.to(dt), "mean": mean, "rstd": rstd}
    dy = s["dy"].float()
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["gamma"].float()
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return {"dx": dx.to(dt), "dgamma": (dy * xhat).sum(0).to(dt), "dbeta": dy.sum(0).to(dt)}


def run(state):
    if not own:
        return _plain(state)
    s, ops = state, _ops()
    if s["op"] == "linear":
        if s["save"]:
            y, pre = ops.linear(s["x"], s["w"], s["b"], residual=s["r"], act=s["act"], slope=SLOPE,
                                save_pre=True)
            return {"y": y, "pre": pre}
        return {"y": ops.linear(s["x"], s["w"], s["b"], residual=s["r"], act=s["act"], slope=SLOPE)}
    if s["op"] == "linear_backward":
        dx, dw, db = ops.linear_backward(s["dy"], s["x"], s["w"], pre=s["pre"], act=s["act"],
                                         slope=SLOPE)
        return {"dx": dx, "dw": dw, "db": db}
    if s["op"] == "layer_norm":
        y, mean, rstd = ops.layer_norm(s["x"], s["gamma"], s["beta"], eps=EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    dx, dgamma, dbeta = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"])
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if case["op"].startswith("linear"):
        n_in, n_out, act = case["in"], case["out"], case["act"] != "none"
        x, w, y = rows * n_in, n_out * n_in, rows * n_out
        if case["op"] == "linear":
            return {"bytes": size * (x + w + n_out + y * (1 + case["residual"] + case["save"])),
                    "flops": 2.0 * rows * n_in * n_out}
        # dy (and pre where the activation needs it), x and W in; dx, dW and db out
        return {"bytes": size * (y * (1 + act) + 2 * x + 2 * w + n_out),
                "flops": 4.0 * rows * n_in * n_out}
    n, cols = rows * case["cols"], case["cols"]
    if case["op"] == "layer_norm":
        return {"bytes": size * (2 * n + 2 * cols) + 8 * rows, "flops": 8.0 * n}
    return {"bytes": size * (3 * n + 3 * cols) + 8 * rows, "flops": 14.0 * n}


def exact(case, seed):
    """The same outputs from torch's float64 functions and their derivatives."""
    import torch.nn.functional as F

    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    acts = {"none": lambda t: t * 1.0, "leaky": lambda t: F.leaky_relu(t, SLOPE), "relu": F.relu,
            "gelu": F.gelu, "silu": F.silu}
    if s["op"] == "linear":
        pre = F.linear(s["x"], s["w"], s["b"])
        y = acts[s["act"]](pre)
        y = y if s["r"] is None else y + s["r"]
        return {"y": y, "pre": pre} if s["save"] else {"y": y}
    if s["op"] == "linear_backward":
        pre = s["pre"].requires_grad_()
        (g,) = torch.autograd.grad(acts[s["act"]](pre), pre, s["dy"])
        return {"dx": torch.matmul(g, s["w"]), "dw": torch.matmul(g.transpose(0, 1), s["x"]),
                "db": torch.sum(g, 0)}
    cols = (case["cols"],)
    if s["op"] == "layer_norm":
        var, mean = torch.var_mean(s["x"], 1, correction=0)
        return {"y": F.layer_norm(s["x"], cols, s["gamma"], s["beta"], EPS), "mean": mean,
                "rstd": (var + EPS) ** -0.5}
    x, gamma = s["x"].requires_grad_(), s["gamma"].requires_grad_()
    beta = s["beta"].requires_grad_()
    dx, dgamma, dbeta = torch.autograd.grad(F.layer_norm(x, cols, gamma, beta, EPS),
                                            (x, gamma, beta), s["dy"])
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
