"""Cases, plain forms and 64-bit values of the decoder operators in
``quantem.cuda.core.ml``: the root-mean-square norm with the residual's
addition (16/32-bit output, or 8-bit output with one scale per row) and the
matrix product with bias, activation and residual in its epilogue (16-bit
operands, trained; 8-bit operands with scales, serving).

They stand behind the K-Planes encoder: its features ``[points, T*C]`` are
normalised and go through the layers of a decoder. Rows are points (from one
point to the samples of many rays), widths are feature counts (T*C = 128 and
256 for one level, 1024 for a four-level encoding) and decoder widths.

``run`` is one pass: a call, or with ``train`` a call and its gradients.
"""

import math
import os
import sys

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ── cases ──────────────────────────────────────────────────────────────────


def _norm(rows, n, x, out, residual, train, name=None):
    c = {"op": "norm", "rows": rows, "n": n, "x": x, "out": out, "residual": residual, "train": train}
    return {"name": name, **c} if name else c


def _norm_fp8(rows, n, x, residual, name=None):
    c = {"op": "norm_fp8", "rows": rows, "n": n, "x": x, "residual": residual}
    return {"name": name, **c} if name else c


def _linear(rows, k, n, x, out, bias, residual, act, train, name=None):
    c = {"op": "linear", "rows": rows, "k": k, "n": n, "x": x, "out": out, "bias": bias, "residual": residual,
         "act": act, "train": train}
    return {"name": name, **c} if name else c


def _linear_fp8(rows, k, n, out, bias, residual, act, name=None):
    c = {"op": "linear_fp8", "rows": rows, "k": k, "n": n, "out": out, "bias": bias, "residual": residual, "act": act}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the features of one point, normalised for a bf16 decoder: a probe of the field
        _norm(1, 128, "fp32", "bf16", False, False, "norm_one_point"),
        # a training step's points: fp32 features of T = 8 rotations, C = 32
        _norm(262144, 256, "fp32", "bf16", False, True, "norm_train_features"),
        # the residual stream of a wide decoder in training
        _norm(65536, 1024, "bf16", "bf16", True, True, "norm_train_stream"),
        # odd rows and an odd width: nothing is a multiple of a vector
        _norm(10007, 999, "fp16", "fp16", True, True, "norm_train_odd"),
        # serving a volume's points: the stream's norm straight to 8 bits
        _norm_fp8(131072, 512, "bf16", True, "norm_fp8_stream"),
        # one point through a wide layer: bound by reading the weights
        _linear(1, 1024, 1024, "bf16", "bf16", True, False, "gelu", False, "linear_one_point"),
        # a narrow field decoder's layer over many points, trained
        _linear(262144, 256, 256, "bf16", "bf16", True, False, "gelu", True, "linear_train_field"),
        # odd rows, an input width and an output width that no vector divides
        _linear(20011, 203, 77, "fp16", "fp16", True, True, "silu", True, "linear_train_odd"),
        # the widening layer of a residual block, trained
        _linear(8192, 1024, 4096, "bf16", "bf16", True, False, "silu", True, "linear_train_wide"),
        # the narrowing layer of a wide block with the stream added: bound by the tensor cores
        _linear(16384, 4096, 4096, "bf16", "bf16", True, True, "none", False, "linear_wide"),
        # a few points through a wide layer with 8-bit weights
        _linear_fp8(16, 4096, 4096, "bf16", False, True, "none", "linear_fp8_few"),
        # a volume's points through a wide layer with 8-bit operands
        _linear_fp8(32768, 2048, 2048, "bf16", True, False, "relu", "linear_fp8_many"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width over the logarithm of [lo, hi]: half of them multiples of 16, the others whatever comes."""
    w = _log(rng, lo, hi)
    return max(16, w // 16 * 16) if rng.random() < 0.5 and w >= 16 else w


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_fp8", "linear", "linear", "linear_fp8"])
    if op in ("norm", "norm_fp8"):
        n = _width(rng, 4, 8192)
        rows = _log(rng, 1, max(1, 2**26 // n))
        x = rng.choice(["fp32", "bf16", "fp16"])
        residual = rng.random() < 0.5
        if op == "norm_fp8":
            return _norm_fp8(rows, n, x, residual)
        out = rng.choice(["bf16", "fp16", "fp32"]) if x == "fp32" else x
        return _norm(rows, n, x, out, residual, rng.random() < 0.5)
    k, n = _width(rng, 8, 4096), _width(rng, 1, 4096)
    rows = _log(rng, 1, max(1, min(2**26 // max(k, n), 2**36 // (k * n))))
    bias, residual = rng.random() < 0.7, rng.random() < 0.4
    act = rng.choice(["none", "relu", "silu", "gelu"])
    if op == "linear_fp8":
        return _linear_fp8(rows, k, n, rng.choice(["bf16", "fp16", "fp32"]), bias, residual, act)
    x = rng.choice(["bf16", "bf16", "fp16"])
    return _linear(rows, k, n, x, rng.choice([x, x, "fp32"]), bias, residual, act, rng.random() < 0.5)


# ── inputs ─────────────────────────────────────────────────────────────────


def _quantized(v):
    """Rows of `v` as e4m3 with one fp32 scale per row."""
    scale = (v.abs().amax(-1) / E4M3_MAX).clamp_min(2.0**-126)
    return (v / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    op, rows, n = case["op"], case["rows"], case["n"]
    s = {"case": case, "call": _calls() if own else None}
    if op in ("norm", "norm_fp8"):
        t = TYPES[case["x"]]
        # rows of different magnitude, as features of different points have
        s["x"] = (randn(rows, n) * torch.exp(randn(rows, 1, scale=0.5))).to(t)
        s["residual"] = randn(rows, n).to(t) if case["residual"] else None
        s["weight"] = (1.0 + randn(n, scale=0.1)).to(t)
        if case.get("train"):
            s["dy"] = randn(rows, n).to(TYPES[case["out"]])
            s["dh"] = randn(rows, n).to(t) if case["residual"] else None
            leaves = ["x", "residual", "weight"]
    else:
        k = case["k"]
        if op == "linear":
            t = TYPES[case["x"]]
            s["x"] = randn(rows, k).to(t)
            s["weight"] = randn(n, k, scale=k**-0.5).to(t)
        else:
            s["x"], s["x_scale"] = _quantized(randn(rows, k))
            s["weight"], s["weight_scale"] = _quantized(randn(n, k, scale=k**-0.5))
        t = TYPES[case["out"]] if op == "linear_fp8" else t
        s["bias"] = randn(n, scale=0.5).to(t) if case["bias"] else None
        s["residual"] = randn(rows, n).to(TYPES[case["out"]]) if case["residual"] else None
        if case.get("train"):
            s["dy"] = randn(rows, n).to(TYPES[case["out"]])
            leaves = ["x", "weight", "bias", "residual"]
    if case.get("train"):
        s["leaves"] = [name for name in leaves if s[name] is not None]
        for name in s["leaves"]:
            s[name].requires_grad_(True)
    return s


def _calls():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quantem-cuda_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from quantem.cuda.core import ml

    return ml


# ── the operators ──────────────────────────────────────────────────────────


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _plain_norm(s):
    case = s["case"]
    x, w = s["x"].detach(), s["weight"].detach()
    h = x.float() if s["residual"] is None else x.float() + s["residual"].detach().float()
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    xn = h * r
    y = xn * w.float()
    if case["op"] == "norm_fp8":
        q, scale = _quantized(y)
        got = {"q": q, "scale": scale}
        if s["residual"] is not None:
            got["h"] = h.to(x.dtype)
        return got
    got = {"y": y.to(TYPES[case["out"]])}
    if s["residual"] is not None:
        got["h"] = h.to(x.dtype)
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w.float()
        dx = r * (g - xn * (g * xn).mean(-1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["dh"].float()
            got["dresidual"] = dx.to(x.dtype)
        got["dx"] = dx.to(x.dtype)
        got["dweight"] = (dy * xn).sum(0, dtype=torch.float64).to(w.dtype)
    return got


def _plain_linear(s):
    case = s["case"]
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    z = x @ w.T
    if case["op"] == "linear_fp8":
        z = z * s["x_scale"][:, None] * s["weight_scale"]
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    got = {"y": y.to(TYPES[case["out"]])}
    if case.get("train"):
        t = s["x"].dtype
        dy = s["dy"]
        dz = dy.float() * _act_grad(z, case["act"])
        got["dx"] = (dz @ w).to(t)
        got["dweight"] = (dz.T @ x).to(t)
        if s["bias"] is not None:
            got["dbias"] = dz.sum(0, dtype=torch.float64).to(t)
        if s["residual"] is not None:
            got["dresidual"] = dy
    return got


def _own_norm(s):
    ml, case, x, w, res = s["call"], s["case"], s["x"], s["weight"], s["residual"]
    if case["op"] == "norm_fp8":
        if res is None:
            q, scale = ml.rms_norm_fp8(x, w, eps=EPS)
            return {"q": q, "scale": scale}
        q, scale, h = ml.add_rms_norm_fp8(x, res, w, eps=EPS)
        return {"q": q, "scale": scale, "h": h}
    out = TYPES[case["out"]]
    if res is None:
        outs = {"y": ml.rms_norm(x, w, eps=EPS, out_dtype=out)}
        ups = [s["dy"]] if case["train"] else []
    else:
        y, h = ml.add_rms_norm(x, res, w, eps=EPS, out_dtype=out)
        outs = {"y": y, "h": h}
        ups = [s["dy"], s["dh"]] if case["train"] else []
    return _with_grads(s, outs, ups)


def _own_linear(s):
    ml, case = s["call"], s["case"]
    out = TYPES[case["out"]]
    if case["op"] == "linear_fp8":
        return {"y": ml.linear_act_fp8(s["x"], s["x_scale"], s["weight"], s["weight_scale"], bias=s["bias"],
                                       residual=s["residual"], activation=case["act"], out_dtype=out)}
    y = ml.linear_act(s["x"], s["weight"], bias=s["bias"], residual=s["residual"], activation=case["act"],
                      out_dtype=out)
    return _with_grads(s, {"y": y}, [s["dy"]] if case["train"] else [])


def _with_grads(s, outs, ups):
    if not s["case"]["train"]:
        return outs
    grads = torch.autograd.grad(list(outs.values()), [s[n] for n in s["leaves"]], ups)
    got = {k: v.detach() for k, v in outs.items()}
    got.update({"d" + n: d for n, d in zip(s["leaves"], grads)})
    return got


def run(state):
    norm = state["case"]["op"].startswith("norm")
    if own:
        return _own_norm(state) if norm else _own_linear(state)
    return _plain_norm(state) if norm else _plain_linear(state)


# ── what a pass cannot do without ──────────────────────────────────────────


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    op, rows, n = case["op"], case["rows"], case["n"]
    if op in ("norm", "norm_fp8"):
        e = size[case["x"]]
        streams = 3 if case["residual"] else 1  # x; with a residual also the residual and their sum
        out = 1 if op == "norm_fp8" else size[case["out"]]
        b = rows * n * (streams * e + out) + n * e + (4 * rows if op == "norm_fp8" else 0)
        f = 6.0 * rows * n
        if case.get("train"):  # the upstream gradients in, the input's and the weight's out
            b += rows * n * (out + e + (e if case["residual"] else 0)) + n * e
            f += 12.0 * rows * n
        return {"bytes": b, "flops": f}
    k = case["k"]
    e = 1 if op == "linear_fp8" else size[case["x"]]
    o = size[case["out"]]
    eb = o if op == "linear_fp8" else e
    b = rows * k * e + n * k * e + rows * n * o * (2 if case["residual"] else 1) + (n * eb if case["bias"] else 0)
    b += 4 * (rows + n) if op == "linear_fp8" else 0
    f = 2.0 * rows * n * k
    if case.get("train"):
        b += rows * n * o + rows * k * e + n * k * e + (n * eb if case["bias"] else 0)
        f *= 3
    return {"bytes": b, "flops": f}


# ── 64 bits ────────────────────────────────────────────────────────────────


def _exact_act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z * torch.special.expit(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z


def exact(case, seed):
    """The definitions evaluated in 64 bits on the same inputs, gradients by differentiating them."""
    s = prepare(case, seed)
    d = {k: v.detach().double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    train = bool(case.get("train"))
    for name in s.get("leaves", []):
        d[name].requires_grad_(True)
    got = {}
    if case["op"].startswith("norm"):
        h = d["x"] if d["residual"] is None else d["x"] + d["residual"]
        y = d["weight"] * h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / case["n"] + EPS)
        if case["op"] == "norm_fp8":
            scale = torch.clamp(y.abs().max(-1).values / E4M3_MAX, min=2.0**-126)
            got = {"q": (y / scale.unsqueeze(-1)).float().to(torch.float8_e4m3fn).double(), "scale": scale}
        else:
            got = {"y": y}
        if d["residual"] is not None:
            got["h"] = h
        outs = {k: got[k] for k in ("y", "h") if k in got}
        ups = [d["dy"], d["dh"]] if train and d["residual"] is not None else [d["dy"]] if train else []
    else:
        x, w = d["x"], d["weight"]
        if case["op"] == "linear_fp8":
            x, w = x * d["x_scale"].unsqueeze(-1), w * d["weight_scale"].unsqueeze(-1)
        y = torch.einsum("rk,nk->rn", x, w)
        y = _exact_act(y if d["bias"] is None else y + d["bias"], case["act"])
        y = y if d["residual"] is None else y + d["residual"]
        got = outs = {"y": y}
        ups = [d["dy"]] if train else []
    got = {k: v.detach() for k, v in got.items()}
    if train:
        grads = torch.autograd.grad([outs[k] for k in outs], [d[n] for n in s["leaves"]], ups)
        got.update({"d" + n: v for n, v in zip(s["leaves"], grads)})
    return got
