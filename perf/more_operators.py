"""The feed-forward half of a layer: the layer norm with a residual in front of it, the gated product (both projections, the
activation and the product of the two), and the products of rows in 8-bit integers that take their place when the layer serves.

``listed()`` names the cases, ``draw(rng)`` gives another one of the same ranges, ``prepare(case, seed)`` makes what a
program holds before the call, ``run(state)`` is one pass (``own``: through this package, otherwise in elementary torch
operations), ``work(case)`` what a pass cannot do without, and ``exact(case, seed)`` the result in 64 bits."""
import math
import os
import sys

import torch

own = False

INT8_MAX = 127.0
AMAX_MIN = 1e-30      # rows whose largest magnitude is below this are scaled as if it were this
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _norm(name, mode, rows, dim, dtype="bf16", residual=None):
    """``mode``: forward, train (gradients of everything); ``residual``: its type."""
    c = {"op": "norm", "mode": mode, "rows": rows, "dim": dim, "dtype": dtype, "residual": residual or dtype}
    return c if name is None else dict(c, name=name)


def _gated(name, mode, rows, dim, inner, dtype="bf16", act="silu", bias=False):
    """``mode``: forward, train (gradients of everything), int8 (rows and weights in 8-bit integers with their scales)."""
    c = {"op": "gated", "mode": mode, "rows": rows, "dim": dim, "inner": inner, "dtype": dtype, "act": act, "bias": bias}
    return c if name is None else dict(c, name=name)


def _linear(name, source, rows, out, inner, dtype="bf16", bias=True, act="none", residual=False):
    """``source``: rows (in 8-bit integers with their scales, as the step ahead leaves them), wide (``dtype``, brought to 8 bits within
    the call)."""
    c = {"op": "linear", "source": source, "rows": rows, "out": out, "inner": inner, "dtype": dtype, "bias": bias, "act": act,
         "residual": residual}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # The norm in front of a decode step's feed-forward: launch and host time.
        _norm("norm_step", "forward", 32, 2048),
        # The pre-norm of a training step: the residual stream, weight and bias, all gradients.
        _norm("norm_train", "train", 16384, 2048),
        # Half precision with the residual stream kept in 32 bits, odd numbers of rows and columns.
        _norm("norm_ragged_train", "train", 5003, 1001, dtype="fp16", residual="fp32"),
        # The next token of one sequence: the weights' bytes.
        _gated("gated_step", "forward", 1, 2048, 5632),
        # The next tokens of a serving batch on a wider model.
        _gated("gated_batch", "forward", 48, 4096, 11008, dtype="fp16"),
        # A prompt of an odd length, the activation of the error function, biases.
        _gated("gated_prompt", "forward", 8191, 2048, 5632, act="gelu", bias=True),
        # A pre-training step of 2 x 4096 tokens.
        _gated("gated_train", "train", 8192, 2048, 5632),
        # Fine-tuning on a short ragged batch, half precision, odd sizes throughout.
        _gated("gated_ragged_train", "train", 1003, 1000, 2731, dtype="fp16", act="gelu", bias=True),
        # A prompt's gated product in 8 bits, behind a norm that leaves 8-bit rows.
        _gated("gated_int8_prompt", "int8", 8191, 2048, 5632),
        # A single token's projection from 16-bit rows: the weight's bytes and the launches.
        _linear("int8_step", "wide", 1, 4096, 2048),
        # The output projection of a decode batch, added to the residual stream.
        _linear("int8_batch", "rows", 48, 2048, 8192, residual=True),
        # The output projection of a prompt from 16-bit rows.
        _linear("int8_prompt", "wide", 8191, 2048, 5632, bias=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["norm", "gated", "gated", "gated", "linear", "linear"])
        dtype = rng.choice(["bf16", "fp16"])
        act = rng.choice(["silu", "gelu", "relu"])
        rows = rng.choice([_spread(rng, 1, 64), _spread(rng, 65, 16384)])
        if op == "norm":
            dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
            dim = rng.choice([8 * _spread(rng, 8, 1024), _spread(rng, 64, 8192)])
            case = _norm(None, rng.choice(["forward", "train"]), _spread(rng, 1, 32768), dim, dtype, rng.choice([dtype, "fp32"]))
        elif op == "gated":
            mode = rng.choice(["forward", "train", "train", "int8"])
            dim = 16 * _spread(rng, 16, 256) if mode == "int8" else rng.choice([8 * _spread(rng, 32, 512), _spread(rng, 256, 4096)])
            inner = rng.choice([8 * _spread(rng, 32, 1376), _spread(rng, 256, 11008)])
            case = _gated(None, mode, rows, dim, inner, dtype, act, rng.random() < 0.4)
        else:
            case = _linear(None, rng.choice(["rows", "wide"]), rows, _spread(rng, 256, 16384), 16 * _spread(rng, 16, 512), dtype,
                           rng.random() < 0.5, rng.choice(["none", act]), rng.random() < 0.5)
        if _cost(case) <= most:
            return case


# ---------------------------------------------------------------------------------------------------- inputs
def _rows8(x):
    """Rows in 8-bit integers with a scale each."""
    scale = x.abs().amax(-1).clamp_min(AMAX_MIN) / INT8_MAX
    return torch.round(x / scale[..., None]).to(torch.int8), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).add_(mean).to(dtype)

    s = {"case": case}
    if case["op"] == "norm":
        M, N = case["rows"], case["dim"]
        s["x"], s["residual"] = normal(M, N), normal(M, N, std=2.0, mean=0.3, dtype=DTYPES[case["residual"]])
        s["w"], s["b"] = normal(N, std=0.2, mean=1.0), normal(N, std=0.2)
        if case["mode"] == "train":
            s["dy"], s["ds"] = normal(M, N), normal(M, N, dtype=DTYPES[case["residual"]])
            for k in ("x", "residual", "w", "b"):
                s[k].requires_grad_()
    elif case["op"] == "gated":
        M, D, F = case["rows"], case["dim"], case["inner"]
        wide = torch.float32 if case["mode"] == "int8" else dtype
        s["x"], s["wg"], s["wu"] = normal(M, D, dtype=wide), normal(F, D, std=D ** -0.5, dtype=wide), normal(F, D, std=D ** -0.5, dtype=wide)
        s["bg"], s["bu"] = (normal(F, std=0.2), normal(F, std=0.2)) if case["bias"] else (None, None)
        if case["mode"] == "int8":
            for k in ("x", "wg", "wu"):
                s[k] = _rows8(s[k])
        if case["mode"] == "train":
            s["dh"] = normal(M, F)
            for k in ("x", "wg", "wu", "bg", "bu"):
                if s[k] is not None:
                    s[k].requires_grad_()
    else:
        M, N, K = case["rows"], case["out"], case["inner"]
        x = normal(M, K, dtype=torch.float32)
        s["x"] = _rows8(x) if case["source"] == "rows" else x.to(dtype)
        s["w"] = _rows8(normal(N, K, std=K ** -0.5, dtype=torch.float32))
        s["bias"] = normal(N, std=0.5) if case["bias"] else None
        s["residual"] = normal(M, N) if case["residual"] else None
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _norm_plain(s):
    x, r, w, b = (s[k].detach().float() for k in ("x", "residual", "w", "b"))
    t = x + r
    kept = t.to(s["residual"].dtype)
    mean = t.mean(-1, keepdim=True)
    rstd = torch.rsqrt((t - mean).square().mean(-1, keepdim=True) + EPS)
    y = ((t - mean) * rstd * w + b).to(s["x"].dtype)
    if s["case"]["mode"] != "train":
        return y, kept
    xh = (kept.float() - mean) * rstd
    dy = s["dy"].float()
    wdy = dy * w
    dt = (wdy - wdy.mean(-1, keepdim=True) - xh * (xh * wdy).mean(-1, keepdim=True)) * rstd + s["ds"].float()
    return y, kept, dt.to(s["x"].dtype), dt.to(s["residual"].dtype), (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)


def _act(y, act):
    """The activation and its derivative."""
    if act == "silu":
        sig = torch.sigmoid(y)
        return y * sig, sig * (1 + y * (1 - sig))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(y * 0.5 ** 0.5))
        return y * cdf, cdf + y * torch.exp(-0.5 * y * y) * (2 * math.pi) ** -0.5
    if act == "relu":
        return y.clamp_min(0), (y > 0).float()
    return y, None


def _sums8(x, w):
    """Products of 8-bit rows, with their scales."""
    (xq, xs), (wq, ws) = x, w
    return (xq.float() @ wq.float().t()) * xs[:, None] * ws


def _gated_plain(s):
    case = s["case"]
    if case["mode"] == "int8":
        g, u = _sums8(s["x"], s["wg"]), _sums8(s["x"], s["wu"])
    else:
        x, wg, wu = (s[k].detach().float() for k in ("x", "wg", "wu"))
        g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["bg"].detach().float(), u + s["bu"].detach().float()
    a, da = _act(g, case["act"])
    h = (a * u).to(DTYPES[case["dtype"]])
    if case["mode"] != "train":
        return h
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    out = [h, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x] + ([dg.sum(0), du.sum(0)] if case["bias"] else [])
    return [o.to(h.dtype) for o in out]


def _linear_plain(s):
    case = s["case"]
    y = _sums8(s["x"] if case["source"] == "rows" else _rows8(s["x"].float()), s["w"])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _act(y, case["act"])[0]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[case["dtype"]])


# ---------------------------------------------------------------------------------------------------- the package
def _package():
    path = os.path.join(os.getcwd(), "flash-linear-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fla_amd
    return fla_amd


def _norm_own(s):
    y, kept = _package().modules.layer_norm(s["x"], s["w"], s["b"], residual=s["residual"], prenorm=True, eps=EPS)
    if s["case"]["mode"] != "train":
        return y, kept
    return [y, kept, *torch.autograd.grad((y, kept), (s["x"], s["residual"], s["w"], s["b"]), (s["dy"], s["ds"]))]


def _gated_own(s):
    modules, case = _package().modules, s["case"]
    if case["mode"] == "int8":
        return modules.quant_gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=case["act"],
                                          output_dtype=DTYPES[case["dtype"]])
    h = modules.gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=case["act"])
    if case["mode"] != "train":
        return h
    return [h, *torch.autograd.grad(h, [s[k] for k in ("x", "wg", "wu", "bg", "bu") if s[k] is not None], s["dh"])]


def _linear_own(s):
    modules, case = _package().modules, s["case"]
    x = s["x"] if case["source"] == "rows" else modules.quantize_rows(s["x"], torch.int8)
    return modules.quant_linear(x, s["w"], s["bias"], activation=None if case["act"] == "none" else case["act"],
                                residual=s["residual"], output_dtype=DTYPES[case["dtype"]])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _norm_own, "gated": _gated_own, "linear": _linear_own}[op](state)
    return {"norm": _norm_plain, "gated": _gated_plain, "linear": _linear_plain}[op](state)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    """Every input read once, every output written once."""
    e = BYTES[case["dtype"]]
    if case["op"] == "norm":
        n, r = case["rows"] * case["dim"], BYTES[case["residual"]]
        forward = n * (2 * e + 2 * r)
        return {"bytes": forward + (n * (e + r + e + r) if case["mode"] == "train" else 0), "flops": n * (24 if case["mode"] == "train" else 8)}
    if case["op"] == "gated":
        M, D, F = case["rows"], case["dim"], case["inner"]
        if case["mode"] == "int8":
            return {"bytes": (M + 2 * F) * (D + 4) + M * F * e, "flops": 4 * M * D * F}
        train = case["mode"] == "train"      # (dh in, dx and the weights' gradients out)
        return {"bytes": ((M * D + 2 * F * D) * (1 + train) + M * F * (1 + train)) * e, "flops": 4 * M * D * F * (3 if train else 1)}
    M, N, K = case["rows"], case["out"], case["inner"]
    x = M * K if case["source"] == "rows" else M * K * e
    return {"bytes": x + N * K + M * N * e * (1 + case["residual"]) + 4 * (M + N), "flops": 2 * M * N * K}


# ---------------------------------------------------------------------------------------------------- 64 bits
_EXACT_ACTS = {"none": lambda v: v, "silu": lambda v: v / (1 + torch.exp(-v)), "relu": torch.relu,
               "gelu": lambda v: v * (1 - torch.erfc(v / math.sqrt(2.0)) / 2)}


def _norm_exact(s):
    x, r, w, b = (s[k].detach().double().requires_grad_() for k in ("x", "residual", "w", "b"))
    t = x + r
    c = t - t.sum(-1, keepdim=True) / t.shape[-1]
    y = c / torch.sqrt((c * c).sum(-1, keepdim=True) / t.shape[-1] + EPS) * w + b
    if s["case"]["mode"] != "train":
        return y.detach(), t.detach()
    return [y.detach(), t.detach(), *torch.autograd.grad((y, t), (x, r, w, b), (s["dy"].double(), s["ds"].double()))]


def _dequantised(rows):
    return rows[0].double() * rows[1].double()[:, None]


def _gated_exact(s):
    case = s["case"]
    names = [k for k in ("x", "wg", "wu", "bg", "bu") if s[k] is not None]
    v = {k: _dequantised(s[k]) if isinstance(s[k], tuple) else s[k].detach().double().requires_grad_(case["mode"] == "train") for k in names}
    g, u = torch.mm(v["x"], v["wg"].t().contiguous()), torch.mm(v["x"], v["wu"].t().contiguous())
    h = _EXACT_ACTS[case["act"]](g + v["bg"] if case["bias"] else g) * (u + v["bu"] if case["bias"] else u)
    if case["mode"] != "train":
        return h
    return [h.detach(), *torch.autograd.grad(h, [v[k] for k in names], s["dh"].double())]


def _linear_exact(s):
    case, x = s["case"], s["x"]
    if case["source"] == "wide":      # the rows' own quantisation, in 64 bits
        x = x.double()
        scale = (x.abs().max(-1).values / INT8_MAX).clamp_min(AMAX_MIN / INT8_MAX)
        x = (torch.round(x / scale[:, None]), scale)
    y = torch.mm(_dequantised(x), _dequantised(s["w"]).t().contiguous())
    y = _EXACT_ACTS[case["act"]](y if s["bias"] is None else y + s["bias"].double())
    return y if s["residual"] is None else y + s["residual"].double()


def exact(case, seed):
    return {"norm": _norm_exact, "gated": _gated_exact, "linear": _linear_exact}[case["op"]](prepare(case, seed))
