"""Oracle of the gated product: the formula in fp64, its gradients, and how far the kernels may be from them.

``g = x Wg' + bg``, ``u = x Wu' + bu``, ``h = act(g) u``; ``dg = dh u act'(g)``, ``du = dh act(g)``, ``dx = dg Wg + du Wu``, ``dWg = dg' x``, ``dWu = du' x``.

Bounds, in units of 2^-24.  A sum of K products of 16-bit values: the products are exact in fp32, an instruction adds sixteen of them, and for each instruction four
roundings of the running sum are allowed, which is at most the sum of the magnitudes: ``(K / 4 + 32)`` of that sum.  Activations: slopes of at most 1.13,
second derivatives of at most 0.8, and errors of the evaluation of 3e-7 |g| (the normal distribution within 1.5e-7, two of the hardware's exponentials and reciprocals).
The backward reads g and u as they were summed and rounds dg and du to the operands' type, half a step each.  Those roundings are independent and of either sign:
by Hoeffding's inequality a sum of such errors, each at most c, exceeds 7 sqrt(sum c^2) with a probability below 5e-11."""
import math

import torch

UNIT = 2.0 ** -24
SLOPE, CURVE = 1.13, 0.8


def act(name, v):
    """The activation and its derivative (relu: 0 at 0)."""
    if name in ("silu", "swish"):
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-v / math.sqrt(2.0))
        return v * c, c + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    if name == "relu":
        return v.clamp_min(0), (v > 0).to(v.dtype)
    return v, torch.ones_like(v)


def sum_bound(a, b, n):
    """Of the error of ``a @ b``, sums of n products."""
    return (n / 4 + 32) * UNIT * (a.abs() @ b.abs())


def forward(x, wg, wu, bg=None, bu=None, name="silu", scale=None):
    """``(h, bound, state)`` for x ``[M, K]`` in fp64; ``state``: what :func:`backward` takes."""
    K = x.shape[-1]
    pre = []
    for w, b in ((wg, bg), (wu, bu)):
        v, e = x @ w.t(), sum_bound(x, w.t(), K)
        if b is not None:
            v = v + b
            e = e + UNIT * (v.abs() + b.abs())
        pre += [v, e]
    g, eg, u, eu = pre
    a, slope = act(name, g)
    ea = SLOPE * eg + 3e-7 * g.abs() + (g.abs() + 8) * UNIT * a.abs()
    h = a * u
    return h, u.abs() * ea + a.abs() * eu + ea * eu + 2 * UNIT * h.abs(), (g, eg, u, eu, a, slope)


def backward(x, wg, wu, state, dh, name, half):
    """Gradients and bounds of their errors ahead of their own rounding; ``half``: half a step of the operands' type, relative."""
    g, eg, u, eu, a, slope = state
    M, F = g.shape
    es = CURVE * eg + 1e-6 * (1 + g.abs())
    if name == "relu":
        es = torch.where(g.abs() <= eg, 1.0, 0.0) + 0 * es
    elif name is None:
        es = 0 * es
    ea = SLOPE * eg + 3e-7 * g.abs() + (g.abs() + 8) * UNIT * a.abs()
    dg, du = dh * u * slope, dh * a
    edg = dh.abs() * (u.abs() * es + slope.abs() * eu + es * eu) + 4 * UNIT * dg.abs()
    edu = dh.abs() * ea + 2 * UNIT * du.abs()
    step = 2.0 ** -25 if half == 2.0 ** -11 else 0.0      # half of fp16's smallest step
    rdg, rdu = edg + half * (dg.abs() + edg) + step, edu + half * (du.abs() + edu) + step       # as they are stored
    out = {"dx": dg @ wg + du @ wu, "dwg": dg.t() @ x, "dwu": du.t() @ x, "dbg": dg.sum(0), "dbu": du.sum(0)}
    root = lambda c, w: 7 * torch.sqrt((c * c) @ (w * w))
    tiny = 1e-30
    out["e_dx"] = root(rdg, wg) + root(rdu, wu) + sum_bound(dg, wg, F) + sum_bound(du, wu, F) + tiny
    out["e_dwg"] = root(rdg.t(), x) + sum_bound(dg.t(), x, M) + tiny
    out["e_dwu"] = root(rdu.t(), x) + sum_bound(du.t(), x, M) + tiny
    for k, d, e in (("dbg", dg, edg), ("dbu", du, edu)):
        out["e_" + k] = 7 * torch.sqrt((e * e).sum(0)) + (M / 4 + 32) * UNIT * d.abs().sum(0) + tiny
    return out
