"""Oracle of the RMS norm with a residual: the formula in fp64, its gradients, rows in 8 bits, and how far fp32 may be from them.

``s = x + r``, ``y = s / sqrt(mean s^2 + eps) * w (+ b)``.  Bounds in units of 2^-24: a row of up to 16384 elements is summed in
chains of at most 32 products a thread and a tree of 6 + 8 sums, the root, the division and the sum with eps take 6 more, so ``rstd``
is off by at most half of 46 + 6 relative, and ``y`` by two roundings more: ``ROW_ULPS`` covers each of these sums once."""
import torch

UNIT = 2.0 ** -24
ROW_ULPS = 64.0


def forward(x, w=None, b=None, residual=None, eps=1e-5):
    """``(y, s, rstd, bound on y's error)``."""
    s = x.double() if residual is None else x.double() + residual.double()
    rstd = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    y = s * rstd
    if w is not None:
        y = y * w.double()
    e = ROW_ULPS * UNIT * y.abs()
    if b is not None:
        y = y + b.double()
        e = e + UNIT * (y.abs() + b.double().abs())
    return y, s, rstd, e


def backward(kept, rstd, dy, w=None, dres=None, chain=200):
    """Gradients from what the forward kept: ``dx, dw, db`` and bounds on their errors; ``chain``: sums a column goes through."""
    kept, dy = kept.double(), dy.double()
    xh = kept * rstd
    wdy = dy if w is None else dy * w.double()
    c = (xh * wdy).mean(-1, keepdim=True)
    dx = (wdy - xh * c) * rstd
    e = ROW_ULPS * UNIT * rstd * (wdy.abs() + xh.abs() * (xh * wdy).abs().mean(-1, keepdim=True))
    if dres is not None:
        dx = dx + dres.double()
        e = e + UNIT * (dx.abs() + dres.double().abs())
    flat = lambda t: t.reshape(-1, t.shape[-1])
    return {"dx": dx, "e_dx": e, "dw": flat(dy * xh).sum(0), "e_dw": (ROW_ULPS + chain) * UNIT * flat(dy * xh).abs().sum(0),
            "db": flat(dy).sum(0), "e_db": chain * UNIT * flat(dy).abs().sum(0)}


def scale_of(y):
    return y.abs().amax(-1).clamp_min(1e-30) / 448.0
