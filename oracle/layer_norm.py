"""Oracle of the layer norm with a residual: the formula in fp64, its gradients, rows in 8-bit integers, and how far fp32 may be from them.

``s = x + r``, ``c = s - mean s``, ``y = c / sqrt(mean c^2 + eps) * w (+ b)``.  Bounds in units of 2^-24: a row of up to 16384 elements is
summed in chains of at most 32 elements a thread and a tree of 6 + 8 sums, and divided: ``ROW_ULPS`` covers each such sum once, relative to
the sum of its magnitudes.  ``c`` carries the errors of s and of the mean, which do not shrink where the two cancel."""
import torch

UNIT = 2.0 ** -24
ROW_ULPS = 64.0


def _mean(t):
    return t.mean(-1, keepdim=True)


def forward(x, w=None, b=None, residual=None, eps=1e-5):
    """``(y, s, stats, bound on y's error)``; ``stats``: what :func:`backward` takes."""
    s = x.double() if residual is None else x.double() + residual.double()
    mean = _mean(s)
    c = s - mean
    var = _mean(c * c) + eps
    rstd = 1.0 / torch.sqrt(var)
    e_mean = ROW_ULPS * UNIT * _mean(s.abs())
    e_c = e_mean + UNIT * ((s.abs() if residual is not None else 0) + c.abs())
    e_rstd = _mean(c.abs() * e_c) / var + (_mean(e_c * e_c) / var) + ROW_ULPS * UNIT      # relative
    xh = c * rstd
    e = rstd * e_c + xh.abs() * (e_rstd + UNIT)
    y = xh
    if w is not None:
        y, e = y * w.double(), e * w.double().abs()
        e = e + UNIT * y.abs()
    if b is not None:
        y = y + b.double()
        e = e + UNIT * (y.abs() + b.double().abs())
    return y, s, (mean, rstd, e_mean, e_rstd), e


def backward(kept, stats, dy, w=None, dres=None, chain=200):
    """Gradients from what the forward kept: ``dx, dw, db`` and bounds on their errors; ``chain``: sums a column goes through."""
    mean, rstd, e_mean, e_rstd = stats
    kept, dy = kept.double(), dy.double()
    c = kept - mean
    xh = c * rstd
    e_xh = rstd * (e_mean + UNIT * c.abs()) + xh.abs() * (e_rstd + UNIT)
    wdy = dy if w is None else dy * w.double()
    c1, c2 = _mean(wdy), _mean(xh * wdy)
    e1, e2 = ROW_ULPS * UNIT * _mean(wdy.abs()), _mean(wdy.abs() * e_xh) + ROW_ULPS * UNIT * _mean((xh * wdy).abs())
    dx = (wdy - c1 - xh * c2) * rstd
    e = rstd * (e1 + xh.abs() * e2 + c2.abs() * e_xh + 4 * UNIT * (wdy.abs() + c1.abs() + (xh * c2).abs())) + dx.abs() * (e_rstd + UNIT)
    if dres is not None:
        dx = dx + dres.double()
        e = e + UNIT * (dx.abs() + dres.double().abs())
    flat = lambda t: t.reshape(-1, t.shape[-1])
    return {"dx": dx, "e_dx": e, "dw": flat(dy * xh).sum(0), "e_dw": flat(dy.abs() * e_xh).sum(0) + chain * UNIT * flat(dy * xh).abs().sum(0),
            "db": flat(dy).sum(0), "e_db": chain * UNIT * flat(dy).abs().sum(0)}


def rows_int8(y):
    """``(q, scale)`` in y's own type: the nearest whole numbers, halves to even."""
    scale = y.abs().amax(-1).clamp_min(1e-30) / 127
    return torch.round(y / scale[..., None]).to(torch.int8), scale
