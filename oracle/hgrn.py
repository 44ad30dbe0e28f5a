"""Oracle of the elementwise gated recurrence: the formula token by token in fp64, its gradients, and how far an evaluation in
fp32 may be from them.

``h_t = a_t h_{t-1} + u_t`` with ``a = exp(g)``, ``u = x``, or from pre-activations ``a = lb + (1-lb) s(f)``, ``u = (1-a) i s(i)``.

Error bounds.  Let one step in fp32 have a relative error of at most ``c`` units of 2^-24 in the decay, the input and the
update together (``STEP_ULPS``).  Then ``e_t <= a_t e_{t-1} + c 2^-24 S_t``, where ``S`` is the same recurrence on magnitudes; joining
runs of steps in another order multiplies decays of at most these errors, which the recurrence for ``e`` counts already.
"""
import torch

# exp (hardware, 1 ulp = 2 units, its argument's product 1 + the argument itself, at most 4 in the tests), sigmoid (exp, sum,
# reciprocal: 6) and the products of the gated input (two sigmoids, four products: 18), the update (2): 32 covers each of them.
STEP_ULPS = 32.0
UNIT = 2.0 ** -24


def operands(x, g, lower_bound=None, gates=False):
    x, g = x.double(), g.double()
    if not gates:
        return torch.exp(g), x
    lb = 0.0 if lower_bound is None else lower_bound.double()
    return lb + (1 - lb) * torch.sigmoid(g), (1 - lb) * torch.sigmoid(-g) * x * torch.sigmoid(x)


def spans(x, offsets=None):
    """(batch row, begin, end) of every sequence."""
    if offsets is None:
        return [(b, 0, x.shape[1]) for b in range(x.shape[0])]
    offs = [int(v) for v in offsets]
    return [(0, lo, hi) for lo, hi in zip(offs[:-1], offs[1:])]


def scan(a, u, h0, seqs):
    """``(h, before, ht)`` in fp64, differentiable: ``before`` is the state ahead of each token; rows of no sequence are 0."""
    h, before, ht = torch.zeros_like(u), torch.zeros_like(u), []
    for n, (b, lo, hi) in enumerate(seqs):
        c = u.new_zeros(u.shape[-1]) if h0 is None else h0[n].double()
        hs, bs = [], []
        for t in range(lo, hi):
            bs.append(c)
            c = a[b, t] * c + u[b, t]
            hs.append(c)
        if hs:
            h = h.index_put((torch.tensor(b), torch.arange(lo, hi)), torch.stack(hs))
            before = before.index_put((torch.tensor(b), torch.arange(lo, hi)), torch.stack(bs))
        ht.append(c)
    return h, before, torch.stack(ht)


def forward(x, g, h0=None, offsets=None, lower_bound=None, gates=False):
    """``(o, ht, bound on o's error in fp32, bound on ht's)``."""
    a, u = operands(x, g, lower_bound, gates)
    seqs = spans(x, offsets)
    h, _, ht = scan(a, u, h0, seqs)
    S, _, St = scan(a, u.abs(), None if h0 is None else h0.abs(), seqs)
    e, _, et = scan(a, S, None, seqs)
    return h, ht, STEP_ULPS * UNIT * e, STEP_ULPS * UNIT * (et + St)


def backward(x, g, do, dht=None, h0=None, offsets=None, lower_bound=None, gates=False):
    """Gradients in fp64 by the formula: dict of ``dx, dg, dh0, dlb`` and of the bounds on their errors in fp32, ``e_...``."""
    a, u = operands(x, g, lower_bound, gates)
    seqs = spans(x, offsets)
    _, before, _ = scan(a, u, h0, seqs)
    S, Sb, _ = scan(a, u.abs(), None if h0 is None else h0.abs(), seqs)
    _, eb, _ = scan(a, S, None, seqs)
    eb = STEP_ULPS * UNIT * (eb + Sb)
    lam, el, mag = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(u)
    dh0, e0 = [], []
    for n, (b, lo, hi) in enumerate(seqs):
        m = u.new_zeros(u.shape[-1]) if dht is None else dht[n].double()
        mm, em = m.abs(), torch.zeros_like(m)
        for t in range(hi - 1, lo - 1, -1):
            lam[b, t] = do[b, t].double() + m
            mag[b, t] = do[b, t].double().abs() + mm
            el[b, t] = em + STEP_ULPS * UNIT * mag[b, t]
            m, mm, em = a[b, t] * lam[b, t], a[b, t] * mag[b, t], a[b, t] * el[b, t]
        dh0.append(m)
        e0.append(em)
    out = {"dh0": torch.stack(dh0), "e_dh0": torch.stack(e0) + UNIT * torch.stack(dh0).abs()}
    c = STEP_ULPS * UNIT
    if not gates:
        dg = lam * before * a
        return dict(out, dx=lam, e_dx=el, dg=dg, e_dg=a * (mag * eb + before.abs() * el + c * Sb * mag))
    x, g = x.double(), g.double()
    lb = torch.zeros(x.shape[-1], dtype=torch.float64) if lower_bound is None else lower_bound.double()
    s, rest, si = torch.sigmoid(g), torch.sigmoid(-g), torch.sigmoid(x)
    z = x * si
    da = lam * (before - z)
    e_da = mag * (eb + c * (z.abs() + Sb)) + (before - z).abs() * el
    slope = si * (1 + x * (1 - si))
    w = (1 - lb) * rest
    inside = torch.zeros_like(u)
    for b, lo, hi in seqs:
        inside[b, lo:hi] = 1
    dlb = inside * da * rest
    n = inside.sum()
    return dict(out, dx=lam * w * slope, e_dx=w * (el * slope.abs() + c * mag * si * (1 + x.abs())), dg=inside * da * w * s,
                e_dg=w * s * (e_da + c * da.abs()), dlb=dlb.sum((0, 1)),
                e_dlb=(rest * (e_da + c * da.abs())).sum((0, 1)) + n * UNIT * dlb.abs().sum((0, 1)))
