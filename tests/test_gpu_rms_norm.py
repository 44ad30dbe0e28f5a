"""GPU: the RMS norm with a residual and its 8-bit rows against the formula in fp64, element by element (bounds: ``oracle/rms_norm.py``)."""
import pytest
import torch

from oracle import rms_norm as oracle

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def _check(name, out, ref, bound):
    assert out is not None and tuple(out.shape) == tuple(ref.shape), name
    got = out.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    half = torch.finfo(out.dtype).eps / 2
    tiny = 2.0 ** -25 if out.dtype == HF else 2.0 ** -126
    over = ((got - ref).abs() / (half * (ref.abs() + bound) + bound + tiny)).max().item() if ref.numel() else 0.0
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, f"{name}: {over:.3f} of the bound"


def _inputs(M, N, dtype, rdtype, wdtype, bias, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    return (r(M, N).to(dtype), None if rdtype is None else (2 * r(M, N)).to(rdtype), None if wdtype is None else (1 + 0.2 * r(N)).to(wdtype),
            r(N).to(wdtype) if bias else None, r(M, N).to(dtype), r(M, N).to(rdtype or dtype))


CASES = [  # M, N, type, residual, weight, bias
    (1, 1, BF, BF, BF, False), (5, 7, HF, FL, HF, True), (33, 64, BF, BF, FL, False), (70001, 16, BF, BF, BF, True),
    (3, 65, FL, FL, FL, True), (100, 200, BF, FL, BF, False), (9, 512, HF, HF, HF, False), (1027, 1000, BF, BF, BF, False),
    (10, 1001, HF, FL, HF, True), (4100, 2048, BF, BF, BF, False), (6, 2050, BF, BF, None, False), (2, 4096, FL, None, FL, False),
    (1030, 4104, BF, FL, FL, True), (3, 8192, BF, None, BF, True), (1100, 1800, HF, HF, HF, True), (7, 777, BF, FL, BF, False), (5, 3001, FL, FL, None, False), (2, 8193, HF, HF, FL, False), (1025, 16384, BF, BF, BF, False),
    (3, 16383, FL, FL, FL, True), (1100, 3000, BF, FL, BF, True),
]


@pytest.mark.parametrize("M,N,dtype,rdtype,wdtype,bias", CASES)
def test_forward_and_gradients(device, M, N, dtype, rdtype, wdtype, bias):
    from fla_amd.modules import rms_norm
    print(M, N, dtype, rdtype, wdtype, bias, flush=True)
    x, res, w, b, dy, ds = _inputs(M, N, dtype, rdtype, wdtype, bias, seed=N)
    ry, rs, rstd, ey = oracle.forward(x, w, b, res)
    put = lambda t: None if t is None else t.to(device).requires_grad_()
    gx, gr, gw, gb = map(put, (x, res, w, b))
    y, s = rms_norm(gx, gw, gb, residual=gr, prenorm=True, eps=1e-5)
    _check("y", y, ry, ey)
    if res is None:
        assert s is gx
    else:
        assert s.dtype == rdtype
        _check("s", s, rs, oracle.UNIT * rs.abs())
    leaves = {k: v for k, v in (("dx", gx), ("dr", gr), ("dw", gw), ("db", gb)) if v is not None}
    grads = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), (dy.to(device), ds.to(device)))))
    want = oracle.backward(s.detach().cpu(), rstd, dy, w, ds, chain=200 + M // 1024)
    if res is None:      # autograd adds the two gradients of x after each was rounded
        want["e_dx"] = want["e_dx"] + torch.finfo(dtype).eps * (want["dx"].abs() + ds.double().abs())
    _check("dx", grads["dx"], want["dx"], want["e_dx"])
    if res is not None:
        assert grads["dr"].dtype == rdtype
        _check("dr", grads["dr"], want["dx"], want["e_dx"])
    for k in ("dw", "db"):
        if k in grads:
            _check(k, grads[k], want[k], want["e_" + k])
    # without the sum, without gradients: the same rows
    assert torch.equal(rms_norm(gx, gw, gb, residual=gr, eps=1e-5), y)
    with torch.no_grad():
        plain = rms_norm(gx, gw, gb, residual=gr, eps=1e-5)
        both = rms_norm(gx, gw, gb, residual=gr, eps=1e-5, prenorm=True)
        assert torch.equal(plain, y) and torch.equal(both[0], y) and torch.equal(both[1], s)


@pytest.mark.parametrize("M,N,dtype,rdtype,wdtype,bias", CASES)
def test_eight_bits(device, M, N, dtype, rdtype, wdtype, bias):
    from fla_amd.modules import quantize_rows, rms_norm
    x, res, w, b, _, _ = _inputs(M, N, dtype, rdtype, wdtype, bias, seed=N + 1)
    ry, rs, _, ey = oracle.forward(x, w, b, res)
    put = lambda t: None if t is None else t.to(device)
    (q, scale), s = rms_norm(put(x), put(w), put(b), residual=put(res), prenorm=True, eps=1e-5, quantize=True)
    (q0, s0) = quantize_rows(put(x))
    for name, got, sc, ref, e in (("norm", q, scale, ry, ey), ("rows", q0, s0, x.double(), torch.zeros(M, N, dtype=torch.float64))):
        assert got.dtype == torch.float8_e4m3fn and got.shape == x.shape and sc.shape == x.shape[:-1] and sc.dtype == FL
        want = oracle.scale_of(ref)
        e_scale = 4 * oracle.UNIT * want + e.amax(-1) / 448
        assert ((sc.double().cpu() - want).abs() <= e_scale).all(), name
        unit = want[:, None]
        # half a step of the 8-bit type: 2^-4 of the value, 2^-10 below its normal numbers; the scale's error moves the value too
        room = (ref.abs() * 2.0 ** -4).clamp_min(unit * 2.0 ** -10) * (1 + 2.0 ** -18) + 2 * e + 8 * oracle.UNIT * ref.abs()
        off = (got.double().cpu() * sc.double().cpu()[:, None] - ref).abs()
        assert (off <= room).all(), (name, (off / room).max())
        assert (got.double().abs().amax(-1).cpu() == 448).all()
    if res is not None:
        _check("s", s, rs, oracle.UNIT * rs.abs())


def test_rows_of_zeros_and_extremes(device):
    from fla_amd.modules import quantize_rows, rms_norm
    x = torch.zeros(6, 40)
    x[1] = 1e-38
    x[2] = 3e38
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    q, s = quantize_rows(x.to(device))
    q, s = q.float().cpu(), s.cpu()
    assert not q[0].any() and s[0] == torch.tensor(1e-30) / 448
    assert q[1].abs().max() < 1e-2 and torch.isfinite(q[2]).all() and (q[2] == 448).all()
    assert q[3, 5].isnan() and not q[3, :5].any() and q[4, 7].isnan() and s[4] == float("inf") and not q[4, :7].any()
    assert not q[5].any()
    y = rms_norm(x[:1].to(device), torch.ones(40, device=device))
    assert not y.any()


def test_addresses_and_strides(device):
    """Rows at odd addresses, columns of a wider tensor, broadcast rows, more than two dimensions."""
    from fla_amd.modules import rms_norm
    gen = torch.Generator().manual_seed(3)
    base = torch.randn(1 + 6 * 64, generator=gen).bfloat16()
    w = torch.randn(1 + 64, generator=gen).bfloat16()
    g, gw = base.to(device), w.to(device)
    ry, _, _, ey = oracle.forward(base[1:].view(2, 3, 64), w[1:])
    _check("odd address", rms_norm(g[1:].view(2, 3, 64), gw[1:], eps=1e-5), ry, ey)
    x = base[:384].view(3, 128)[:, 16:80]
    ry, _, _, ey = oracle.forward(x, w[:64], None, x)
    gx = g[:384].view(3, 128)[:, 16:80]
    _check("columns", rms_norm(gx, gw[:64], residual=gx, eps=1e-5), ry, ey)
    one = base[:64].expand(4, 64)
    ry, _, _, ey = oracle.forward(one, None)
    _check("broadcast", rms_norm(g[:64].expand(4, 64), None, eps=1e-5), ry, ey)
    _check("one row", rms_norm(g[:64], None, eps=1e-5), ry[0], ey[0])


def test_module_and_what_it_refuses(device):
    from fla_amd.modules import RMSNorm, rms_norm
    m = RMSNorm(48, bias=True).to(device)
    x = torch.randn(3, 5, 48, device=device)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(x, quantize=True)
    with torch.no_grad():
        (q, s), kept = m(x, residual=x, prenorm=True, quantize=True)
    assert q.shape == x.shape and s.shape == (3, 5) and torch.equal(kept, x + x)
    y, kept = m(x.bfloat16(), prenorm=True, residual_in_fp32=True)
    assert kept.dtype == FL and torch.equal(kept, x.bfloat16().float()) and y.dtype == BF
    (y.float().sum() + kept.sum()).backward()
    assert m.weight.grad.shape == (48,) and torch.equal(m.bias.grad, torch.full((48,), 15.0, device=device))
    empty = torch.zeros(0, 48, device=device, requires_grad=True)
    y, kept = rms_norm(empty, m.weight, residual=empty, prenorm=True)
    gx, gw = torch.autograd.grad(y.sum() + kept.sum(), (empty, m.weight))
    assert gx.shape == (0, 48) and not gw.any()
    with torch.no_grad():
        q, s = rms_norm(empty, None, quantize=True)
    assert q.shape == (0, 48) and s.shape == (0,)


def test_against_differences(device):
    """Slopes along a direction from the gradients and from central differences of the kernel's own forward in fp32: a step of 2^-6
    leaves 2^-12 of the third derivative (below one here, of values of about one) and 2^-24 * 64 * sqrt(37 * 100) / 2^-6 of rounding."""
    from fla_amd.modules import rms_norm
    x, res, w, b, dy, ds = [t.to(device) for t in _inputs(37, 100, FL, FL, FL, True)]
    leaves = [t.requires_grad_() for t in (x, res, w, b)]

    def loss(x, res, w, b):
        y, s = rms_norm(x, w, b, residual=res, prenorm=True, eps=1e-5)
        return (y.double() * dy).sum() + (s.double() * ds).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    gen = torch.Generator(device=device).manual_seed(1)
    e = 2.0 ** -6
    with torch.no_grad():
        for i, leaf in enumerate(leaves):
            d = torch.randn(leaf.shape, generator=gen, device=device)
            at = lambda k: loss(*[t + k * d if j == i else t for j, t in enumerate(leaves)])
            slope, want = ((at(e) - at(-e)) / (2 * e)).item(), (grads[i].double() * d).sum().item()
            print(i, slope, want, flush=True)
            assert abs(slope - want) <= 0.03 + 2.0 ** -12 * (37 * 100) ** 0.5 + 1e-3 * abs(want)


def test_captured_and_other_streams(device):
    from fla_amd.modules import rms_norm
    x, res, w, _, dy, ds = [None if t is None else t.to(device) for t in _inputs(300, 4096, BF, BF, BF, False)]
    leaves = [t.requires_grad_() for t in (x, res, w)]

    def train():
        y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1], prenorm=True)
        return [y, s, *torch.autograd.grad((y, s), leaves, (dy, ds))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = train()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, train()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)))
        want = train()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), k


def test_more_rows_than_a_launch_takes(device):
    from fla_amd.modules import rms_norm
    M, N = (1 << 22) + 5, 8
    gen = torch.Generator(device=device).manual_seed(1)
    x, r = torch.randn(M, N, generator=gen, device=device).bfloat16(), torch.randn(M, N, generator=gen, device=device)
    w = torch.randn(N, generator=gen, device=device)
    with torch.no_grad():
        (q, scale), s = rms_norm(x, w, None, r, prenorm=True, quantize=True)
        y, _ = rms_norm(x, w, None, r, prenorm=True)
        for rows in (slice(0, 40), slice(M - 45, M)):
            (q1, scale1), s1 = rms_norm(x[rows], w, None, r[rows], prenorm=True, quantize=True)
            assert torch.equal(q[rows].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(scale[rows], scale1) and torch.equal(s[rows], s1)
            assert torch.equal(y[rows], rms_norm(x[rows], w, None, r[rows]))
    x, r = x.requires_grad_(), r.requires_grad_()
    dy = torch.randn(M, N, generator=gen, device=device).bfloat16()
    dx, dr = torch.autograd.grad(rms_norm(x, w, None, r), (x, r), dy)
    rows = slice(M - 45, M)
    a, b = x[rows].detach().requires_grad_(), r[rows].detach().requires_grad_()
    da, db = torch.autograd.grad(rms_norm(a, w, None, b), (a, b), dy[rows])
    assert torch.equal(dx[rows], da) and torch.equal(dr[rows], db)


def test_one_tensor_twice(device):
    from fla_amd.modules import rms_norm
    x = torch.randn(7, 264, generator=torch.Generator().manual_seed(2)).to(device).requires_grad_()
    y, s = rms_norm(x, None, None, x, prenorm=True)
    got, = torch.autograd.grad((y.square().sum() + s.sum()), x)
    z = x.detach().double().requires_grad_()
    t = 2 * z
    want, = torch.autograd.grad((t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)).square().sum() + t.sum(), z)
    # The sum of y^2 is N up to eps, so its gradient (dy - y mean(dy y)) rstd is a difference of two equal terms of at most 2 * 5 * 0.6.  Each is off by
    # less than 16 roundings of fp32 (the mean's sum in 3 + 6 levels, rstd, products), both twice (x and residual): 4 * 6 * 16 * 2^-24.  The rest is 2.
    assert (got.double() - want).abs().max() <= 4 * 6 * 16 * 2.0 ** -24 + 2.0 ** -22
