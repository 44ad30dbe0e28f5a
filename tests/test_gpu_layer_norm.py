"""GPU: the layer norm with a residual and rows in 8-bit integers against the formula in fp64, element by element (bounds: ``oracle/layer_norm.py``)."""
import pytest
import torch

from oracle import layer_norm as oracle

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


def _inputs(M, N, dtype, rdtype, wdtype, bias, seed=0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    return (r(M, N).to(dtype), None if rdtype is None else (2 * r(M, N) + mean).to(rdtype), None if wdtype is None else (1 + 0.2 * r(N)).to(wdtype),
            r(N).to(wdtype) if bias else None, r(M, N).to(dtype), r(M, N).to(rdtype or dtype))


CASES = [  # M, N, type, residual, weight, bias, mean of the residual
    (1, 1, BF, BF, BF, True, 0.0), (5, 7, HF, FL, HF, True, 3.0), (33, 64, BF, BF, FL, False, 0.0), (70001, 16, BF, BF, BF, True, 0.5),
    (3, 65, FL, FL, FL, True, 1e4), (100, 200, BF, FL, BF, False, 100.0), (9, 512, HF, HF, HF, True, 0.0), (1027, 1000, BF, BF, BF, True, 0.0),
    (10, 1001, HF, FL, HF, True, 0.3), (4100, 2048, BF, BF, BF, True, 0.3), (6, 2050, BF, BF, None, False, 0.0), (2, 4096, FL, None, FL, False, 0.0),
    (1030, 4104, BF, FL, FL, True, 10.0), (3, 8192, BF, None, BF, True, 0.0), (1100, 1800, HF, HF, HF, True, 0.0), (5, 3001, FL, FL, None, False, 0.0),
    (2, 8193, HF, HF, FL, False, 0.0), (1025, 16384, BF, BF, BF, True, 0.0), (3, 16383, FL, FL, FL, True, 1000.0),
]


@pytest.mark.parametrize("M,N,dtype,rdtype,wdtype,bias,mean", CASES)
def test_forward_and_gradients(device, M, N, dtype, rdtype, wdtype, bias, mean):
    from fla_amd.modules import layer_norm
    print(M, N, dtype, rdtype, wdtype, bias, flush=True)
    x, res, w, b, dy, ds = _inputs(M, N, dtype, rdtype, wdtype, bias, N, mean)
    ry, rs, stats, ey = oracle.forward(x, w, b, res)
    put = lambda t: None if t is None else t.to(device).requires_grad_()
    gx, gr, gw, gb = map(put, (x, res, w, b))
    y, s = layer_norm(gx, gw, gb, residual=gr, prenorm=True, eps=1e-5)
    _check("y", y, ry, ey)
    if res is None:
        assert s is gx
    else:
        assert s.dtype == rdtype
        _check("s", s, rs, oracle.UNIT * rs.abs())
    leaves = {k: v for k, v in (("dx", gx), ("dr", gr), ("dw", gw), ("db", gb)) if v is not None}
    grads = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), (dy.to(device), ds.to(device)))))
    want = oracle.backward(s.detach().cpu(), stats, dy, w, ds, chain=200 + M // 1024)
    if res is None:      # autograd adds the two gradients of x after each was rounded
        want["e_dx"] = want["e_dx"] + torch.finfo(dtype).eps * (want["dx"].abs() + ds.double().abs())
    _check("dx", grads["dx"], want["dx"], want["e_dx"])
    if res is not None:
        assert grads["dr"].dtype == rdtype
        _check("dr", grads["dr"], want["dx"], want["e_dx"])
    for k in ("dw", "db"):
        if k in grads:
            _check(k, grads[k], want[k], want["e_" + k])
    with torch.no_grad():
        plain = layer_norm(gx, gw, gb, residual=gr, eps=1e-5)
        both = layer_norm(gx, gw, gb, residual=gr, eps=1e-5, prenorm=True)
        assert torch.equal(plain, y) and torch.equal(both[0], y) and torch.equal(both[1], s)


@pytest.mark.parametrize("M,N", [(3, 1), (40, 64), (500, 1000), (2000, 2048), (300, 4096), (64, 7001), (64, 16384)])
@pytest.mark.parametrize("dtype", [FL, BF, HF])
def test_rows_of_integers(device, M, N, dtype):
    """Bit for bit the fp32 quotients, rounded to the nearest whole number."""
    from fla_amd.modules import quantize_rows
    gen = torch.Generator().manual_seed(M + N)
    x = (torch.randn(M, N, generator=gen) * torch.exp(4 * torch.randn(M, 1, generator=gen) - 3 * torch.rand(M, N, generator=gen))).to(dtype)
    q, scale = quantize_rows(x.to(device), torch.int8)
    rq, rs = oracle.rows_int8(x.float())
    assert q.dtype == torch.int8 and scale.dtype == FL and torch.equal(scale.cpu(), rs) and torch.equal(q.cpu(), rq)


@pytest.mark.parametrize("norm", ["layer_norm", "rms_norm"])
@pytest.mark.parametrize("M,N", [(40, 64), (2000, 2048), (70, 1001), (64, 16384)])
def test_rows_of_the_norm(device, norm, M, N):
    """An fp32 norm's own result, quantised by the formula, is what it gives in 8 bits, of either type."""
    from fla_amd import modules
    norm = getattr(modules, norm)
    gen = torch.Generator().manual_seed(M + N)
    x, r, w, b = (torch.randn(*s, generator=gen).to(device) for s in ((M, N), (M, N), (N,), (N,)))
    with torch.no_grad():
        y = norm(x, w, b, residual=r)
        (q, scale), kept = norm(x, w, b, residual=r, prenorm=True, quantize=torch.int8)
        rq, rs = oracle.rows_int8(y.cpu())
        assert torch.equal(scale.cpu(), rs) and torch.equal(q.cpu(), rq) and torch.equal(kept, x + r)
        q8, s8 = norm(x, w, b, residual=r, quantize=torch.float8_e4m3fn)
        scale = y.cpu().abs().amax(-1).clamp_min(1e-30) / 448      # (on the CPU: on a GPU torch takes a product with 1 / 448)
        want = (y.cpu() / scale[:, None]).to(torch.float8_e4m3fn)
        assert torch.equal(s8.cpu(), scale) and torch.equal(q8.cpu().view(torch.uint8), want.view(torch.uint8))


def test_long_rows_of_integers_and_extremes(device):
    from fla_amd.modules import quantize_rows
    x = torch.randn(5, 16384 + 1003, generator=torch.Generator().manual_seed(1))
    q, s = quantize_rows(x.to(device), torch.int8)
    rq, rs = oracle.rows_int8(x)
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    for N in (40, 20000):
        x = torch.zeros(6, N)
        x[1] = 1e-38
        x[2] = 3e38
        x[3, 5] = float("nan")
        x[4, 7] = float("inf")
        q, s = (t.cpu() for t in quantize_rows(x.to(device), torch.int8))
        assert not q[0].any() and s[0] == torch.tensor(1e-30) / 127 and not q[1].any() and (q[2] == 127).all()
        assert s[3].isnan() and not q[3].any() and s[4] == float("inf") and not q[4].any() and not q[5].any()


def test_infinite_rows_stay_in_their_row(device):
    from fla_amd.modules import layer_norm
    x = torch.randn(9, 72, generator=torch.Generator().manual_seed(2))
    bad = x.clone()
    bad[4, 3] = float("inf")
    y, ybad = (layer_norm(t.to(device), None) for t in (x, bad))
    assert ybad[4].isnan().all() and torch.equal(ybad[:4], y[:4]) and torch.equal(ybad[5:], y[5:])


def test_addresses_and_strides(device):
    """Rows at odd addresses, columns of a wider tensor, broadcast rows and their gradient, more than two dimensions."""
    from fla_amd.modules import layer_norm
    gen = torch.Generator().manual_seed(3)
    base = torch.randn(1 + 6 * 64, generator=gen).bfloat16()
    w = torch.randn(1 + 64, generator=gen).bfloat16()
    g, gw = base.to(device), w.to(device)
    ry, _, _, ey = oracle.forward(base[1:].view(2, 3, 64), w[1:])
    _check("odd address", layer_norm(g[1:].view(2, 3, 64), gw[1:], eps=1e-5), ry, ey)
    x = base[:384].view(3, 128)[:, 16:80]
    ry, _, _, ey = oracle.forward(x, w[:64], None, x)
    gx = g[:384].view(3, 128)[:, 16:80]
    _check("columns", layer_norm(gx, gw[:64], residual=gx, eps=1e-5), ry, ey)
    leaf = torch.randn(64, generator=gen).to(device).requires_grad_()
    dy = torch.randn(4, 64, generator=gen)
    ry, _, stats, ey = oracle.forward(leaf.detach().cpu().expand(4, 64))
    y = layer_norm(leaf.expand(4, 64), None, eps=1e-5)
    _check("broadcast", y, ry, ey)
    want = oracle.backward(leaf.detach().cpu().expand(4, 64), stats, dy)
    _check("its gradient", torch.autograd.grad(y, leaf, dy.to(device))[0], want["dx"].sum(0),
           want["e_dx"].sum(0) + 4 * oracle.UNIT * want["dx"].abs().sum(0))


def test_frozen_leaves_and_absent_gradients(device):
    """Each subset of leaves, and each output's gradient alone."""
    from fla_amd.modules import layer_norm
    gen = torch.Generator().manual_seed(4)
    full = [torch.randn(*s, generator=gen).to(device) for s in ((6, 40), (6, 40), (40,), (40,))]
    cot = [torch.randn(6, 40, generator=gen).to(device) for _ in range(2)]
    for which in range(3):
        pick = lambda both: [t for i, t in enumerate(both) if which in (i, 2)]
        every = [t.clone().requires_grad_() for t in full]
        ref = torch.autograd.grad(pick(layer_norm(every[0], every[2], every[3], residual=every[1], prenorm=True)), every, pick(cot), allow_unused=True)
        for i in range(4):
            if ref[i] is None:
                continue
            some = [t.clone().requires_grad_(i == j) for j, t in enumerate(full)]
            out = pick(layer_norm(some[0], some[2], some[3], residual=some[1], prenorm=True))
            if which == 1 and i > 1:
                continue
            (got,) = torch.autograd.grad(out, some[i], pick(cot))
            assert torch.equal(got, ref[i]), (which, i)


def test_module_and_what_it_refuses(device):
    from fla_amd.modules import LayerNorm, layer_norm
    m = LayerNorm(48, bias=True).to(device)
    x = torch.randn(3, 5, 48, device=device)
    for kind in (True, torch.int8):
        with pytest.raises(RuntimeError, match="no gradient"):
            m(x, quantize=kind)
    with torch.no_grad():
        (q, s), kept = m(x, residual=x, prenorm=True, quantize=torch.int8)
    assert q.shape == x.shape and s.shape == (3, 5) and torch.equal(kept, x + x)
    y, kept = m(x.bfloat16(), prenorm=True, residual_in_fp32=True)
    assert kept.dtype == FL and torch.equal(kept, x.bfloat16().float()) and y.dtype == BF
    (y.float().sum() + kept.sum()).backward()
    assert m.weight.grad.shape == (48,) and torch.equal(m.bias.grad, torch.full((48,), 15.0, device=device))
    empty = torch.zeros(0, 48, device=device, requires_grad=True)
    y, kept = layer_norm(empty, m.weight, residual=empty, prenorm=True)
    gx, gw = torch.autograd.grad(y.sum() + kept.sum(), (empty, m.weight))
    assert gx.shape == (0, 48) and not gw.any()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        layer_norm(fwAD.make_dual(x, x), m.weight)
