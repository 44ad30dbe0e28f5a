"""GPU: the product of 8-bit rows and its epilogue against fp64, element by element.

Bound of a sum of e4m3 products.  The matrix instruction aligns eight products (consecutive k) to the largest of them and cuts each, towards
zero, at 2^-13 of the largest one's power of two: seen with two products 2^E and 2^(E-s) in one such group, of which the second is whole
in the sum up to s = 13 and gone from s = 14 on, for either sign, and in different groups whole at every s.  A cut error therefore has its product's sign and is below
u = 2^-13 2^E.  With operands of random signs these errors are independent and symmetric, and by Hoeffding's inequality their sum exceeds
t = 7 sqrt(sum u^2) with a probability below 2 exp(-t^2 / (2 sum u^2)) = 5e-11: 2e-3 over all 4e7 elements of this file.  The sums of groups
are in fp32 (K / 8 roundings of at most 2^-24 of sum |x w|); scaling, bias, activation and residual add a few units of fp32, the
activations being of slope 1.13 at most; the result is rounded to its type."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

BF, HF, FL, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
ACTS = {None: lambda v: v, "silu": F.silu, "gelu": F.gelu, "relu": F.relu}


def _rows(M, K, gen, std=1.0):
    x = torch.randn(M, K, generator=gen) * std
    scale = x.abs().amax(-1).clamp_min(1e-30) / 448
    return (x / scale[:, None]).to(F8), scale


def _reference(x, w, bias, act, res, device="cpu"):
    xd, wd = [r[0].to(device).double() * r[1].to(device).double()[:, None] for r in (x, w)]
    y, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    # sum of the squares of the groups' largest powers of two, the rows' scales apart
    power = lambda q: torch.where(q == 0, 0.0, torch.ldexp(torch.ones_like(q), torch.frexp(q).exponent - 1))
    px, pw = power(x[0].to(device).float()), power(w[0].to(device).float())
    sq = torch.zeros(px.shape[0], pw.shape[0], device=device)
    for g in range(0, px.shape[1], 8):
        top = torch.zeros_like(sq)
        for k in range(g, g + 8):
            torch.maximum(top, px[:, k, None] * pw[None, :, k], out=top)
        sq += 8 * top * top
    unit = x[1].to(device).double()[:, None] * w[1].to(device).double()
    e = 7 * 2.0 ** -13 * sq.double().sqrt() * unit + (px.shape[1] / 8 + 4) * 2.0 ** -24 * mag
    put = lambda t: t.to(device).double()
    if bias is not None:
        y = y + put(bias)
    y0, y = y, ACTS[act](y)
    e = 1.13 * (e + 2.0 ** -22 * y0.abs()) + 2.0 ** -20 * y.abs()
    if res is not None:
        y = y + put(res)
    return y.cpu(), (e + 2.0 ** -23 * y.abs()).cpu()


def _check(name, out, ref, e):
    assert tuple(out.shape) == tuple(ref.shape)
    got, half = out.double().cpu(), torch.finfo(out.dtype).eps / 2
    assert torch.isfinite(got).all(), name
    over = ((got - ref).abs() / (half * (ref.abs() + e) + e + 2.0 ** -25)).max().item()
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, f"{name}: {over:.3f} of the bound"


CASES = [  # M, N, K, type, bias, activation, residual
    (1, 1, 16, BF, None, None, None), (1, 256, 2048, BF, BF, None, BF), (1, 100, 144, HF, FL, "silu", FL), (3, 130, 112, BF, BF, "gelu", None),
    (16, 64, 128, HF, None, "relu", HF), (17, 72, 272, BF, BF, None, BF), (33, 48, 1040, BF, FL, "silu", FL), (48, 200, 4096, HF, HF, None, HF),
    (64, 17, 240, BF, BF, "gelu", BF), (65, 64, 128, BF, None, None, None), (65, 70, 144, HF, HF, "silu", FL), (100, 129, 656, BF, BF, None, BF),
    (250, 1000, 528, BF, BF, "gelu", BF), (1400, 1411, 272, HF, FL, "relu", HF), (3500, 4000, 384, BF, BF, "silu", BF), (3601, 3333, 208, HF, None, None, FL),
    (130, 65, 16, BF, None, None, None), (70, 130, 4112, BF, BF, "silu", FL), (60, 258, 6400, HF, None, "gelu", HF), (300, 2050, 400, BF, FL, None, BF),
    (2000, 2040, 128, BF, BF, None, None),
    # panels of four waves, tiles for few rows, slices of K, tiles of three slices and more
    (5, 4100, 1040, BF, BF, "silu", BF), (20, 4112, 272, HF, None, None, FL), (45, 4200, 144, BF, FL, "relu", None), (64, 4099, 1168, BF, BF, None, BF),
    (64, 12300, 1040, BF, None, None, BF), (100, 256, 6288, HF, HF, "silu", HF), (1100, 2100, 400, BF, BF, "gelu", BF),
]


@pytest.mark.parametrize("M,N,K,dtype,bias,act,res", CASES)
def test_product(device, M, N, K, dtype, bias, act, res):
    from fla_amd.modules import quant_linear
    print(M, N, K, dtype, bias, act, res, flush=True)
    gen = torch.Generator().manual_seed(M + N + K)
    x, w = _rows(M, K, gen), _rows(N, K, gen, K ** -0.5)
    b = None if bias is None else torch.randn(N, generator=gen).to(bias)
    r = None if res is None else torch.randn(M, N, generator=gen).to(res)
    ref, e = _reference(x, w, b, act, r, device)
    put = lambda t: None if t is None else t.to(device)
    args = ([put(t) for t in x], [put(t) for t in w], put(b), act, put(r), dtype)
    y = quant_linear(*args)
    assert y.dtype == dtype
    _check("y", y, ref, e)
    assert torch.equal(y, quant_linear(*args))


def test_every_element_is_where_it_belongs(device):
    """Small whole numbers, whose sums are exact: no tolerance at all, at tiles' borders and beyond."""
    from fla_amd.modules import quant_linear
    gen = torch.Generator().manual_seed(0)
    for M, N, K in ((7, 33, 64), (40, 90, 400), (200, 300, 160), (1300, 1500, 96), (3700, 3400, 144)):
        x, w = torch.randint(-2, 3, (M, K), generator=gen).float(), torch.randint(-1, 2, (N, K), generator=gen).float()
        x[:, K // 2:] = 0
        x[:, K - 1] = torch.arange(M) % 3
        want = (x @ w.t()).clamp(-256, 256)
        y = quant_linear((x.to(F8).to(device), torch.ones(M, device=device)), (w.to(F8).to(device), torch.ones(N, device=device)))
        print(M, N, K, flush=True)
        assert torch.equal(y.float().cpu().clamp(-256, 256), want)


def test_not_a_number_stays_in_its_row(device):
    """A row of x that is not a number, and none of its neighbours: K ends inside a slice and the rows behind it are valid data."""
    from fla_amd.modules import quant_linear
    gen = torch.Generator().manual_seed(0)
    for M in (20, 300, 3700):
        (x, sx), (w, sw) = _rows(M, 80, gen), _rows(3400, 80, gen)
        want = quant_linear((x.to(device), sx.to(device)), (w.to(device), sw.to(device)))
        bad = x.clone().view(torch.uint8)
        bad[11] = 0x7f
        y = quant_linear((bad.view(F8).to(device), sx.to(device)), (w.to(device), sw.to(device)))
        assert y[11].isnan().all()
        keep = torch.arange(M) != 11
        assert torch.equal(y[keep], want[keep])


def test_shapes_addresses_and_refusals(device):
    from fla_amd.modules import QuantLinear, quant_linear, quantize_rows
    gen = torch.Generator().manual_seed(0)
    x, w = _rows(6, 48, gen), _rows(10, 48, gen)
    ref, e = _reference(x, w, None, None, None)
    gx, gw = [t.to(device) for t in x], [t.to(device) for t in w]
    y = quant_linear((gx[0].view(2, 3, 48), gx[1].view(2, 3)), gw)
    _check("three dimensions", y, ref.view(2, 3, 10), e.view(2, 3, 10))
    _check("one row", quant_linear((gx[0][2], gx[1][2]), gw), ref[2], e[2])
    odd = torch.zeros(6 * 48 + 1, dtype=torch.uint8, device=device)
    odd[1:] = gx[0].view(torch.uint8).flatten()
    _check("odd address", quant_linear((odd[1:].view(F8).view(6, 48), gx[1]), gw), ref, e)
    wide = torch.zeros(6, 96, dtype=torch.uint8, device=device)
    wide[:, 16:64] = gx[0].view(torch.uint8)
    _check("columns", quant_linear((wide.view(F8)[:, 16:64], gx[1]), gw), ref, e)
    assert quant_linear((gx[0][:0], gx[1][:0]), gw).shape == (0, 10)
    with pytest.raises(RuntimeError, match="no gradient"):
        quant_linear(gx, gw, torch.zeros(10, device=device, requires_grad=True))
    # the layer, from a torch.nn.Linear
    lin = torch.nn.Linear(48, 10).to(device, BF)
    layer = QuantLinear.from_linear(lin, activation="silu")
    assert "QuantLinear(48, 10, bias=True, activation=silu)" == repr(layer) and set(layer.state_dict()) == {"weight", "weight_scale", "bias"}
    h = torch.randn(4, 48, generator=gen).to(BF).to(device)
    q, s = quantize_rows(h)
    wq, ws = quantize_rows(lin.weight.detach())
    ref, e = _reference((q.cpu(), s.cpu()), (wq.cpu(), ws.cpu()), lin.bias.detach().cpu(), "silu", h[:, :10].cpu())
    out = layer(h, residual=h[:, :10])
    assert out.dtype == BF
    _check("layer", out, ref, e)
    assert torch.equal(layer((q, s), residual=h[:, :10]), out)
    other = QuantLinear(48, 10, activation="silu", device=device)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(h, residual=h[:, :10]), out)
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(h.requires_grad_())


def test_captured_and_two_streams(device):
    from fla_amd.modules import quant_linear
    gen = torch.Generator().manual_seed(0)
    for M, N, K in ((1, 2048, 2048), (48, 512, 4096), (600, 700, 256)):
        x, w = [[t.to(device) for t in _rows(n, K, gen)] for n in (M, N)]
        res = torch.randn(M, N, generator=gen).to(BF).to(device)
        quant_linear(x, w, residual=res)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = quant_linear(x, w, residual=res)
        side = torch.cuda.Stream()
        for k in range(3):
            x[1].copy_(torch.rand(M, generator=gen))
            want = quant_linear(x, w, residual=res)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                other = quant_linear(x, w, residual=res)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(other, want), (M, k)


def test_module_in_another_type(device):
    """module.to(dtype) is for the bias alone"""
    from fla_amd.modules import QuantLinear
    layer = QuantLinear.from_linear(torch.nn.Linear(64, 48).to(device))
    weight, scale = layer.weight.clone(), layer.weight_scale.clone()
    layer = torch.nn.Sequential(layer).half()[0]
    assert layer.bias.dtype == HF and layer.weight.dtype == F8 and layer.weight_scale.dtype == FL
    assert torch.equal(layer.weight.view(torch.uint8), weight.view(torch.uint8)) and torch.equal(layer.weight_scale, scale)
    assert layer(torch.randn(3, 64, device=device)).shape == (3, 48)
    assert layer.cpu().weight.device.type == "cpu" and layer.weight.dtype == F8
