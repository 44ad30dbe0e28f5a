"""GPU: products of rows in 8-bit integers, plain and gated, and their epilogues against exact sums and fp64, element by element.

Bound.  The sums are exact; fp32 takes them with one rounding, one for the product of the scales and one for that product and the bias: 3 units of 2^-24 of
the magnitudes.  Activations as in ``oracle/gated_linear.py``; the residual is added with one rounding more, and the result rounded to its type."""
import pytest
import torch

from oracle import gated_linear as oracle

pytestmark = pytest.mark.gpu

BF, HF, FL, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
U = oracle.UNIT


def rows(M, K, gen, device):
    q = torch.randint(-127, 128, (M, K), generator=gen, device=device, dtype=I8)
    return q, torch.rand(M, generator=gen, device=device) * 0.02 + 1e-4


def pre(x, w, bias):
    """The sums with scales and bias, and their bound."""
    t = (x[0].double() @ w[0].double().t()) * x[1].double()[:, None] * w[1].double()
    e = 3 * U * t.abs()
    if bias is not None:
        t = t + bias.double()
        e = e + U * t.abs()
    return t, e


def close(name, got, ref, e):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == HF else 2.0 ** -126
    over = ((got.double() - ref).abs() / (half * (ref.abs() + e) + e + tiny)).max().item()
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert torch.isfinite(got).all() and over <= 1.0, f"{name}: {over:.3f} of the bound"


CASES = [  # M, N, K, result, bias, residual, activation
    (1, 1, 16, BF, None, None, None), (1, 130, 2048, BF, BF, None, "silu"), (3, 17, 48, HF, FL, HF, None), (16, 260, 1040, FL, FL, FL, "gelu"),
    (17, 100, 208, BF, None, FL, "relu"), (33, 64, 4096, BF, BF, BF, None), (48, 300, 8192, BF, BF, BF, None), (64, 1000, 272, HF, HF, None, "gelu"),
    (65, 200, 8192, BF, FL, None, None), (100, 57, 2064, FL, None, None, None), (130, 1030, 528, HF, None, HF, "silu"), (300, 2731, 1008, BF, BF, FL, "gelu"),
    (700, 512, 64, FL, FL, FL, "silu"), (2049, 1500, 400, BF, None, BF, None), (3000, 4100, 1040, BF, BF, None, "silu"), (2050, 2056, 2000, FL, None, FL, None),
]


@pytest.mark.parametrize("M,N,K,out,btype,rtype,name", CASES)
def test_linear(device, M, N, K, out, btype, rtype, name):
    from fla_amd.modules import quant_linear
    print(M, N, K, out, btype, rtype, name, flush=True)
    gen = torch.Generator(device=device).manual_seed(M + N + K)
    x, w = rows(M, K, gen, device), rows(N, K, gen, device)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)
    bias = None if btype is None else r(N).to(btype)
    res = None if rtype is None else r(M, N).to(rtype)
    y = quant_linear(x, w, bias, activation=name, residual=res, output_dtype=out)
    t, e = pre(x, w, bias)
    ref = oracle.act(name, t)[0]
    if name is not None:
        e = oracle.SLOPE * e + 3e-7 * t.abs() + (t.abs() + 8) * U * ref.abs()
    if res is not None:
        ref = ref + res.double()
        e = e + U * (ref.abs() + res.double().abs())
    assert y.dtype == out and y.shape == (M, N)
    close("y", y, ref, e)


@pytest.mark.parametrize("M,F,K,out,btype,name", [
    (1, 1, 16, BF, None, "silu"), (2, 40, 2048, BF, BF, "gelu"), (17, 33, 208, HF, FL, None), (64, 500, 1040, BF, None, "relu"), (65, 129, 4096, HF, HF, "silu"),
    (200, 1000, 2048, BF, None, "silu"), (1003, 1501, 512, HF, FL, "gelu"), (2049, 2824, 1040, BF, BF, "silu")])
def test_gated(device, M, F, K, out, btype, name):
    from fla_amd.modules import quant_gated_linear
    gen = torch.Generator(device=device).manual_seed(M + F + K)
    x, wg, wu = rows(M, K, gen, device), rows(F, K, gen, device), rows(F, K, gen, device)
    # (scales as of weights of a layer, so that gates lie where the activation bends)
    x, wg, wu = ((q, s * (2 / (127 * 127 * 0.0101 ** 2 * K ** 0.5)) ** 0.5 * 1.2) for q, s in (x, wg, wu))
    bias = lambda: None if btype is None else torch.randn(F, generator=gen, device=device).to(btype)
    bg, bu = bias(), bias()
    h = quant_gated_linear(x, wg, wu, bg, bu, activation=name, output_dtype=out)
    (g, eg), (u, eu) = pre(x, wg, bg), pre(x, wu, bu)
    a = oracle.act(name, g)[0]
    ea = oracle.SLOPE * eg + 3e-7 * g.abs() + (g.abs() + 8) * U * a.abs()
    ref = a * u
    assert h.dtype == out and h.shape == (M, F)
    close("h", h, ref, u.abs() * ea + a.abs() * eu + ea * eu + 2 * U * ref.abs())


def test_largest_sums_are_exact(device):
    """Rows of -128 of the longest that is taken: 131056 * 2^14 is next to 2^31."""
    from fla_amd.modules import quant_gated_linear, quant_linear
    K = 131056
    for M in (2, 70):
        x = torch.full((M, K), -128, dtype=I8, device=device)
        w = torch.full((40, K), -128, dtype=I8, device=device)
        w[1], w[2, 0] = 127, 0
        one = lambda n: torch.ones(n, device=device)
        y = quant_linear((x, one(M)), (w, one(40)), output_dtype=FL)
        want = torch.tensor([K * 16384, -K * 128 * 127, (K - 1) * 16384], dtype=torch.float64).float().to(device)
        assert torch.equal(y[:, :3], want.expand(M, 3)) and torch.equal(y[:, 3:], want[:1].expand(M, 37))
        h = quant_gated_linear((x, one(M)), (w, one(40) * 2.0 ** -31), (w, one(40) * 2.0 ** -31), activation=None)
        assert (h[:, 0].float() - (K * 2.0 ** -17) ** 2).abs().max() <= 2.0 ** -8


def test_strides_addresses_and_dimensions(device):
    from fla_amd.modules import quant_gated_linear, quant_linear
    gen = torch.Generator(device=device).manual_seed(5)
    x, w = rows(30, 64, gen, device), rows(48, 64, gen, device)
    ref, gref = quant_linear(x, w), quant_gated_linear(x, w, w)
    odd = torch.empty(1 + 30 * 64, device=device, dtype=I8)[1:].view(30, 64).copy_(x[0])
    wide = torch.empty(30, 100, device=device, dtype=I8)[:, 20:84].copy_(x[0])
    scale = torch.empty(60, device=device)[::2].copy_(x[1])
    for q in (odd, wide):
        assert torch.equal(quant_linear((q, scale), w), ref) and torch.equal(quant_gated_linear((q, scale), w, w), gref)
    deep = (x[0].view(2, 3, 5, 64), x[1].view(2, 3, 5))
    assert torch.equal(quant_linear(deep, w).view(30, 48), ref) and torch.equal(quant_gated_linear(deep, w, w).view(30, 48), gref)
    one = quant_linear((x[0][0], x[1][0]), w)
    assert one.shape == (48,) and torch.equal(one, ref[0])
    assert quant_linear((x[0][:0], x[1][:0]), w).shape == (0, 48) and quant_gated_linear((x[0][:0], x[1][:0]), w, w).shape == (0, 48)


def test_scales_that_are_not_finite_stay_in_their_row(device):
    from fla_amd.modules import quant_linear, quantize_rows
    gen = torch.Generator(device=device).manual_seed(6)
    v, w = torch.randn(80, 64, generator=gen, device=device), rows(48, 64, gen, device)
    bad = v.clone()
    bad[3, 5], bad[70, 0] = float("nan"), float("inf")
    y, z = (quant_linear(quantize_rows(t, I8), w) for t in (v, bad))
    keep = [i for i in range(80) if i not in (3, 70)]
    assert torch.equal(y[keep], z[keep]) and z[3].isnan().all() and z[70].isnan().all()


def test_module(device):
    from fla_amd.modules import QuantLinear, quant_linear, quantize_rows
    torch.manual_seed(0)
    lin = torch.nn.Linear(96, 40, device=device)
    m = QuantLinear.from_linear(lin, activation="relu", dtype=I8)
    assert m.weight.dtype == I8 and m.output_dtype == BF
    x, res = torch.randn(7, 96, device=device), torch.randn(7, 40, device=device)
    y = m(x, residual=res)
    assert torch.equal(y, m(quantize_rows(x, I8), res)) and y.dtype == BF
    ref = torch.relu(lin(x)) + res
    assert ((y.float() - ref).norm() / ref.norm()).item() <= 0.02      # (8-bit rows and weights: steps of 1/127 of each row's largest)
    m = m.to(HF)
    assert m.weight.dtype == I8 and m.weight_scale.dtype == FL and m.bias.dtype == HF
    assert torch.equal(QuantLinear.from_linear(lin, dtype=I8).to("cpu").weight, m.weight.cpu())
    other = QuantLinear(96, 40, device=device, dtype=I8)
    other.load_state_dict(QuantLinear.from_linear(lin, dtype=I8).state_dict())
    assert torch.equal(other.weight, m.weight) and torch.equal(other(x), quant_linear(quantize_rows(x, I8), (m.weight, m.weight_scale), lin.bias.detach()))


def test_refusals(device):
    from fla_amd.modules import quant_gated_linear, quant_linear
    gen = torch.Generator(device=device).manual_seed(7)
    x, w = rows(4, 32, gen, device), rows(8, 32, gen, device)
    b = torch.zeros(8, device=device, requires_grad=True)
    for call in (lambda: quant_linear(x, w, b), lambda: quant_gated_linear(x, w, w, b)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(RuntimeError, match="GPU"):
        quant_linear(x, (w[0].cpu(), w[1]))
    with pytest.raises(RuntimeError, match="GPU"):
        quant_gated_linear(x, w, (w[0], w[1].cpu()))


def test_captured(device):
    """A projection with slices of K and a gated product in a graph, replayed with other inputs, eager work between the replays."""
    from fla_amd.modules import quant_gated_linear, quant_linear, quantize_rows
    gen = torch.Generator(device=device).manual_seed(8)
    M = 100
    wg, wu, wd = rows(136, 2048, gen, device), rows(136, 2048, gen, device), rows(72, 144, gen, device)
    wg, wu = (wg[0], wg[1] * 1e-3), (wu[0], wu[1] * 1e-3)
    pad = lambda h: torch.nn.functional.pad(h, (0, 8))
    run = lambda x: quant_linear(quantize_rows(pad(quant_gated_linear(quantize_rows(x, I8), wg, wu)), I8), wd)
    xs = [torch.randn(M, 2048, generator=gen, device=device).to(BF) for _ in range(3)]
    eager = [run(x) for x in xs]
    static = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run(static), eager[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    for i in (1, 2, 0, 1):
        static.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), i
        run(xs[2])
