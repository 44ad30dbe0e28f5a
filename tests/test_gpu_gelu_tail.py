"""GPU: GELU and its slope relative to their own value where they are small, against erfc in fp64.

Bound of the tail Phi(v), v < 0, in units of 2^-24: 1.32 for the fit (7.9e-8), 2 each for the hardware's reciprocal and exponential (1 ulp), 0.5 for each of the ten other
roundings on the way, and v^2 / 2 times 2.5 for v^2, its product with log2(e) / 2 and that constant, each half a unit at most in an exponent of v^2 / 2: below 1.25 v^2 + 16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, FL, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
U = 2.0 ** -24


def reference(v):
    """GELU and its slope in fp64, and the bounds of both relative errors ahead of a result's own rounding."""
    v = v.double()
    cdf, bell = 0.5 * torch.erfc(-v / math.sqrt(2.0)), v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    e = (1.25 * v * v + 16) * U
    return v * cdf, (e + U) * (v * cdf).abs(), cdf + bell, (e + 3 * U) * (cdf.abs() + bell.abs())


def close(name, got, ref, e):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == HF else 2.0 ** -126
    over = ((got.double() - ref).abs() / (half * (ref.abs() + e) + e + tiny)).max().item()
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, f"{name}: {over:.3f} of the bound"


N = 4003


@pytest.mark.parametrize("M,K", [(1, 16), (70, 32), (70, 4096), (300, 32)])
@pytest.mark.parametrize("out", [FL, HF, BF])
def test_integers(device, M, K, out):
    """Sums of -1 and weights' scales of any fp32 value: the pre-activation is that value."""
    from fla_amd.modules import quant_gated_linear, quant_linear
    v = torch.linspace(-12, 0, N, device=device)
    x, w = torch.zeros(M, K, device=device, dtype=I8), torch.zeros(N, K, device=device, dtype=I8)
    x[:, 0], w[:, 0] = -1, 1
    one = torch.ones(M, device=device)
    ref, e, _, _ = reference(v)
    y = quant_linear((x, one), (w, -v), activation="gelu", output_dtype=out)
    close("y", y, ref.expand(M, N), e.expand(M, N))
    if out != FL:
        h = quant_gated_linear((x, one), (w, -v), (-w, torch.ones(N, device=device)), activation="gelu", output_dtype=out)
        close("h", h, ref.expand(M, N), e.expand(M, N))


@pytest.mark.parametrize("M,K", [(1, 8), (70, 64), (70, 4096)])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_gate_and_slope(device, M, K, dtype):
    from fla_amd.modules import gated_linear
    v = torch.linspace(-12, 0, N, device=device).to(dtype)
    x, wg, wu = torch.zeros(M, K, device=device, dtype=dtype), torch.zeros(N, K, device=device, dtype=dtype), torch.zeros(N, K, device=device, dtype=dtype)
    x[:, 0], wg[:, 0], wu[:, 0] = 1, v, 1
    bias = torch.zeros(N, device=device, requires_grad=True)
    ref, e, slope, es = reference(v)
    h = gated_linear(x, wg, wu, bias, None, activation="gelu")
    close("h", h, ref.expand(M, N), e.expand(M, N))
    dh = torch.zeros_like(h)
    dh[-1] = 1
    (d,) = torch.autograd.grad(h, bias, dh)
    close("slope", d, slope, es)
