"""GPU: gradients of the gated product start from the pre-activations as they were summed, in fp32: their digits, and gates and factors beyond the range of fp16."""
import pytest
import torch

from oracle import gated_linear as oracle

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
ACTS = ("silu", "gelu", "relu", None)


def close(name, got, ref, bound):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == HF else 2.0 ** -126
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = ((got.double() - ref).abs() / (half * (ref.abs() + bound) + bound + tiny)).max().item()
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, f"{name}: {over:.3f} of the bound"


def way(M, F, K):
    """Which of the three places that keep the pre-activations a call goes through."""
    from fla_amd import _backend as be
    return "panel" if M <= 64 else "slices" if be.lib().fla_gated_linear_splits(M, F, K, 2) > 1 else "tile"


WAYS = [("panel", 1, 8), ("tile", 70, 64), ("slices", 70, 4096)]      # rows, columns of x


@pytest.mark.parametrize("which,M,K", WAYS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_digits(device, which, M, K, dtype):
    """One row of x is (1, 1, 0, ...) and all others are zeros, so g and u are sums of two numbers, exact in fp32 and not in 16 bits, and the weights' gradients
    are dg and du themselves, rounded once.  Pre-activations in 16 bits would add half a step of their own."""
    from fla_amd.modules import gated_linear
    F = 4001
    assert way(M, F, K) == which
    gen = torch.Generator().manual_seed(M)
    x = torch.zeros(M, K)
    x[-1, :2] = 1
    w = torch.zeros(2, F, K)
    w[0, :, 0], w[1, :, 0] = torch.linspace(-6, 6, F), 2 * torch.rand(F, generator=gen) - 4
    w[:, :, 1] = torch.randn(2, F, generator=gen) * 2.0 ** -8
    dh = torch.randn(M, F, generator=gen).to(dtype).to(device)
    x, (wg, wu) = x.to(dtype).to(device), (t.to(dtype).to(device).requires_grad_() for t in w)
    g, u = (t[:, :2].detach().double().sum(1) for t in (wg, wu))
    for name in ACTS:
        dwg, dwu = torch.autograd.grad(gated_linear(x, wg, wu, activation=name), (wg, wu), dh)
        a, slope = oracle.act(name, g)
        d = dh[-1].double()
        # (the evaluation of the activation and its slope, and their products' roundings)
        ea, es = 3e-7 * g.abs() + (g.abs() + 8) * oracle.UNIT * a.abs(), 1e-6 * (1 + g.abs()) if name in ("silu", "gelu") else 0 * g
        for k, got, ref, e in (("dwg", dwg, d * u * slope, (d * u).abs() * es), ("dwu", dwu, d * a, d.abs() * ea)):
            close(f"{name} {k}", got[:, 0], ref, e + 4 * oracle.UNIT * ref.abs())
            assert torch.equal(got[:, 0], got[:, 1]) and not got[:, 2:].any()


@pytest.mark.parametrize("which,M,K", WAYS)
def test_beyond_the_range_of_fp16(device, which, M, K):
    """Gates of +-70000 with small factors and factors of +-70000 with small gates: h is in fp16's range, and so are all gradients of the formula."""
    from fla_amd.modules import gated_linear
    F = 264
    big = torch.tensor([70000.0, -70000.0, 131072.0, -131072.0]).repeat(F // 4)
    small = torch.linspace(-0.25, 0.25, F)
    gen = torch.Generator().manual_seed(K)
    w = torch.zeros(2, F, K)
    half = F // 2
    w[0, :, 0], w[1, :, 0] = torch.where(torch.arange(F) < half, big, small) / 64, torch.where(torch.arange(F) < half, small, big) / 64
    x = torch.randn(M, K, generator=gen) * 0.25
    x[:, 0] = 64 * torch.linspace(1, 0.5, M)
    dh = torch.randn(M, F, generator=gen) * 2.0 ** -13
    x, wg, wu, dh = (t.to(HF).to(device) for t in (x, w[0], w[1], dh))
    assert way(M, F, K) == which
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    for name in ACTS:
        args = [t.detach().double() for t in leaves]
        h_ref, e_h, state = oracle.forward(*args, name=name)
        assert state[0].abs().max() > 65504 and state[2].abs().max() > 65504 and h_ref.abs().max() < 65504
        h = gated_linear(*leaves, activation=name)
        close(f"{name} h", h.detach(), h_ref, e_h)
        want = oracle.backward(*args, state, dh.double(), name, 2.0 ** -11)
        for k, got in zip(("dx", "dwg", "dwu"), torch.autograd.grad(h, leaves, dh)):
            close(f"{name} {k}", got, want[k], want["e_" + k])
