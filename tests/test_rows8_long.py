"""Rows in 8 bits of more elements than a norm takes, and the projections over them."""
import ctypes

import pytest
import torch

F8 = torch.float8_e4m3fn


def test_a_layer_is_refused_where_it_is_made():
    from fla_amd.modules import QuantLinear
    for inner in (24, 8, 0, (1 << 23) + 16):
        with pytest.raises(NotImplementedError, match=f"multiple of 16 elements, at most 2\\^23, not {inner}"):
            QuantLinear(inner, 1)
    assert QuantLinear(20480, 2).weight.shape == (2, 20480)


def test_lengths_of_the_library_entry():
    from fla_amd import _backend as be
    p = ctypes.c_void_p(torch.zeros(64).data_ptr())
    rows = lambda N, res=None, out=None, M=0: be.lib().fla_rms_norm_fwd(p, res, 0, None, None, 0, p, p, out, 0, None, M, N, 0.0, 0, 0, None)
    assert rows(16385) == 0 and rows(1 << 23) == 0 and rows((1 << 23) + 1) == -2
    assert rows(16384, p) == 0 and rows(16385, p) == -2 and rows(16385, None, p) == -2      # with a sum: rows that stay in registers


def test_the_error_names_the_call():
    from fla_amd.modules import quantize_rows
    with pytest.raises(NotImplementedError, match="quantize_rows: rows of at most 8388608"):
        quantize_rows(torch.zeros(1, (1 << 23) + 8, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="quantize_rows"):
        quantize_rows(torch.zeros(1, 8).long())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N", [(1, 16385), (3, 16392), (70, 28672), (2, 53248), (5, 100003), (1, 1 << 23)])
def test_long_rows(device, M, N, dtype):
    """Bit for bit the fp32 quotients by the scale, rounded once; at an odd address, and with a row that is no number between others."""
    from fla_amd.modules import quantize_rows
    gen = torch.Generator().manual_seed(M + N)
    x = (torch.randn(M, N, generator=gen) * torch.exp(3 * torch.randn(M, 1, generator=gen))).to(dtype)
    x[0, N - 1] = x[0].abs().max() * 2        # the maximum in the row's last place
    want = x.float().abs().amax(-1).clamp_min(1e-30) / 448
    wq = (x.float() / want[:, None]).to(F8).view(torch.uint8)
    base = torch.zeros(M * N + 1, dtype=dtype, device=device)
    base[1:] = x.to(device).flatten()
    for name, given in (("rows", x.to(device)), ("odd address", base[1:].view(M, N))):
        q, scale = quantize_rows(given)
        assert q.dtype == F8 and q.shape == x.shape and torch.equal(scale.cpu(), want), name
        assert torch.equal(q.cpu().view(torch.uint8), wq), name
    if M > 2:
        x[1, N // 2] = float("nan")
        q2, scale2 = quantize_rows(x.to(device))
        keep = torch.arange(M) != 1
        assert torch.equal(q2.cpu().view(torch.uint8)[keep], wq[keep]) and torch.equal(scale2.cpu()[keep], want[keep])
        assert q2[1, N // 2].isnan()


@pytest.mark.gpu
def test_a_projection_of_long_rows(device):
    """The whole layer against fp64 on its 8-bit operands.  Products of eight are cut at 2^-13 of the largest of them, each with its own
    sign: seven standard deviations of their sum, at most 8 max^2 <= 8 sum of squares a group; K / 8 sums in fp32; half a step of bf16."""
    from fla_amd.modules import QuantLinear, quantize_rows
    gen = torch.Generator().manual_seed(0)
    for M, N, K in ((1, 40, 20480), (70, 72, 28672)):
        lin = torch.nn.Linear(K, N)
        with torch.no_grad():
            lin.weight.copy_(torch.randn(N, K, generator=gen) * K ** -0.5)
        layer = QuantLinear.from_linear(lin.to(device, torch.bfloat16))
        x = torch.randn(M, K, generator=gen).bfloat16().to(device)
        q, s = quantize_rows(x)
        y = layer(x)
        assert torch.equal(y, layer((q, s)))
        xd, wd = q.cpu().double() * s.cpu().double()[:, None], layer.weight.cpu().double() * layer.weight_scale.cpu().double()[:, None]
        ref = xd @ wd.t() + layer.bias.cpu().double()
        e = 7 * 2.0 ** -13 * (8 * (xd.square() @ wd.square().t())).sqrt() + (K / 8 + 8) * 2.0 ** -24 * (xd.abs() @ wd.abs().t())
        off = ((y.double().cpu() - ref).abs() / (2.0 ** -8 * (ref.abs() + e) + e)).max().item()
        print(M, N, K, off, flush=True)
        assert off <= 1.0
