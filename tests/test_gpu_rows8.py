"""GPU: rows in 8 bits, bit for bit: they are the fp32 quotients by the scale, rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def _expected(y):
    scale = y.abs().amax(-1).clamp_min(1e-30) / 448
    return (y / scale[..., None]).to(F8), scale


def _same(name, got, want):
    q, scale = got[0].cpu().view(torch.uint8), got[1].cpu()
    wq, ws = want[0].view(torch.uint8), want[1]
    assert torch.equal(scale, ws), name
    off = (q != wq).sum().item()
    print(f"{name}: {off} of {q.numel()} differ", flush=True)
    assert off == 0, f"{name}: {off} of {q.numel()} differ"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N", [(3, 1), (40, 64), (500, 1000), (2000, 2048), (300, 4096), (64, 7001), (64, 16384)])
def test_rows(device, M, N, dtype):
    from fla_amd.modules import quantize_rows
    gen = torch.Generator().manual_seed(M + N)
    # (a spread of sizes: the 8-bit type's numbers below the normal ones too)
    x = (torch.randn(M, N, generator=gen) * torch.exp(4 * torch.randn(M, 1, generator=gen) - 3 * torch.rand(M, N, generator=gen))).to(dtype)
    _same("rows", quantize_rows(x.to(device)), _expected(x.float()))


@pytest.mark.parametrize("M,N", [(40, 64), (2000, 2048), (300, 4096), (70, 1001), (64, 16384)])
def test_rows_of_the_norm(device, M, N):
    """An fp32 norm's own result, quantised by the formula, is what it gives in 8 bits."""
    from fla_amd.modules import rms_norm
    gen = torch.Generator().manual_seed(M + N)
    x, r, w = (torch.randn(*s, generator=gen).to(device) for s in ((M, N), (M, N), (N,)))
    with torch.no_grad():
        y = rms_norm(x, w, residual=r)
        _same("norm", rms_norm(x, w, residual=r, quantize=True), _expected(y.cpu()))
