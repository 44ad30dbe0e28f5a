"""CPU: the oracle of the RMS norm (against torch, its gradients against autograd and differences) and the entry points' refusals."""
import ctypes

import pytest
import torch

from oracle import rms_norm as oracle


def test_formula_and_gradients():
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    x, res, w, b, dy, ds = r(6, 10), r(6, 10), r(10), r(10), r(6, 10), r(6, 10)
    y, s, rstd, _ = oracle.forward(x, w, b, res)
    assert torch.allclose(y, torch.nn.functional.rms_norm(x + res, (10,), w, eps=1e-5) + b, rtol=1e-12)
    leaves = [t.clone().requires_grad_() for t in (x, res, w, b)]

    def loss(x, res, w, b):
        y, s, _, _ = oracle.forward(x, w, b, res)
        return (y * dy).sum() + (s * ds).sum()

    assert torch.autograd.gradcheck(loss, leaves)
    want = torch.autograd.grad(loss(*leaves), leaves)
    got = oracle.backward(s, rstd, dy, w, ds)
    for g, v in zip(("dx", "dx", "dw", "db"), want):
        assert torch.allclose(got[g], v, rtol=1e-11, atol=1e-12), g


def test_refusals():
    from fla_amd.modules import RMSNorm, quantize_rows, rms_norm
    x, w = torch.zeros(4, 16), torch.ones(16)
    for call in (lambda: rms_norm(x, w), lambda: quantize_rows(x), lambda: RMSNorm(16)(x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="16 values"):
        rms_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="16 values"):
        rms_norm(x, w, torch.ones(1, 16))
    with pytest.raises(ValueError, match="x's shape"):
        rms_norm(x, w, residual=torch.zeros(4, 8))
    with pytest.raises(TypeError, match="x's type or in fp32"):
        rms_norm(x.bfloat16(), w, residual=x.half())
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        rms_norm(x.long(), w)
    with pytest.raises(ValueError, match="N at least 1"):
        rms_norm(torch.zeros(()), w)
    with pytest.raises(NotImplementedError, match="16384"):
        rms_norm(torch.zeros(1, 16385), None)
    assert repr(RMSNorm(16)) == "RMSNorm(16, eps=1e-05)" and RMSNorm(16, elementwise_affine=False).weight is None
    assert RMSNorm(16, bias=True).bias.shape == (16,) and RMSNorm(16).bias is None


def test_library_arguments():
    from fla_amd import _backend as be
    lib = be.lib()
    p = ctypes.c_void_p(torch.zeros(64).data_ptr())
    fwd = lambda N=8, scale=None, w=None, rt=0, norm=1, dtype=0, x=p: lib.fla_rms_norm_fwd(x, None, rt, w, None, 0, p, scale, None, 0, None, 1, N,
                                                                                         1e-5, norm, dtype, None)
    assert fwd(x=None) == -1 and fwd(N=0) == -1 and fwd(N=16385) == -2
    assert fwd(norm=0) == -1 and fwd(norm=0, scale=p, w=p) == -1
    assert lib.fla_rms_norm_fwd(p, p, 2, None, None, 0, p, None, None, 0, None, 1, 8, 1e-5, 1, 1, None) == -2    # residual in another 16-bit type
    assert lib.fla_rms_norm_bwd(p, p, 0, None, 0, None, None, p, None, None, None, 1, 8, 0, None) == -1          # no rstd
    assert lib.fla_rms_norm_bwd(p, p, 2, None, 0, p, None, p, None, None, None, 1, 8, 1, None) == -2
    assert lib.fla_rms_norm_workgroups(1, 16384) == 1 and lib.fla_rms_norm_workgroups(1 << 30, 64) == 1024
