"""CPU: the oracle of the layer norm against torch's and autograd, in fp64."""
import pytest
import torch

from oracle import layer_norm as oracle


@pytest.mark.parametrize("M,N", [(1, 1), (3, 10), (7, 64)])
@pytest.mark.parametrize("affine", [False, True])
def test_forward_and_gradients(M, N, affine):
    gen = torch.Generator().manual_seed(M + N)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64, requires_grad=True)
    x, res, dy, ds = r(M, N), r(M, N), r(M, N).detach(), r(M, N).detach()
    w, b = (r(N), r(N)) if affine else (None, None)
    y, s, stats, _ = oracle.forward(x, w, b, res)
    assert torch.allclose(y, torch.nn.functional.layer_norm(x + res, (N,), w, b, eps=1e-5), rtol=1e-11, atol=1e-11)
    leaves = [x, res] + ([w, b] if affine else [])
    want = torch.autograd.grad((y, s), leaves, (dy, ds))
    got = oracle.backward((x + res).detach(), [t.detach() for t in stats], dy, None if w is None else w.detach(), ds)
    for name, ref in zip(("dx", "dx", "dw", "db"), want):
        assert torch.allclose(got[name], ref, rtol=1e-9, atol=1e-9), name


def test_gradient_is_the_difference_quotient():
    gen = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((2, 9), (9,), (9,)))
    f = lambda t: oracle.forward(t, w, b)[0]
    assert torch.autograd.gradcheck(f, (x.requires_grad_(),), eps=1e-6, atol=1e-6)


def test_rows_of_integers():
    x = torch.tensor([[0.5, -127.0, 1.5, 126.5, 2.5], [0.0, 0.0, 0.0, 0.0, 0.0]], dtype=torch.float64)
    q, scale = oracle.rows_int8(x)
    assert q.tolist() == [[0, -127, 2, 126, 2], [0, 0, 0, 0, 0]] and scale.tolist() == [1.0, 1e-30 / 127]


@pytest.mark.parametrize("quantize", [torch.int16, "int8", 3, torch.float32])
def test_other_types_of_rows_are_refused(quantize):
    from fla_amd.modules import layer_norm, quantize_rows, rms_norm
    x, w = torch.zeros(2, 16), torch.ones(16)
    for call in (lambda: layer_norm(x, w, quantize=quantize), lambda: rms_norm(x, w, quantize=quantize), lambda: quantize_rows(x, quantize)):
        with pytest.raises(ValueError, match="rows in 8 bits"):
            call()
    with pytest.raises(ValueError, match="dtype"):
        quantize_rows(x, False)


def test_cpu_tensors_and_shapes_are_refused():
    from fla_amd.modules import LayerNorm, layer_norm
    x, w = torch.zeros(2, 16), torch.ones(16)
    with pytest.raises(RuntimeError, match="GPU"):
        layer_norm(x, w)
    with pytest.raises(ValueError, match="hold 16"):
        layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="residual"):
        layer_norm(x, w, residual=torch.zeros(2, 8))
    with pytest.raises(TypeError, match="residual"):
        layer_norm(x, w, residual=x.bfloat16())
    with pytest.raises(TypeError, match="bf16"):
        layer_norm(x.double(), w)
    with pytest.raises(NotImplementedError, match="16384"):
        layer_norm(torch.zeros(1, 16385), None)
    m = LayerNorm(16)
    assert m.bias is None and m.weight.shape == (16,) and repr(m) == "LayerNorm(16, eps=1e-05)"


def test_library_entry_refuses():
    import ctypes
    from fla_amd import _backend as be
    lib, buf = be.lib(), (ctypes.c_float * 64)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    fwd = lambda scale, rows8, N=16, dtype=0: lib.fla_layer_norm_fwd(at, None, 0, None, None, 0, at, scale, None, 0, None, None, 1, N, 1e-5, rows8,
                                                                     dtype, None)
    assert fwd(None, 1) == -1 and fwd(at, 0) == -1 and fwd(at, 3) == -1 and fwd(None, 0, N=16385) == -2 and fwd(None, 0, N=0) == -1
    assert lib.fla_layer_norm_bwd(at, at, 0, None, 0, None, at, None, at, None, None, None, 16, 1, 16, 0, None) == -1      # no mean
    assert lib.fla_layer_norm_bwd(at, at, 0, None, 0, at, at, None, at, None, at + 4, None, 16, 1, 16, 0, None) == -3
    assert lib.fla_layer_norm_bwd(at, at, 0, None, 0, at, at, None, at, None, at, None, 8, 1, 16, 0, None) == -1
    assert lib.fla_rms_norm_rows8_fwd(at, None, 0, None, None, 0, at, None, None, 0, 1, 16, 1e-5, 1, 2, 0, None) == -1
