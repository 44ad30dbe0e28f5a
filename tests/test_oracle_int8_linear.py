"""CPU: what the products of rows in 8-bit integers refuse ahead of a launch."""
import pytest
import torch

I8, F8 = torch.int8, torch.float8_e4m3fn


def _rows(M, K, dtype=I8):
    return torch.zeros(M, K).to(dtype), torch.ones(M)


def test_refusals():
    from fla_amd.modules import QuantLinear, quant_gated_linear, quant_linear
    x, w = _rows(2, 32), _rows(8, 32)
    both = (lambda a, b, **k: quant_linear(a, b, **k), lambda a, b, **k: quant_gated_linear(a, b, b, **k))
    for call in both:
        with pytest.raises(RuntimeError, match="GPU"):
            call(x, w)
        with pytest.raises(TypeError, match="pairs"):
            call(x, _rows(8, 32, F8))
        with pytest.raises(TypeError, match="pairs"):
            call((x[0].to(torch.uint8), x[1]), w)
        with pytest.raises(TypeError, match="pairs"):
            call((x[0], x[1].half()), w)
        with pytest.raises(ValueError, match="weight"):
            call(_rows(2, 16), w)
        with pytest.raises(ValueError, match="scale"):
            call((x[0], x[1][:1]), w)
        with pytest.raises(ValueError, match="scale"):
            call(x, (w[0], w[1][:4]))
        with pytest.raises(NotImplementedError, match="multiple of 16"):
            call(_rows(2, 24), _rows(8, 24))
        with pytest.raises(NotImplementedError, match="131056"):
            call(_rows(1, 131072), _rows(1, 131072))
        with pytest.raises(ValueError, match="activation"):
            call(x, w, activation="tanh")
    with pytest.raises(ValueError, match="residual"):
        quant_linear(x, w, residual=torch.zeros(2, 4))
    with pytest.raises(TypeError, match="residual"):
        quant_linear(x, w, residual=torch.zeros(2, 8).half())
    with pytest.raises(ValueError, match="bias"):
        quant_linear(x, w, torch.zeros(4))
    with pytest.raises(NotImplementedError, match="results"):
        quant_linear(x, w, output_dtype=torch.float64)
    with pytest.raises(NotImplementedError, match="results"):
        quant_linear(_rows(2, 32, F8), _rows(8, 32, F8), output_dtype=torch.float32)
    with pytest.raises(NotImplementedError, match="results"):
        quant_gated_linear(x, w, w, output_dtype=torch.float32)
    with pytest.raises(NotImplementedError, match="int8"):
        quant_gated_linear(_rows(2, 32, F8), _rows(8, 32, F8), _rows(8, 32, F8))
    with pytest.raises(ValueError, match="weight"):
        quant_gated_linear(x, w, _rows(4, 32))
    with pytest.raises(ValueError, match="biases"):
        quant_gated_linear(x, w, w, torch.zeros(4))
    with pytest.raises(ValueError, match="weights in"):
        QuantLinear(32, 8, dtype=torch.int16)
    with pytest.raises(NotImplementedError, match="131056"):
        QuantLinear(131072, 1, dtype=I8)
    assert QuantLinear(131072, 1).weight.dtype == F8


def test_library_entries_refuse():
    import ctypes
    from fla_amd import _backend as be
    lib, buf = be.lib(), (ctypes.c_float * 64)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    lin = lambda x=at, M=2, N=8, K=32, act=0, dtype=1, bt=1, ws=None: lib.fla_int8_linear(x, at, at, at, at, bt, None, 0, at, M, N, K, act, dtype, ws, None)
    assert lin(x=None) == -1 and lin(N=0) == -1 and lin(act=7) == -1 and lin(dtype=3) == -2 and lin(bt=2) == -2
    assert lin(K=24) == -2 and lin(K=131072) == -2 and lin(N=(1 << 22) + 1) == -2 and lin(x=at + 8) == -3 and lin(M=0) == 0
    split = lib.fla_int8_linear_splits(100, 128, 8192, 1)
    assert split > 1 and lin(M=100, N=128, K=8192) == -1 and lin(M=100, N=128, K=8192, ws=at + 4) == -3
    gated = lambda x=at, K=32, act=1, dtype=1: lib.fla_int8_gated_linear_fwd(x, at, at, at, at, at, None, None, 0, at, 2, 8, K, act, dtype, None, None)
    assert gated(x=None) == -1 and gated(K=24) == -2 and gated(K=131072) == -2 and gated(act=9) == -1 and gated(dtype=0) == -2 and gated(x=at + 4) == -3
