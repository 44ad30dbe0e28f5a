"""CPU: refusals of the 8-bit products and of the library entry under them."""
import ctypes

import pytest
import torch

F8 = torch.float8_e4m3fn


def _rows(M, K):
    return torch.zeros(M, K).to(F8), torch.ones(M)


def test_refusals():
    from fla_amd.modules import QuantLinear, quant_linear
    x, w = _rows(3, 32), _rows(5, 32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        quant_linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        QuantLinear(32, 5)(x)
    with pytest.raises(TypeError, match="pairs of rows"):
        quant_linear((x[0].float(), x[1]), w)
    with pytest.raises(TypeError, match="pairs of rows"):
        quant_linear(x, (w[0], w[1].double()))
    with pytest.raises(ValueError, match="weight \\[N, K\\]"):
        quant_linear(x, _rows(5, 16))
    with pytest.raises(ValueError, match="one scale for every row"):
        quant_linear((x[0], torch.ones(1)), w)
    with pytest.raises(ValueError, match="one scale for every row"):
        quant_linear(x, (w[0], torch.ones(5, 1)))
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        quant_linear(_rows(3, 24), _rows(5, 24))
    with pytest.raises(ValueError, match="5 values"):
        quant_linear(x, w, torch.zeros(4))
    with pytest.raises(ValueError, match="residual is"):
        quant_linear(x, w, residual=torch.zeros(5))
    with pytest.raises(TypeError, match="output's type or in fp32"):
        quant_linear(x, w, residual=torch.zeros(3, 5).half())
    with pytest.raises(ValueError, match="unknown activation"):
        quant_linear(x, w, activation="tanh")
    with pytest.raises(NotImplementedError, match="bf16 or fp16"):
        quant_linear(x, w, output_dtype=torch.float32)
    with pytest.raises(ValueError, match="unknown activation"):
        QuantLinear(32, 5, activation="tanh")


def test_library_arguments():
    from fla_amd import _backend as be
    lib = be.lib()
    buf = torch.zeros(64)
    p, odd = ctypes.c_void_p(buf.data_ptr()), ctypes.c_void_p(buf.data_ptr() + 4)
    call = lambda x=p, K=16, act=0, dtype=1, res=None, rt=0, N=4: lib.fla_quant_linear(x, p, p, p, None, 0, res, rt, p, 1, N, K, act, dtype, None, None)
    assert call(x=None) == -1 and call(K=0) == -1 and call(act=4) == -1 and call(N=0) == -1
    assert call(K=24) == -2 and call(dtype=0) == -2 and call(res=p, rt=2) == -2
    assert call(x=odd) == -3
    # few tiles and a long K: in slices, which need a workspace; single rows and large products are not cut
    splits = lib.fla_quant_linear_splits
    assert splits(100, 2048, 8192) > 1 and splits(48, 2048, 8192) == 1 and splits(1, 4096, 2048) == 1 and splits(8191, 8192, 2048) == 1 and splits(0, 1, 1) == 1
    assert lib.fla_quant_linear(p, p, p, p, None, 0, None, 0, p, 100, 2048, 8192, 0, 1, None, None) == -1
