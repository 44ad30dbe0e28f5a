"""CPU: sizes that a launch does not take are refused by the library entries."""
import ctypes

import torch

from fla_amd import _backend as be


def test_columns_of_a_product_of_few_rows():
    p = ctypes.c_void_p(torch.zeros(64).data_ptr())
    call = lambda M, N: be.lib().fla_quant_linear(p, p, p, p, None, 0, None, 0, p, M, N, 16, 0, 1, None, None)
    unsupported = -2
    assert call(1, 1 << 28) == unsupported and call(48, (1 << 31) - 1) == unsupported
    assert call(0, 1 << 28) == 0 and call(0, 1 << 31) == unsupported
