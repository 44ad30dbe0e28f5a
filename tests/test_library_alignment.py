"""CPU: workspaces that the kernels write 16 bytes at a time are refused at other addresses by the library entries."""
import ctypes

import torch

from fla_amd import _backend as be

ALIGNMENT = -3


def test_workspaces_of_the_recurrence_and_the_norm():
    lib = be.lib()
    buf = torch.zeros(64)
    p, odd = ctypes.c_void_p(buf.data_ptr()), ctypes.c_void_p(buf.data_ptr() + 4)
    fwd = lambda states: lib.fla_hgrn_fwd(p, p, None, None, p, None, states, None, None, None, None, 0, 256, 0, 0, 0, 1, 8, 8, 1, 8, 8, None)
    bwd = lambda states: lib.fla_hgrn_bwd(p, p, None, states, None, None, p, p, None, None, None, None, None, None, 0, 256, 0, 0, 0, 1, 8, 8, 1,
                                          8, 8, None)
    assert fwd(odd) == ALIGNMENT and bwd(odd) == ALIGNMENT
    norm = lambda dw, db: lib.fla_rms_norm_bwd(p, p, 0, None, 0, p, None, p, None, dw, db, 0, 8192, 0, None)
    assert norm(odd, None) == ALIGNMENT and norm(None, odd) == ALIGNMENT and norm(p, p) == 0
