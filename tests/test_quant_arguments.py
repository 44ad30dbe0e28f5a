"""CPU: which values the arguments of rows in 8 bits take."""
import pytest
import torch


def test_quantize_none_is_false():
    """(a call that goes on to the check of the device has been taken)"""
    from fla_amd.modules import LayerNorm, RMSNorm, layer_norm, quantize_rows, rms_norm
    x = torch.zeros(2, 8)
    for call in (lambda q: rms_norm(x, None, quantize=q), lambda q: layer_norm(x, None, quantize=q), lambda q: RMSNorm(8)(x, quantize=q),
                 lambda q: LayerNorm(8)(x, quantize=q)):
        for q in (None, False, 0):
            with pytest.raises(RuntimeError, match="GPU"):
                call(q)
        with pytest.raises(ValueError, match="rows in 8 bits"):
            call(torch.int16)
    with pytest.raises(ValueError, match="dtype"):
        quantize_rows(x, None)
