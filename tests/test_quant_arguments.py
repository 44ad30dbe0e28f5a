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


def test_state_of_another_type_is_refused():
    """Rows of 8-bit integers and of e4m3 have the same names and shapes; converted number by number they would not fit their scales."""
    from fla_amd.modules import QuantLinear
    F8, I8 = torch.float8_e4m3fn, torch.int8
    for mine, other in ((F8, I8), (I8, F8)):
        layer, state = QuantLinear(32, 8, dtype=mine), QuantLinear(32, 8, dtype=other).state_dict()
        state["weight_scale"] = torch.ones(8)
        with pytest.raises(RuntimeError, match="make it with dtype"):
            torch.nn.Sequential(layer).load_state_dict({"0." + k: v for k, v in state.items()})
        assert layer.weight.dtype == mine and not layer.weight_scale.any()
        layer.load_state_dict(state, assign=True)
        assert layer.weight.dtype == other and layer.weight_scale.all()
        same = QuantLinear(32, 8, dtype=mine)
        state = same.state_dict()
        state["weight"] = torch.ones(8, 32).to(mine)
        same.load_state_dict(state)
        assert (same.weight.float() == 1).all()
