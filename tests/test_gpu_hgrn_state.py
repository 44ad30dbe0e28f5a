"""GPU: states of the elementwise recurrence that are updated in place, seen by the rest of a program."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40])
def test_a_graph_that_saved_the_state_refuses_its_backward(device, T):
    from fla_amd.ops.hgrn import fused_recurrent_hgrn
    x, g = torch.randn(2, T, 16, device=device), torch.randn(2, T, 16, device=device)
    state, w = torch.randn(2, 16, device=device), torch.ones(16, device=device, requires_grad=True)
    y = (state * w).sum()
    version = state._version
    fused_recurrent_hgrn(x, g, state, True, use_gate_in_kernel=True, inplace_state=True)
    assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("T", [1, 40])
def test_in_inference_mode(device, T):
    from fla_amd.ops.hgrn import chunk_hgrn, fused_recurrent_hgrn
    x, g, h0 = torch.randn(2, T, 16, device=device), torch.randn(2, T, 16, device=device), torch.randn(2, 16, device=device)
    want = chunk_hgrn(x, g, h0, True, use_gate_in_kernel=True)
    outside = h0.clone()
    with torch.inference_mode():
        for state in (h0.clone(), outside):      # one that has no version, and one that has
            o, ht = fused_recurrent_hgrn(x, g, state, True, use_gate_in_kernel=True, inplace_state=True)
            assert ht.data_ptr() == state.data_ptr()
            assert torch.equal(o, want[0]) and torch.equal(state, want[1])
