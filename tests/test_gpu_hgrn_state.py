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


@pytest.mark.parametrize("packed", [False, True])
def test_a_batch_without_tokens_keeps_its_graph(device, packed):
    """Every operand that asks for a gradient gets one: zeros, and the final state's for the initial one."""
    from fla_amd.ops.hgrn import chunk_hgrn
    B, N = (1, 2) if packed else (2, 2)
    leaves = [torch.zeros(B, 0, 16, device=device), torch.zeros(B, 0, 16, device=device, dtype=torch.bfloat16), torch.rand(16, device=device) * 0.5,
              torch.randn(N, 16, device=device)]
    leaves = [t.requires_grad_() for t in leaves]
    x, g, lb, h0 = leaves
    offs = torch.zeros(N + 1, device=device, dtype=torch.int64) if packed else None
    o, ht = chunk_hgrn(x, g, h0, True, cu_seqlens=offs, use_gate_in_kernel=True, lower_bound=lb)
    dx, dg, dlb, dh0 = torch.autograd.grad(o.sum() + ht.sum(), leaves)
    assert dx.shape == x.shape and dg.shape == g.shape and dg.dtype == g.dtype
    assert dlb.shape == lb.shape and not dlb.any() and torch.equal(dh0, torch.ones_like(h0))
    # one operand alone that asks
    o, _ = chunk_hgrn(x.detach(), g.detach(), h0.detach(), True, cu_seqlens=offs, use_gate_in_kernel=True, lower_bound=lb)
    assert not torch.autograd.grad(o.sum(), lb)[0].any()
    o, ht = chunk_hgrn(x.detach(), g.detach(), h0, True, cu_seqlens=offs, use_gate_in_kernel=True, lower_bound=lb.detach())
    assert torch.equal(torch.autograd.grad(o.sum() + 2 * ht.sum(), h0)[0], torch.full_like(h0, 2.0))
