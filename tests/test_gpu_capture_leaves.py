"""GPU: a captured call with gradients is refused while an eager graph of the default stream holds a leaf behind its operands (no backward pass is reached),
and is captured once that graph is gone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def refused_then_captured(device, call):
    """``call()`` with its eager graph alive, under capture; then without it, replayed."""
    eager = call()
    torch.cuda.synchronize()
    expected = eager.detach().clone()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.ones(1, device=device)
        with pytest.raises(RuntimeError, match="eager graph"):
            call()
        with torch.no_grad():
            call()
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    assert out.requires_grad
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.detach(), expected)
        torch.ones(10, device=device).sum().item()


def test_parameters_behind_a_cast_of_autocast(device):
    from fla_amd.modules import GatedMLP, gated_linear
    torch.manual_seed(0)
    m = GatedMLP(64, 200, bias=True, device=device)
    x = torch.randn(40, 64, device=device)

    def block():
        with torch.autocast("cuda", dtype=BF, cache_enabled=False):
            return m(x)

    def product():
        with torch.autocast("cuda", dtype=BF, cache_enabled=False):
            return gated_linear(x, m.gate_proj.weight, m.up_proj.weight)

    refused_then_captured(device, product)
    refused_then_captured(device, block)


def test_leaves_behind_other_operators(device):
    from fla_amd.modules import gated_linear, layer_norm, rms_norm
    torch.manual_seed(1)
    leaf = lambda *s: torch.randn(*s, device=device).to(BF).requires_grad_()
    e, w = leaf(40, 64), leaf(64)
    wg, wu = leaf(96, 64), leaf(96, 64)
    refused_then_captured(device, lambda: gated_linear((e * 2).view(4, 10, 64), wg.detach(), wu.detach()))
    refused_then_captured(device, lambda: layer_norm(e + 1, w.detach(), None))
    refused_then_captured(device, lambda: gated_linear(layer_norm(rms_norm(e.detach(), w), None), wg.detach(), wu.detach()))
    refused_then_captured(device, lambda: gated_linear(e.detach(), wg.t().contiguous().t(), wu.detach()))


def test_leaves_that_no_graph_holds(device):
    """An eager graph of other leaves is no reason."""
    from fla_amd.modules import gated_linear
    torch.manual_seed(2)
    leaf = lambda *s: torch.randn(*s, device=device).to(BF).requires_grad_()
    e, wg, wu, other = leaf(40, 64), leaf(96, 64), leaf(96, 64), leaf(40, 64)
    held = gated_linear(other, wg.detach(), wu.detach())
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        h = gated_linear(e * 2, wg, wu)
    assert h.requires_grad and held.requires_grad
