"""CPU: the oracle of the gated product against autograd and differences in fp64, and what the entries refuse ahead of a launch."""
import pytest
import torch

from oracle import gated_linear as oracle


def _inputs(M=3, F=5, K=4, bias=True):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64, requires_grad=True)
    return [r(M, K), r(F, K), r(F, K)] + ([r(F), r(F)] if bias else [])


@pytest.mark.parametrize("name", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("bias", [False, True])
def test_gradients(name, bias):
    leaves = _inputs(bias=bias)
    h, _, state = oracle.forward(*leaves, **({} if bias else {"bg": None, "bu": None}), name=name)
    fn = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, None: lambda v: v}[name]
    lin = lambda w, b: leaves[0] @ w.t() + (b if bias else 0)
    assert torch.allclose(h, fn(lin(leaves[1], leaves[3] if bias else 0)) * lin(leaves[2], leaves[4] if bias else 0), rtol=1e-12)
    dh = torch.randn(*h.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    want = torch.autograd.grad(h, leaves, dh)
    got = oracle.backward(*(t.detach() for t in leaves[:3]), [t.detach() for t in state], dh, name, 2.0 ** -9)
    for k, ref in zip(("dx", "dwg", "dwu", "dbg", "dbu"), want):
        assert torch.allclose(got[k], ref, rtol=1e-9, atol=1e-12), k


@pytest.mark.parametrize("name", ["silu", "gelu", None])
def test_differences(name):
    assert torch.autograd.gradcheck(lambda *a: oracle.forward(*a, name=name)[0], _inputs(), eps=1e-6, atol=1e-6)


@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_slopes(name):
    v = torch.linspace(-12, 12, 200001, dtype=torch.float64)
    _, d = oracle.act(name, v)
    assert d.abs().max() <= oracle.SLOPE and (d.diff() / v.diff()).abs().max() <= oracle.CURVE


def test_published_erf():
    """The formula that the kernels take for the normal distribution, in fp64: within 0.75e-7 of it."""
    v = torch.linspace(-9, 9, 100001, dtype=torch.float64)
    x = v.abs() / 2 ** 0.5
    t = 1 / (1 + 0.3275911 * x)
    tail = 0.5 * t * torch.exp(-x * x) * ((((1.061405429 * t - 1.453152027) * t + 1.421413741) * t - 0.284496736) * t + 0.254829592)
    assert (torch.where(v < 0, tail, 1 - tail) - 0.5 * torch.erfc(-v / 2 ** 0.5)).abs().max() <= 0.76e-7


def test_refusals():
    from fla_amd.modules import GatedMLP, gated_linear
    x, w = torch.zeros(2, 16).bfloat16(), torch.zeros(24, 16).bfloat16()
    with pytest.raises(RuntimeError, match="GPU"):
        gated_linear(x, w, w)
    with pytest.raises(ValueError, match="activation"):
        gated_linear(x, w, w, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        GatedMLP(16, 24, hidden_act="tanh")
    with pytest.raises(ValueError, match="weights"):
        gated_linear(x, w, w[:8])
    with pytest.raises(ValueError, match="weights"):
        gated_linear(x[:, :8], w, w)
    with pytest.raises(ValueError, match="weights"):
        gated_linear(x, w[:0], w[:0])
    with pytest.raises(TypeError, match="bf16"):
        gated_linear(x.float(), w.float(), w.float())
    with pytest.raises(TypeError, match="bf16"):
        gated_linear(x, w, w.half())
    with pytest.raises(ValueError, match="biases"):
        gated_linear(x, w, w, torch.zeros(16))
    with pytest.raises(TypeError, match="biases"):
        gated_linear(x, w, w, None, torch.zeros(24, dtype=torch.int64))
    assert GatedMLP(64).intermediate_size == 256


def test_library_entries_refuse():
    import ctypes
    from fla_amd import _backend as be
    lib, buf = be.lib(), (ctypes.c_float * 64)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    fwd = lambda x=at, K=16, F=24, ld=24, dtype=1, act=1, g=None, u=None, M=2: lib.fla_gated_linear_fwd(x, at, at, None, None, 0, at, g, u, ld, M, F, K,
                                                                                                     act, dtype, None, None)
    assert fwd(x=None) == -1 and fwd(K=0) == -1 and fwd(act=4) == -1 and fwd(g=at) == -1
    assert fwd(K=12) == -2 and fwd(dtype=0) == -2 and fwd(g=at, u=at, ld=32) == -2 and fwd(K=(1 << 22) + 8) == -2
    assert fwd(x=at + 8) == -3 and fwd(M=0) == 0
    assert lib.fla_gated_linear_bwd_gate(at, at, at, at, at, None, None, 0, 20, 2, 24, 1, 1, None) == -2
    assert lib.fla_gated_linear_bwd_gate(at, at, at + 4, at, at, None, None, 0, 24, 2, 24, 1, 1, None) == -3
    assert lib.fla_gated_linear_bwd_gate(at, at, at, at, at, at, None, 8, 24, 2, 24, 1, 1, None) == -1
    assert lib.fla_gated_linear_bwd_dx(at, at, at, at, at, 24, 12, 2, 24, 12, 1, None, None) == -2
    assert lib.fla_gated_linear_bwd_dx(at, at, at, at, at, 24, 17, 2, 24, 16, 1, None, None) == -2
    assert lib.fla_gated_linear_bwd_dw(at, at, at, None, None, 24, 16, 2, 24, 16, 1, None, None) == -1
    assert lib.fla_gated_linear_bwd_dw(at, at, at, at, at, 24, 16, 0, 24, 16, 1, None, None) == -1
    split = lib.fla_gated_linear_bwd_dw_splits(8192, 256, 256, 1)
    assert split > 1 and lib.fla_gated_linear_bwd_dw(at, at, at, at, at, 256, 256, 8192, 256, 256, 1, None, None) == -1      # no workspace
