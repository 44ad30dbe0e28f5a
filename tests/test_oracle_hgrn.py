"""CPU: the oracle of the elementwise gated recurrence (its gradients against autograd and against differences), the entry points'
refusals, and the rule that cuts sequences."""
import pytest
import torch

from oracle import hgrn as oracle


def _inputs(gates, T=7, D=5, lens=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    B = 2 if lens is None else 1
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    x, g = r(B, T, D), r(B, T, D)
    g = g if gates else torch.nn.functional.logsigmoid(g)
    offs = None if lens is None else torch.tensor([0] + lens).cumsum(0)
    N = B if lens is None else len(lens)
    return x, g, r(N, D), (torch.rand(D, generator=gen, dtype=torch.float64) * 0.9 if gates else None), offs, r(B, T, D), r(N, D)


@pytest.mark.parametrize("gates", [False, True])
@pytest.mark.parametrize("lens", [None, [3, 0, 4]])
def test_gradients_are_those_of_the_forward(gates, lens):
    x, g, h0, lb, offs, do, dht = _inputs(gates, lens=lens)
    leaves = [t.clone().requires_grad_() for t in (x, g, h0) + (() if lb is None else (lb,))]

    def loss(*t):
        h, ht, _, _ = oracle.forward(t[0], t[1], t[2], offs, t[3] if gates else None, gates)
        return (h * do).sum() + (ht * dht).sum()

    want = torch.autograd.grad(loss(*leaves), leaves)
    assert torch.autograd.gradcheck(loss, leaves)            # against differences
    got = oracle.backward(x, g, do, dht, h0, offs, lb, gates)
    for name, w in zip(("dx", "dg", "dh0", "dlb"), want):
        assert torch.allclose(got[name], w, rtol=1e-12, atol=1e-12), name


def test_segments():
    from fla_amd import _backend as be
    seg = be.lib().fla_hgrn_segment
    tile = 256
    for n, tokens, longest, D in ((1, 1, 1, 1), (8, 8 * 4096, 4096, 2048), (1, 8192, 8192, 2048), (12, 16384, 9000, 1000),
                                  (1, 1 << 20, 1 << 20, 64), (300, 300, 1, 64), (1, 255, 255, 4096)):
        s = seg(n, tokens, longest, D)
        assert s > 0 and s % tile == 0 and -(-longest // s) <= 64, (n, tokens, longest, D, s)
    assert seg(8, 8 * 4096, 4096, 2048) >= 4096               # a workgroup for every CU: whole sequences
    assert seg(1, 8192, 8192, 2048) < 8192                    # 32 workgroups: cut


def test_refusals():
    from fla_amd.ops.hgrn import chunk_hgrn, fused_recurrent_hgrn
    x = torch.zeros(1, 8, 16)
    offs = torch.tensor([0, 4, 8])
    for fn in (chunk_hgrn, fused_recurrent_hgrn):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            fn(x, x)
        with pytest.raises(ValueError, match="one shape"):
            fn(x, x[:, :4])
        with pytest.raises(ValueError, match=r"\[B, T, D\]"):
            fn(x[0], x[0])
        with pytest.raises(ValueError, match=r"\[B, T, D\]"):
            fn(x[0], x[0], offsets=offs)
        with pytest.raises(TypeError, match="floating"):
            fn(x.long(), x.long())
        with pytest.raises(ValueError, match="batch size"):
            fn(x.expand(2, 8, 16), x.expand(2, 8, 16), offsets=offs)
        with pytest.raises(ValueError, match="initial states"):
            fn(x, x, offsets=offs, initial_state=torch.zeros(3, 16))
        with pytest.raises(ValueError, match="initial_state is"):
            fn(x, x, initial_state=torch.zeros(1, 8))
        with pytest.raises(ValueError, match="either"):
            fn(x, x, offsets=offs, cu_seqlens=offs)
        with pytest.raises(ValueError, match="leave the"):
            fn(x, x, cu_seqlens=torch.tensor([0, 9]))
        with pytest.raises(ValueError, match="leave the"):
            fn(x, x, cu_seqlens=torch.tensor([-1, 8]))
        with pytest.raises(ValueError, match="non-decreasing"):
            fn(x, x, cu_seqlens=torch.tensor([0, 6, 4, 8]))
        with pytest.raises(ValueError, match="use_gate_in_kernel"):
            fn(x, x, lower_bound=torch.zeros(16))
        with pytest.raises(ValueError, match="per channel"):
            fn(x, x, lower_bound=torch.zeros(8), use_gate_in_kernel=True)


def test_library_arguments():
    import ctypes
    from fla_amd import _backend as be
    lib = be.lib()
    p = ctypes.c_void_p(torch.zeros(64).data_ptr())
    fwd = lambda seg=256, maps=None, B=1, N=1, T=8, D=8, ldx=8, lb=None, types=(0, 0): lib.fla_hgrn_fwd(
        p, p, lb, None, p, None, None, maps, None, None, None, 0, seg, 0, *types, B, T, D, N, ldx, 8, None)
    assert fwd(seg=100) == -1 and fwd(seg=0) == -1            # not whole tiles
    assert fwd(T=300) == -1                                   # cut, and no workspace
    assert fwd(N=2) == -1 and fwd(ldx=4) == -1 and fwd(T=0) == -1 and fwd(lb=p) == -1
    assert fwd(types=(1, 2)) == -2
    assert fwd(B=1 << 23, N=1 << 23, T=1) == -2               # more workgroups than a launch takes
    bwd = lambda states, dlb=None: lib.fla_hgrn_bwd(p, p, None, states, None, None, p, p, None, dlb, None, None, None, None, 0, 256, 0, 0, 0,
                                                    1, 8, 8, 1, 8, 8, None)
    assert bwd(None) == -1 and bwd(p, p) == -1
    assert lib.fla_hgrn_step(p, p, None, None, p, None, 0, 1, 2, 1, 8, 8, 8, None) == -2
    assert lib.fla_hgrn_step(p, p, None, None, p, None, 0, 0, 0, 1, 8, 4, 8, None) == -1


def test_install_rebinds_the_recurrence(monkeypatch):
    """``fla_amd.install()`` on stub modules: the package's names and those that the layer bound at import."""
    import sys
    import types
    import fla_amd
    from fla_amd.ops import hgrn
    names = ("chunk_hgrn", "fused_recurrent_hgrn")
    mods = {}
    for name in ("fla", "fla.ops", "fla.ops.hgrn", "fla.layers", "fla.layers.hgrn"):
        mods[name] = types.ModuleType(name)
        mods[name].__path__ = []
        monkeypatch.setitem(sys.modules, name, mods[name])
    for name in ("fla.ops.hgrn", "fla.layers.hgrn"):
        for n in names:
            setattr(mods[name], n, object())
    patched = fla_amd.install()
    assert {f"{m}.{n}" for m in ("fla.ops.hgrn", "fla.layers.hgrn") for n in names} == set(patched)
    assert all(getattr(mods[m], n) is getattr(hgrn, n) for m in ("fla.ops.hgrn", "fla.layers.hgrn") for n in names)
