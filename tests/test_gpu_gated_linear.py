"""GPU: the gated product and its gradients against the formula in fp64, element by element (bounds: ``oracle/gated_linear.py``)."""
import pytest
import torch

from oracle import gated_linear as oracle

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def check(name, out, ref, bound):
    assert out is not None and tuple(out.shape) == tuple(ref.shape), name
    got = out.detach().double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    half = torch.finfo(out.dtype).eps / 2
    tiny = 2.0 ** -25 if out.dtype == HF else 2.0 ** -126
    over = ((got - ref).abs() / (half * (ref.abs() + bound) + bound + tiny)).max().item()
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, f"{name}: {over:.3f} of the bound"


def inputs(device, M, F, K, dtype, btype, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)
    bias = lambda: None if btype is None else (0.3 * r(F)).to(btype)
    return [r(M, K).to(dtype), (r(F, K) * K ** -0.5).to(dtype), (r(F, K) * K ** -0.5).to(dtype), bias(), bias()], r(M, F).to(dtype)


def double(ts):
    return [None if t is None else t.detach().double() for t in ts]


def everything(leaves, dh, name, splits=None):
    """Forward with and without a graph, and all gradients, against the oracle."""
    from fla_amd.modules import gated_linear
    args = double(leaves)
    h_ref, e_h, state = oracle.forward(*args, name=name)
    with torch.no_grad():
        plain = gated_linear(*leaves, activation=name)
    check("h", plain, h_ref, e_h)
    own = [None if t is None else t.clone().requires_grad_() for t in leaves]
    h = gated_linear(*own, activation=name)
    assert torch.equal(h, plain)
    want = oracle.backward(*args[:3], state, dh.double(), name, torch.finfo(h.dtype).eps / 2)
    grads = torch.autograd.grad(h, [t for t in own if t is not None], dh)
    for k, got in zip([k for k, t in zip(("dx", "dwg", "dwu", "dbg", "dbu"), own) if t is not None], grads):
        check(k, got, want[k], want["e_" + k])


CASES = [  # M, F, K, type, biases, activation
    (1, 1, 1, BF, BF, "silu"), (3, 5, 7, HF, FL, "gelu"), (1, 40, 64, BF, None, "silu"), (16, 17, 8, BF, BF, "relu"), (17, 100, 200, HF, HF, None),
    (33, 64, 136, BF, None, "gelu"), (48, 260, 1000, HF, FL, "silu"), (64, 24, 2056, BF, BF, "silu"), (65, 129, 1000, BF, BF, "gelu"),
    (100, 33, 4104, HF, None, "silu"), (129, 520, 264, BF, None, "relu"), (200, 1000, 2048, BF, None, "silu"), (300, 2731, 1000, HF, HF, "gelu"),
    (1000, 300, 72, BF, FL, "silu"), (2050, 640, 520, HF, None, None), (4097, 96, 40, BF, BF, "silu"), (1003, 1501, 501, BF, BF, "gelu"),
    (2049, 2824, 1032, BF, None, "silu"), (2300, 2733, 1400, HF, HF, "gelu"),
]


@pytest.mark.parametrize("M,F,K,dtype,btype,name", CASES)
def test_forward_and_gradients(device, M, F, K, dtype, btype, name):
    print(M, F, K, dtype, btype, name, flush=True)
    leaves, dh = inputs(device, M, F, K, dtype, btype, M + F)
    everything(leaves, dh, name)


def test_activations_over_their_range(device):
    """One column of K: g runs over -30 .. 30 and u is 1, so h is the activation itself and dbg its slope."""
    from fla_amd.modules import gated_linear
    for dtype in (BF, HF):
        g = torch.linspace(-30, 30, 4001).to(dtype).to(device)
        x, one = torch.ones(1, 8, device=device, dtype=dtype), torch.zeros(4001, 8, device=device, dtype=dtype)
        wg, wu = one.clone(), one.clone()
        wg[:, 0], wu[:, 0] = g, 1
        for name in ("silu", "gelu", "relu", None):
            a, slope = oracle.act(name, g.double())
            bg = torch.zeros(4001, device=device, requires_grad=True)
            h = gated_linear(x, wg, wu, bg, None, activation=name)[0]
            check(f"{name}", h, a, 3e-7 * g.double().abs() + (g.double().abs() + 8) * oracle.UNIT * a.abs())
            (d,) = torch.autograd.grad(h.float().sum(), bg)
            check(f"{name} slope", d, slope, 1e-6 * (1 + g.double().abs()))


def test_strides_addresses_and_dimensions(device):
    from fla_amd.modules import gated_linear
    (x, wg, wu, bg, bu), dh = inputs(device, 30, 48, 64, BF, BF)
    ref = gated_linear(x, wg, wu, bg, bu)
    odd = torch.empty(1 + 30 * 64, device=device, dtype=BF)[1:].view(30, 64).copy_(x)
    wide = torch.empty(30, 100, device=device, dtype=BF)[:, 20:84].copy_(x)
    both = torch.cat([wg, wu])
    turned = wu.t().contiguous().t()
    for y in (gated_linear(odd, wg, wu, bg, bu), gated_linear(wide, wg, wu, bg, bu), gated_linear(x, both[:48], both[48:], bg, bu),
              gated_linear(x, wg, turned, bg, bu), gated_linear(x.view(2, 3, 5, 64), wg, wu, bg, bu).view(30, 48)):
        assert torch.equal(y, ref)
    row = gated_linear(x[0], wg, wu, bg, bu)
    assert row.shape == (48,) and torch.equal(row, ref[0])
    # gradients of a broadcast x, of a strided dh and of one weight in both places
    leaf = x[0].clone().requires_grad_()
    w = wg.clone().requires_grad_()
    h = gated_linear(leaf.expand(30, 64), w, w)
    dleaf, dw = torch.autograd.grad(h, (leaf, w), dh.t().contiguous().t())
    one, a, b = x[0].expand(30, 64).clone().requires_grad_(), wg.clone().requires_grad_(), wg.clone().requires_grad_()
    dx, da, db = torch.autograd.grad(gated_linear(one, a, b), (one, a, b), dh)
    assert torch.equal(dw, da + db)
    assert (dleaf.double() - dx.double().sum(0)).abs().max() <= 2.0 ** -8 * dx.double().abs().sum(0).max()


def test_frozen_operands(device):
    """Each gradient alone is what it is among all of them."""
    from fla_amd.modules import gated_linear
    for M, F, K in ((20, 40, 72), (300, 136, 264)):
        leaves, dh = inputs(device, M, F, K, BF, FL)
        every = [t.clone().requires_grad_() for t in leaves]
        ref = torch.autograd.grad(gated_linear(*every), every, dh)
        for i in range(5):
            some = [t.clone().requires_grad_(i == j) for j, t in enumerate(leaves)]
            (got,) = torch.autograd.grad(gated_linear(*some), some[i], dh)
            if i in (1, 2):     # (of one weight alone the sums may be cut into other slices)
                assert (got.float() - ref[i].float()).abs().max() <= 2.0 ** -8 * ref[i].float().abs().max() + 1e-3 * M ** 0.5
            else:
                assert torch.equal(got, ref[i]), i


def test_infinities_stay_in_their_row(device):
    from fla_amd.modules import gated_linear
    for M in (20, 300):
        (x, wg, wu, _, _), _ = inputs(device, M, 136, 200, BF, None)
        bad = x.clone()
        bad[7, 3], bad[11, 199] = float("inf"), float("nan")
        y, z = gated_linear(x, wg, wu), gated_linear(bad, wg, wu)
        keep = [i for i in range(M) if i not in (7, 11)]
        assert torch.equal(y[keep], z[keep]) and z[11].isnan().all() and not torch.isfinite(z[7]).any()


def test_empty_and_refusals(device):
    from fla_amd.modules import gated_linear
    (x, wg, wu, bg, bu), _ = inputs(device, 4, 24, 16, BF, BF)
    empty = x[:0].clone().requires_grad_()
    w = wg.clone().requires_grad_()
    h = gated_linear(empty, w, wu, bg, bu)
    dx, dw = torch.autograd.grad(h.sum(), (empty, w))
    assert h.shape == (0, 24) and dx.shape == (0, 16) and not dw.any()
    assert gated_linear(x.new_zeros(2, 0, 16), wg, wu).shape == (2, 0, 24)
    with pytest.raises(RuntimeError, match="GPU"):
        gated_linear(x, wg.cpu(), wu)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        gated_linear(fwAD.make_dual(x, x), wg, wu)
    x = x.requires_grad_()
    h = gated_linear(x, wg, wu)
    (g,) = torch.autograd.grad(h.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), x)
    # written to between forward and backward
    h = gated_linear(x, w, wu)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.float().sum().backward()


def test_streams_and_captured_steps(device):
    """A training step captured into a graph, replayed with other inputs, eager work between the replays; the same on another stream."""
    from fla_amd.modules import gated_linear
    for M, F, K in ((300, 264, 520), (40, 100, 64)):
        leaves, dh = inputs(device, M, F, K, BF, FL)
        step = lambda ts, d: (lambda h: [h, *torch.autograd.grad(h, ts, d)])(gated_linear(*ts))
        fresh = lambda seed: (lambda p: ([t.requires_grad_() for t in p[0]], p[1]))(inputs(device, M, F, K, BF, FL, seed))
        eager = [[t.clone() for t in step(*fresh(s))] for s in range(3)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = step(*fresh(1))
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, eager[1]))
        static, d = fresh(0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static, d)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(static, d)
        for seed in (1, 2, 0, 1):
            ts, dd = inputs(device, M, F, K, BF, FL, seed)
            with torch.no_grad():
                for a, b in zip(static, ts):
                    a.copy_(b)
                d.copy_(dd)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager[seed])), seed
            step(*fresh(2))


def test_module(device):
    """The block against its parts, its gradients, a batch of sequences, autocast."""
    from fla_amd.modules import GatedMLP, gated_linear
    torch.manual_seed(0)
    m = GatedMLP(64, 200, hidden_act="gelu", bias=True, device=device, dtype=BF)
    x = torch.randn(2, 50, 64, device=device).to(BF).requires_grad_()
    y = m(x)
    h = gated_linear(x, m.gate_proj.weight, m.up_proj.weight, m.gate_proj.bias, m.up_proj.bias, "gelu")
    assert torch.equal(y, torch.nn.functional.linear(h, m.down_proj.weight, m.down_proj.bias))
    dy = torch.randn_like(y)
    y.backward(dy)
    f = {k: v.detach().float() for k, v in m.named_parameters()}
    xf = x.detach().float().requires_grad_()
    ps = {k: v.requires_grad_() for k, v in f.items()}
    lin = lambda n, t: torch.nn.functional.linear(t, ps[n + ".weight"], ps[n + ".bias"])
    lin("down_proj", torch.nn.functional.gelu(lin("gate_proj", xf)) * lin("up_proj", xf)).backward(dy.float())
    # each value goes through at most four roundings to 16 bits and sums of random sign: 2^-8 a rounding, relative to the whole tensor
    for k, got, ref in [("x", x.grad, xf.grad)] + [(k, p.grad, ps[k].grad) for k, p in m.named_parameters()]:
        assert ((got.float() - ref).norm() / ref.norm()).item() <= 4 * 2.0 ** -8, k
    wide = GatedMLP(64, 200, device=device)
    with torch.autocast("cuda", dtype=BF):
        out = wide(torch.randn(3, 64, device=device))
    assert out.dtype == BF
    out.float().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == FL and torch.isfinite(p.grad).all() for p in wide.parameters())
