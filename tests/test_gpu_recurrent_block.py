"""GPU: the norm, the 8-bit products and the gated recurrence together, as a layer uses them.

Serving: a prompt and then single tokens through norm -> projection -> recurrence -> projection + residual, the state in a ``Cache``;
each stage is held to its own formula on what it was given (a rounding to 8 bits that goes the other way ahead of a stage would hide or
fake an error of that stage otherwise).  Training: the same layer with 32-bit projections, all gradients against fp64 autograd."""
import pytest
import torch

from oracle import hgrn as hgrn_oracle
from oracle import rms_norm as norm_oracle

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _within(name, out, ref, bound):
    got, half = out.detach().double().cpu(), torch.finfo(out.dtype).eps / 2
    over = ((got - ref).abs() / (half * (ref.abs() + bound) + bound + 2.0 ** -126)).max().item()
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, name


def _deq(q, s):
    return q.double().cpu() * s.double().cpu()[..., None]


def test_serving(device):
    from fla_amd.models import Cache
    from fla_amd.modules import QuantLinear, RMSNorm, quantize_rows
    from fla_amd.ops.hgrn import chunk_hgrn, fused_recurrent_hgrn
    gen = torch.Generator().manual_seed(0)
    D, B, T = 128, 2, 300
    norm = RMSNorm(D).to(device, BF)
    wide = QuantLinear.from_linear(torch.nn.Linear(D, 2 * D).to(device, BF))
    back = QuantLinear.from_linear(torch.nn.Linear(D, D, bias=False).to(device, BF))
    bound = (torch.rand(D, generator=gen) * 0.5).to(device)
    cache = Cache()

    def product(x, layer, residual=None):
        """The formula on the operands' values, and a bound: products of eight cut at 2^-13 of the largest, each with its sign (the sum of
        K = 128 of them by seven standard deviations), the rest in fp32."""
        xd, wd = _deq(*x), _deq(layer.weight, layer.weight_scale)
        y, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
        # each of a group's eight is cut by at most 2^-13 of the largest: sum over groups of 8 max^2 <= 8 sum of squares
        e = 7 * 2.0 ** -13 * (8 * (xd.square() @ wd.square().t())).sqrt() + 2.0 ** -18 * mag
        if layer.bias is not None:
            y = y + layer.bias.double().cpu()
        return (y if residual is None else y + residual.double().cpu()), e + 2.0 ** -22 * y.abs()

    def layer(h, residual, state, step):
        (q, s), kept = norm(h, residual=residual, prenorm=True, quantize=True)
        ny, ns, _, ne = norm_oracle.forward(h.cpu(), norm.weight.detach().cpu(), None, residual.cpu(), norm.eps)
        _within("residual stream", kept, ns, norm_oracle.UNIT * ns.abs())
        room = (ny.abs() * 2.0 ** -4).clamp_min(s.double().cpu()[..., None] * 2.0 ** -10) * (1 + 2.0 ** -16) + 2 * ne
        assert ((_deq(q, s) - ny).abs() <= room).all()
        both = wide((q, s))
        _within("input projection", both, *product((q, s), wide))
        i, f = both.chunk(2, -1)
        if step:
            at = state.data_ptr()
            o, new = fused_recurrent_hgrn(i, f, state.clone(), True, use_gate_in_kernel=True, lower_bound=bound)
            o2, kept_state = fused_recurrent_hgrn(i, f, state, True, use_gate_in_kernel=True, lower_bound=bound, inplace_state=True)
            assert torch.equal(o, o2) and torch.equal(new, kept_state) and kept_state.data_ptr() == at
            before, state = None, kept_state
        else:
            before = None if state is None else state.cpu()
            o, state = chunk_hgrn(i, f, state, True, use_gate_in_kernel=True, lower_bound=bound)
            ho, hht, eo, eht = hgrn_oracle.forward(i.cpu(), f.cpu(), before, None, bound.cpu(), True)
            _within("recurrence", o, ho, eo)
            _within("state", state, hht, eht)
        rows = quantize_rows(o)
        y = back(rows, residual=kept)
        _within("output projection", y, *product(rows, back, kept))
        return y, kept, state

    h, residual = (torch.randn(B, T, D, generator=gen).to(BF).to(device) for _ in range(2))
    with torch.no_grad():
        y, _, state = layer(h, residual, None, False)
        cache.update(recurrent_state=state, layer_idx=0, offset=T)
        held = cache[0]["recurrent_state"].data_ptr()
        # three more tokens, one at a time; and the same as one short call from the same state
        more = torch.randn(2, B, 3, D, generator=gen).to(BF).to(device)
        start = cache[0]["recurrent_state"].clone()
        for t in range(3):
            _, _, s = layer(more[0][:, t:t + 1], more[1][:, t:t + 1], cache[0]["recurrent_state"], True)
            cache.update(recurrent_state=s, layer_idx=0, offset=1)
        assert cache[0]["recurrent_state"].data_ptr() == held and cache.get_seq_length() == T + 3
        layer(more[0], more[1], start, False)


def test_training(device):
    """fp32 throughout: each of the seven steps is off by some 64 units of 2^-24 of what it adds up (4e-6), and the later ones carry the
    earlier ones' errors on with factors of a few (norms and gates of slope about one): 1e-4 of a gradient's norm holds them."""
    from fla_amd.modules import RMSNorm
    from fla_amd.ops.hgrn import chunk_hgrn
    gen = torch.Generator().manual_seed(1)
    D, T = 96, 330
    r = lambda *s: torch.randn(*s, generator=gen)
    offs = torch.tensor([0, 101, 101, 330])
    values = {"h": r(1, T, D), "res": r(1, T, D), "w": 1 + 0.2 * r(D), "win": r(2 * D, D) * D ** -0.5, "wout": r(D, D) * D ** -0.5,
              "bound": torch.rand(D, generator=gen) * 0.9, "h0": r(3, D), "w2": 1 + 0.2 * r(D)}
    dy = r(1, T, D)

    def ours(v):
        norm, norm2 = RMSNorm(D).to(device), RMSNorm(D).to(device)
        norm.weight, norm2.weight = torch.nn.Parameter(v["w"]), torch.nn.Parameter(v["w2"])
        y, stream = norm(v["h"], residual=v["res"], prenorm=True)
        i, f = (y @ v["win"].t()).chunk(2, -1)
        o, ht = chunk_hgrn(i, f, v["h0"], True, cu_seqlens=offs.to(device), use_gate_in_kernel=True, lower_bound=v["bound"])
        y2 = norm2(o @ v["wout"].t(), residual=stream)
        return y2, ht, (norm.weight, norm2.weight)

    def plain(v):
        y, stream, _, _ = norm_oracle.forward(v["h"], v["w"], None, v["res"])
        i, f = (y @ v["win"].t()).chunk(2, -1)
        o, ht, _, _ = hgrn_oracle.forward(i, f, v["h0"], offs, v["bound"], True)
        return norm_oracle.forward(o @ v["wout"].t(), v["w2"], None, stream)[0], ht

    a = {k: t.double().requires_grad_() for k, t in values.items()}
    y, ht = plain(a)
    want = dict(zip(a, torch.autograd.grad((y * dy.double()).sum() + ht.sum(), list(a.values()))))
    b = {k: t.to(device).requires_grad_() for k, t in values.items()}
    y2, ht2, weights = ours(b)
    leaves = [weights[0] if k == "w" else weights[1] if k == "w2" else b[k] for k in b]
    got = dict(zip(b, torch.autograd.grad((y2 * dy.to(device)).sum() + ht2.sum(), leaves)))
    for name, x, z in [("y", y, y2), ("ht", ht, ht2)] + [(k, want[k], got[k]) for k in want]:
        off = ((x - z.double().cpu()).norm() / x.norm()).item()
        print(name, off, flush=True)
        assert off < 1e-4, name


def test_a_training_step_in_a_graph(device):
    """Forward, backward and the weights' gradients of norm and recurrence in one captured graph, replayed with other inputs."""
    from fla_amd.modules import RMSNorm
    from fla_amd.ops.hgrn import chunk_hgrn
    gen = torch.Generator().manual_seed(2)
    norm = RMSNorm(256).to(device, BF)
    x, res, dy = (torch.randn(1, 700, 256, generator=gen).to(BF).to(device) for _ in range(3))
    x.requires_grad_()

    def step():
        y, s = norm(x, residual=res, prenorm=True)
        o, _ = chunk_hgrn(y[..., :128], y[..., 128:], use_gate_in_kernel=True)
        return [o, *torch.autograd.grad((o, s), (x, norm.weight), (dy[..., :128].contiguous(), dy))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), k


def test_tangents_are_refused(device):
    """None of the three has a forward-mode derivative: an operand with a tangent raises, also where no gradient is asked for."""
    import torch.autograd.forward_ad as fwd
    from fla_amd.modules import quant_linear, quantize_rows, rms_norm
    from fla_amd.ops.hgrn import chunk_hgrn, fused_recurrent_hgrn
    x = torch.randn(1, 6, 32, device=device)
    w = quantize_rows(x[0])
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwd.dual_level():
            dual = fwd.make_dual(x, torch.ones_like(x))
            for call in (lambda: chunk_hgrn(dual, x), lambda: fused_recurrent_hgrn(x[:, :1], dual[:, :1]), lambda: rms_norm(dual, None),
                         lambda: quantize_rows(dual), lambda: quant_linear(w, w, residual=dual[0, :, :6])):
                with pytest.raises(RuntimeError):
                    call()
