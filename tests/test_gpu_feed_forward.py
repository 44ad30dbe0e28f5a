"""GPU: the feed-forward half of a layer as it is used: the norm with the residual's addition, the gated product and the projection back, in a training step and,
in 8-bit integers, for prompts and single tokens."""
import pytest
import torch

from oracle import gated_linear, layer_norm

pytestmark = pytest.mark.gpu

BF, FL, I8 = torch.bfloat16, torch.float32, torch.int8


def _block(device, D, F, seed=0):
    from fla_amd.modules import GatedMLP, LayerNorm
    torch.manual_seed(seed)
    norm, mlp = LayerNorm(D, bias=True).to(device=device, dtype=BF), GatedMLP(D, F, hidden_act="silu", bias=True, device=device, dtype=BF)
    with torch.no_grad():
        norm.weight.add_(0.2 * torch.randn(D, device=device))
        norm.bias.add_(0.2 * torch.randn(D, device=device))
    return norm, mlp


@pytest.mark.parametrize("B,T,D,F", [(1, 1, 64, 200), (2, 50, 64, 200), (1, 333, 256, 700), (3, 700, 512, 1408)])
def test_training_step(device, B, T, D, F):
    """Output, residual stream and all gradients against the same block in fp64.  Every value goes through at most eight roundings to bf16 on its way (the norm, both
    projections, their product, the last projection, and as many back), sums of which the errors are of either sign: 2^-8 each, relative to the whole tensor."""
    print(B, T, D, F, flush=True)
    norm, mlp = _block(device, D, F)
    gen = torch.Generator(device=device).manual_seed(1)
    r = lambda: torch.randn(B, T, D, generator=gen, device=device).to(BF)
    x, res, dy, ds = r().requires_grad_(), r().requires_grad_(), r(), r()
    y, kept = norm(x, residual=res, prenorm=True)
    out = mlp(y)
    leaves = {"x": x, "res": res, **dict(norm.named_parameters(prefix="norm")), **dict(mlp.named_parameters(prefix="mlp"))}
    grads = torch.autograd.grad((out, kept), list(leaves.values()), (dy, ds))
    d = {k: v.detach().double().requires_grad_() for k, v in leaves.items()}
    s = d["x"] + d["res"]
    h = torch.nn.functional.layer_norm(s, (D,), d["norm.weight"], d["norm.bias"], eps=norm.eps)
    lin = lambda n, t: torch.nn.functional.linear(t, d[f"mlp.{n}.weight"], d[f"mlp.{n}.bias"])
    ref = lin("down_proj", torch.nn.functional.silu(lin("gate_proj", h)) * lin("up_proj", h))
    want = torch.autograd.grad((ref, s), list(d.values()), (dy.double(), ds.double()))
    for name, got, w in [("out", out, ref), ("kept", kept, s)] + list(zip(leaves, grads, want)):
        off = ((got.double() - w).norm() / w.norm()).item()
        print(f"{name}: {off / (8 * 2.0 ** -8):.3f} of the bound", flush=True)
        assert off <= 8 * 2.0 ** -8, name


def test_captured_training_steps(device):
    """Two graphs of one block, replayed in turn with other inputs, eager steps and synchronisations between the replays; a second stream."""
    norm, mlp = _block(device, 128, 264)
    leaves = [*norm.parameters(), *mlp.parameters()]

    def step(x, res, dy):
        y, kept = norm(x, residual=res, prenorm=True)
        out = mlp(y) + kept
        grads = torch.autograd.grad(out, leaves, dy)
        # (detached: with an eager graph of the same leaves alive torch cannot capture a backward pass, its accumulation nodes belong to another stream)
        return [out.detach(), *grads]

    gen = torch.Generator(device=device).manual_seed(2)
    data = [[torch.randn(M, 128, generator=gen, device=device).to(BF) for _ in range(3)] for M in (300, 40) for _ in range(3)]
    eager = [step(*d) for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in (0, 3):
            assert all(torch.equal(a, b) for a, b in zip(step(*data[i]), eager[i]))
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for i in (0, 3):
        static = [t.clone() for t in data[i]]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*static)
        graphs.append((g, static, out))
    for k in (1, 2, 0, 2):
        for base, (g, static, out) in zip((0, 3), graphs):
            for a, b in zip(static, data[base + k]):
                a.copy_(b)
            g.replay()
        torch.cuda.synchronize()
        for base, (g, static, out) in zip((0, 3), graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, eager[base + k])), (base, k)
        step(*data[1])


def _served(device, D, F):
    from fla_amd.modules import QuantLinear, quantize_rows
    norm, mlp = _block(device, D, F)
    wg, wu = quantize_rows(mlp.gate_proj.weight.detach(), I8), quantize_rows(mlp.up_proj.weight.detach(), I8)
    down = QuantLinear.from_linear(mlp.down_proj, dtype=I8)
    return norm, mlp, wg, wu, down


def _serve(norm, mlp, wg, wu, down, x, res):
    from fla_amd.modules import quant_gated_linear, quantize_rows
    with torch.no_grad():
        rows, kept = norm(x, residual=res, prenorm=True, quantize=I8)
        h = quant_gated_linear(rows, wg, wu, mlp.gate_proj.bias, mlp.up_proj.bias)
        return rows, kept, h, quantize_rows(h, I8), down(h, residual=kept)


@pytest.mark.parametrize("M,D,F", [(1, 64, 208), (40, 256, 704), (200, 512, 1408), (2100, 256, 2816)])
def test_served_block(device, M, D, F):
    """Each stage against its formula in fp64 on what the stage before left; the whole against the block in 16 bits."""
    print(M, D, F, flush=True)
    block = _served(device, D, F)
    norm, mlp, wg, wu, down = block
    gen = torch.Generator(device=device).manual_seed(3)
    x, res = (torch.randn(M, D, generator=gen, device=device).to(BF) for _ in range(2))
    (q, scale), kept, h, (hq, hs), y = _serve(*block, x, res)
    assert torch.equal(kept, (x.float() + res.float()).to(BF))
    ny, _, _, e = layer_norm.forward(x.double(), norm.weight.detach(), norm.bias.detach(), res, eps=norm.eps)
    # half a step of the row's scale, and what the scale and the value are off
    assert ((q.double() * scale.double()[:, None] - ny).abs() <= scale.double()[:, None] * 0.5 * (1 + 1e-5) + 2 * e + 128 * e.amax(-1, keepdim=True) / 127).all()
    deq = lambda r: r[0].double() * r[1].double()[:, None]
    g, u = (deq((q, scale)) @ deq(w).t() + b.detach().double() for w, b in ((wg, mlp.gate_proj.bias), (wu, mlp.up_proj.bias)))
    ref = gated_linear.act("silu", g)[0] * u
    assert ((h.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5 * (1 + g.abs()) * (1 + u.abs())).all()
    rq, rs = layer_norm.rows_int8(h.float().cpu())
    assert torch.equal(hq.cpu(), rq) and torch.equal(hs.cpu(), rs)
    ref = deq((hq, hs)) @ deq((down.weight, down.weight_scale)).t() + down.bias.double() + kept.double()
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5 * (1 + ref.abs())).all()
    with torch.no_grad():
        full = mlp(norm(x, residual=res)) + kept
    assert ((y - full).double().norm() / full.double().norm()).item() <= 0.05      # (three roundings of rows and weights to steps of 1/127 of the largest)


def test_single_tokens_are_rows_of_the_prompt(device):
    """The sums are exact and the epilogues the same: a row is the same bits by itself, in a small batch and in a prompt, from whatever kernel."""
    block = _served(device, 256, 704)
    gen = torch.Generator(device=device).manual_seed(4)
    x, res = (torch.randn(700, 256, generator=gen, device=device).to(BF) for _ in range(2))
    whole = _serve(*block, x, res)[-1]
    for rows in (slice(0, 1), slice(5, 6), slice(100, 117), slice(300, 364), slice(300, 400), slice(0, 699)):
        assert torch.equal(_serve(*block, x[rows], res[rows])[-1], whole[rows]), rows


def test_captured_serving(device):
    block = _served(device, 256, 704)
    gen = torch.Generator(device=device).manual_seed(5)
    data = [[torch.randn(3, 256, generator=gen, device=device).to(BF) for _ in range(2)] for _ in range(3)]
    eager = [_serve(*block, *d)[-1] for d in data]
    static = [t.clone() for t in data[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _serve(*block, *static)[-1]
    for i in (1, 2, 0, 1):
        for a, b in zip(static, data[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), i
        _serve(*block, *data[2])


def test_capture_refuses_leaves_of_an_eager_graph(device):
    """Refused ahead of any launch: the backward pass is never reached.  Without gradients, and once the eager graph is gone, the calls are captured."""
    from fla_amd.modules import gated_linear, layer_norm
    g = torch.Generator().manual_seed(3)
    leaf = lambda *s: torch.randn(*s, generator=g).to(device, torch.bfloat16).requires_grad_()
    x, wg, wu, bg, w, b = leaf(40, 64), leaf(96, 64), leaf(96, 64), leaf(96), leaf(64), leaf(64)
    calls = [lambda: gated_linear(x.detach(), wg, wu, bg), lambda: gated_linear(x.detach(), wg.detach(), wu.detach(), bg),
             lambda: layer_norm(x, w, b), lambda: layer_norm(x.detach(), w.detach(), b)]
    for call in calls:
        y = call()
        torch.cuda.synchronize()
        expected = y.detach().clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            still = torch.ones(1, device=device)
            with pytest.raises(RuntimeError, match="eager graph"):
                call()
            with torch.no_grad():
                out = call()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, expected) and still.item() == 1
        del y, out
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            out = call()
        assert out.requires_grad
        del out


MANY, LAST = 1_100_003, 2000      # rows of 2048 elements: offsets of the last ones pass 2^31


def test_rows_behind_32_bit_offsets_of_the_norm(device):
    """The last rows of 2.25e9 elements.  One rounding to bf16 (2^-8 of the value), and below it some tens of fp32 roundings of values of at most 8."""
    from fla_amd.modules import layer_norm
    g = torch.Generator().manual_seed(5)
    some = lambda *s: torch.randn(*s, generator=g).to(device, torch.bfloat16)
    x, dy = (torch.zeros(MANY, 2048, device=device, dtype=torch.bfloat16) for _ in range(2))
    x[-LAST:], dy[-LAST:] = some(LAST, 2048), some(LAST, 2048)
    w, b = some(2048), some(2048)
    x.requires_grad_()
    y = layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    xs, ws, bs, ds = (t.detach()[-LAST:].double().cpu() if t.dim() == 2 else t.double().cpu() for t in (x, w, b, dy))
    c = xs - xs.mean(1, keepdim=True)
    r = (c.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    h, d = c * r, ds * ws
    for a, e in ((y, h * ws + bs), (dx, r * (d - d.mean(1, keepdim=True) - h * (d * h).mean(1, keepdim=True)))):
        a = a.detach()[-LAST:].double().cpu()
        assert ((a - e).abs() <= e.abs() / 256 + 2.0 ** -16).all()


def test_rows_behind_32_bit_offsets_of_the_gated_product(device):
    """The last rows of 2.25e9 elements of h and of what is kept, against the same rows by themselves: one slice of K, so the same sums; one row with a
    gradient, so one product in each of the weights'.  Those of x are sums of 4096 products in two orders, each rounded once to bf16."""
    from fla_amd.modules import gated_linear
    g = torch.Generator().manual_seed(6)
    some = lambda *s: torch.randn(*s, generator=g).to(device, torch.bfloat16)
    x, dh = torch.zeros(MANY, 64, device=device, dtype=torch.bfloat16), torch.zeros(MANY, 2048, device=device, dtype=torch.bfloat16)
    x[-LAST:], dh[-1] = some(LAST, 64), some(2048)
    wg, wu = ((some(2048, 64) / 8).requires_grad_() for _ in range(2))
    results = []
    for rows in (MANY, LAST):
        xs = x[-rows:].detach().requires_grad_()
        h = gated_linear(xs, wg, wu)
        dx, dwg, dwu = torch.autograd.grad(h, (xs, wg, wu), dh[-rows:])
        results.append([h.detach()[-LAST:].clone(), dx[-LAST:].clone(), dwg, dwu])
        del h, dx
    (h, dx, dwg, dwu), (h0, dx0, dwg0, dwu0) = results
    assert h0.abs().sum() > 0 and torch.equal(h, h0) and torch.equal(dwg, dwg0) and torch.equal(dwu, dwu0)
    p, q = wg.detach().double().cpu(), wu.detach().double().cpu()
    a, d = x[-1].double().cpu(), dh[-1].double().cpu()
    gate, up = p @ a, q @ a
    s = gate.sigmoid()
    terms = (d * up * s * (1 + gate * (1 - s))).abs() @ p.abs() + (d * gate * s).abs() @ q.abs()
    assert not dx[:-1].any() and dx0[-1].abs().sum() > 0
    assert ((dx[-1].double() - dx0[-1].double()).abs().cpu() <= dx0[-1].double().abs().cpu() / 128 + 2 * 4096 * 2.0 ** -24 * 1.02 * terms).all()


@pytest.mark.parametrize("K, N", ((2048, 48), (64, 2048)))
def test_rows_behind_32_bit_offsets_of_integers(device, K, N):
    """The last rows of 2.25e9 elements of x, or of the results: sums are exact, so the same bits as by themselves."""
    from fla_amd.modules import quant_gated_linear, quant_linear
    g = torch.Generator().manual_seed(7)
    ints = lambda *s: torch.randint(-127, 128, s, generator=g, dtype=torch.int8).to(device)
    scales = lambda n: (torch.rand(n, generator=g) / 100 + 0.001).to(device)
    x, sx = torch.zeros(MANY, K, device=device, dtype=torch.int8), torch.ones(MANY, device=device)
    x[-LAST:], sx[-LAST:] = ints(LAST, K), scales(LAST)
    w, wu, sw, su = ints(N, K), ints(N, K), scales(N), scales(N)
    with torch.no_grad():
        for call in (lambda r: quant_linear((x[-r:], sx[-r:]), (w, sw)),
                     lambda r: quant_gated_linear((x[-r:], sx[-r:]), (w, sw), (wu, su))):
            y = call(MANY)[-LAST:].clone()
            assert y.abs().sum() > 0 and torch.equal(y, call(LAST))
