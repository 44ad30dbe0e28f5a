"""GPU: the elementwise gated recurrence against the formula in fp64, element by element.

A value may be off by half a step of the type it is stored in plus what the fp32 evaluation may be off by, which the oracle
derives with the value (``oracle/hgrn.py``)."""
import pytest
import torch
import torch.nn.functional as F

from oracle import hgrn as oracle

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def _check(name, out, ref, bound):
    assert out is not None and tuple(out.shape) == tuple(ref.shape), name
    got = out.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    half = torch.finfo(out.dtype).eps / 2
    tiny = 2.0 ** -25 if out.dtype == HF else 2.0 ** -126     # half the smallest step; fp32 numbers below the normal ones may be zero
    room = half * (ref.abs() + bound) + bound + tiny
    over = ((got - ref).abs() / room).max().item() if ref.numel() else 0.0
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, f"{name}: {over:.3f} of the bound"


def _inputs(B, T, D, dtype, gtype, gates, bound, state, lens, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    x, g = r(B, T, D).to(dtype), r(B, T, D) + (1.0 if gates else 0.0)
    g = (g if gates else F.logsigmoid(g) / 4).to(gtype)
    offs = None if lens is None else torch.tensor(lens)
    N = B if lens is None else len(lens) - 1
    return (x, g, r(N, D) if state else None, torch.rand(D, generator=gen) * 0.9 if bound else None, offs, r(B, T, D).to(dtype), r(N, D))


def _run(x, g, h0, lb, offs, do, dht, gates, device, fn=None, grad=True):
    from fla_amd.ops.hgrn import chunk_hgrn
    put = lambda t, leaf=True: None if t is None else t.to(device).requires_grad_(grad and leaf)
    x, g, h0, lb = put(x), put(g), put(h0), put(lb)
    o, ht = (fn or chunk_hgrn)(x, g, initial_state=h0, output_final_state=True, cu_seqlens=put(offs, False) if offs is not None else None,
                               use_gate_in_kernel=gates, lower_bound=lb)
    if not grad:
        return o, ht
    leaves = {k: v for k, v in (("dx", x), ("dg", g), ("dh0", h0), ("dlb", lb)) if v is not None}
    grads = torch.autograd.grad((o, ht), list(leaves.values()), (do.to(device), dht.to(device)))
    return o, ht, dict(zip(leaves, grads))


def _compare(args, gates, device, grad=True, fn=None):
    x, g, h0, lb, offs, do, dht = args
    ho, hht, eo, eht = oracle.forward(x, g, h0, offs, lb, gates)
    got = _run(*args, gates, device, fn, grad)
    _check("o", got[0], ho, eo)
    _check("ht", got[1], hht, eht)
    assert got[0].dtype == x.dtype and got[1].dtype == FL
    if grad:
        want = oracle.backward(x, g, do, dht, h0, offs, lb, gates)
        for k, v in got[2].items():
            _check(k, v, want[k], want["e_" + k])
    return got


CASES = [
    # B, T, D, type, gate type, gates, bound, state, lens
    (2, 1, 64, BF, BF, True, True, True, None),           # one token, through the scan (gradients)
    (1, 16, 1, FL, FL, False, False, True, None),         # one channel
    (3, 17, 72, HF, FL, False, False, False, None),
    (2, 128, 200, BF, FL, True, False, True, None),
    (1, 129, 64, FL, FL, True, True, True, None),
    (2, 255, 7, HF, HF, False, False, True, None),
    (2, 256, 8, BF, BF, True, True, False, None),         # one tile
    (1, 257, 136, BF, BF, False, False, True, None),      # cut in two, one token behind
    (1, 1030, 67, FL, FL, True, True, True, None),        # five segments, odd channels
    (1, 770, 128, HF, FL, True, True, True, None),
    (200, 300, 64, BF, BF, True, True, True, None),       # a workgroup for every CU: whole sequences, two tiles each
    (260, 130, 72, HF, FL, True, True, True, None),       # short sequences that share CUs
    (1, 600, 96, BF, BF, True, True, True, [0, 1, 1, 300, 317, 600]),          # an empty sequence, one of a single token
    (1, 900, 30, HF, FL, False, False, True, [5, 40, 40, 40, 850]),            # rows outside, empty ones, segments
    (1, 64, 64, FL, FL, False, False, True, [0, 0, 0]),                        # no sequence has a token
]


@pytest.mark.parametrize("B,T,D,dtype,gtype,gates,bound,state,lens", CASES)
def test_forward_and_gradients(device, B, T, D, dtype, gtype, gates, bound, state, lens):
    args = _inputs(B, T, D, dtype, gtype, gates, bound, state, lens, seed=T + D)
    print(B, T, D, dtype, gtype, gates, lens, flush=True)
    o, _, grads = _compare(args, gates, device)
    if lens is not None:
        outside = torch.ones(T, dtype=torch.bool)
        outside[lens[0]:lens[-1]] = False
        for t in (o, grads["dx"], grads["dg"]):
            assert not t.detach().cpu()[0, outside].any()
    again = _run(*args, gates, device)
    assert torch.equal(o, again[0]) and all(torch.equal(grads[k], again[2][k]) for k in grads)      # nothing depends on an order
    plain = _run(*args, gates, device, grad=False)
    assert torch.equal(o, plain[0])


@pytest.mark.parametrize("N,D,dtype,gtype,gates,bound", [(1, 1, BF, BF, True, True), (5, 2048, HF, FL, False, False),
                                                         (3, 100, FL, FL, True, False), (33, 264, BF, BF, True, True)])
def test_step_in_place(device, N, D, dtype, gtype, gates, bound):
    from fla_amd.ops.hgrn import fused_recurrent_hgrn
    x, g, h0, lb, _, _, _ = _inputs(N, 1, D, dtype, gtype, gates, bound, True, None, seed=N)
    ho, hht, eo, eht = oracle.forward(x, g, h0, None, lb, gates)
    state = h0.to(device)
    at = state.data_ptr()
    how = dict(use_gate_in_kernel=gates, lower_bound=None if lb is None else lb.to(device))
    o, ht = fused_recurrent_hgrn(x.to(device), g.to(device), initial_state=state.clone(), output_final_state=True, **how)
    o2, ht2 = fused_recurrent_hgrn(x.to(device), g.to(device), initial_state=state, output_final_state=True, inplace_state=True, **how)
    assert ht2.data_ptr() == at and torch.equal(ht, ht2) and torch.equal(o, o2)
    _check("o", o, ho, eo)
    _check("ht", ht, hht, eht)
    o3, none = fused_recurrent_hgrn(x.to(device), g.to(device), **how)         # from nothing, final state not asked for
    ho, _, eo, _ = oracle.forward(x, g, None, None, lb, gates)
    _check("o from zero", o3, ho, eo)
    assert none is None


def test_in_place_over_several_tokens_and_steps_continue_a_prompt(device):
    """A cut prompt that writes the final state over the initial one, then single steps: the whole is one sequence."""
    from fla_amd.ops.hgrn import fused_recurrent_hgrn
    x, g, h0, lb, _, _, _ = _inputs(2, 520, 80, BF, BF, True, True, True, None)
    ho, hht, eo, eht = oracle.forward(x, g, h0, None, lb, True)
    x, g, lb, state = x.to(device), g.to(device), lb.to(device), h0.to(device)
    at, how = state.data_ptr(), dict(use_gate_in_kernel=True, lower_bound=lb, output_final_state=True, inplace_state=True)
    o = [fused_recurrent_hgrn(x[:, :517], g[:, :517], initial_state=state, **how)[0]]
    for t in range(517, 520):
        step, state = fused_recurrent_hgrn(x[:, t:t + 1], g[:, t:t + 1], initial_state=state, **how)
        o.append(step)
    assert state.data_ptr() == at
    _check("o", torch.cat(o, 1), ho, eo)
    _check("ht", state, hht, eht)
    with pytest.raises(ValueError, match="inplace_state"):
        fused_recurrent_hgrn(x, g, output_final_state=True, inplace_state=True)
    with pytest.raises(ValueError, match="inplace_state"):
        fused_recurrent_hgrn(x, g, initial_state=state.bfloat16(), output_final_state=True, inplace_state=True)
    with pytest.raises(ValueError, match="gradient"):
        fused_recurrent_hgrn(x.requires_grad_(), g, initial_state=state, output_final_state=True, inplace_state=True)


@pytest.mark.parametrize("T", [1, 300])
@pytest.mark.parametrize("shift", [0, 1])
def test_slices_of_a_projection(device, T, shift):
    """x and g as the two halves of one projection's output, read where they lie, at a 16-byte address and off one."""
    from fla_amd.ops.hgrn import chunk_hgrn
    D = 72
    wide = torch.randn(2, T, 2 * D + 8, generator=torch.Generator().manual_seed(T)).bfloat16()
    view = lambda w: (w[..., shift:shift + D], w[..., shift + D:shift + 2 * D])
    ho, hht, eo, eht = oracle.forward(*view(wide), gates=True)
    w = wide.to(device).requires_grad_()
    o, ht = chunk_hgrn(*view(w), output_final_state=True, use_gate_in_kernel=True)
    _check("o", o, ho, eo)
    _check("ht", ht, hht, eht)
    do = torch.randn(2, T, D, generator=torch.Generator().manual_seed(9)).bfloat16()
    want = oracle.backward(*view(wide), do, gates=True)
    got, = torch.autograd.grad(o, w, do.to(device))
    for k, v in zip(("dx", "dg"), view(got)):
        _check(k, v, want[k], want["e_" + k])
    with torch.no_grad():
        t = w.transpose(0, 1)                                  # rows that have no one pitch: copied first
        o2, _ = chunk_hgrn(t.contiguous()[..., :D].transpose(0, 1), view(w)[1], use_gate_in_kernel=True)
        o3, _ = chunk_hgrn(w[..., :D], view(w)[1], use_gate_in_kernel=True)
        assert torch.equal(o2, o3)
        one = w[:1, :, :D].expand(3, T, D)
        o4, _ = chunk_hgrn(one, one, use_gate_in_kernel=True)
        o5, _ = chunk_hgrn(one.contiguous(), one.contiguous(), use_gate_in_kernel=True)
        assert torch.equal(o4, o5)


@pytest.mark.parametrize("dtype", [FL, BF])
def test_resets(device, dtype):
    """Log decays that reset the state (-inf, the type's lowest value), several in a row, at both ends and on a tile's border."""
    T, D = 600, 40
    x, g, h0, _, _, do, dht = _inputs(1, T, D, dtype, dtype, False, False, True, None, seed=4)
    for t, v in ((0, float("-inf")), (100, torch.finfo(dtype).min), (101, float("-inf")), (255, -1e30), (256, float("-inf")),
                 (T - 1, float("-inf"))):
        g[:, t, ::2] = v
    _compare((x, g, h0, None, None, do, dht), False, device)
    # pre-activations of infinite size: a = 0 and a = 1 exactly
    x, g, h0, lb, _, do, dht = _inputs(1, T, D, dtype, dtype, True, False, True, None, seed=5)
    g[:, 7, ::2], g[:, 300, ::3], g[:, 299, 1] = float("-inf"), float("inf"), -200.0
    _compare((x, g, h0, None, None, do, dht), True, device)


def test_not_a_number_stays_in_its_sequence_and_channel(device):
    from fla_amd.ops.hgrn import chunk_hgrn
    x, g, h0, _, _, _, _ = _inputs(1, 700, 24, FL, FL, False, False, True, [0, 300, 700])
    offs = torch.tensor([0, 300, 700], device=device)
    want, _ = chunk_hgrn(x.to(device), g.to(device), h0.to(device), cu_seqlens=offs)
    x[0, 310, 5] = float("nan")
    got, _ = chunk_hgrn(x.to(device), g.to(device), h0.to(device), cu_seqlens=offs)
    bad = torch.zeros(1, 700, 24, dtype=torch.bool)
    bad[0, 310:, 5] = True
    assert torch.equal(got.isnan().cpu(), bad) and torch.equal(got.cpu()[~bad], want.cpu()[~bad])


def test_against_differences(device):
    """The slope of sum(w o) + sum(v ht) along a direction, from the gradients and from differences of the kernel's own forward.

    Central differences with a step of 2^-6 are off by step^2/6 of the third derivative (each operand enters through functions
    whose derivatives stay below their arguments' size here) and by the forward's fp32 rounding over the step: 600 tokens of 24
    channels with random signs, 2^-24 * 32 * sqrt(600 * 24) * S / 2^-6 with S about 4: 1.5e-2 on a slope of about ten."""
    from fla_amd.ops.hgrn import chunk_hgrn
    x, g, h0, lb, _, do, dht = [None if t is None else t.to(device) for t in _inputs(1, 600, 24, FL, FL, True, True, True, None, seed=8)]
    leaves = [t.requires_grad_() for t in (x, g, h0, lb)]
    gen = torch.Generator(device=device).manual_seed(1)
    dirs = [torch.randn(t.shape, generator=gen, device=device) * s for t, s in zip(leaves, (1.0, 1.0, 1.0, 0.05))]

    def loss(*t):
        o, ht = chunk_hgrn(t[0], t[1], t[2], True, use_gate_in_kernel=True, lower_bound=t[3])
        return (o.double() * do).sum() + (ht.double() * dht).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    e = 2.0 ** -6
    with torch.no_grad():
        for name, i in (("x", 0), ("f", 1), ("h0", 2), ("bound", 3)):
            at = lambda s: loss(*[t + s * dirs[i] if j == i else t for j, t in enumerate(leaves)])
            slope = ((at(e) - at(-e)) / (2 * e)).item()
            want = (grads[i].double() * dirs[i]).sum().item()
            print(name, slope, want, flush=True)
            assert abs(slope - want) <= 0.05 + 2e-3 * abs(want), name


def test_types_of_the_operands(device):
    """Operands of other types than the kernels': converted, and their gradients come back in their own."""
    from fla_amd.ops.hgrn import chunk_hgrn
    x, g, h0, lb, _, do, _ = [None if t is None else t.to(device) for t in _inputs(2, 40, 16, FL, FL, True, True, True, None)]
    leaves = [x.requires_grad_(), g.bfloat16().requires_grad_(), h0.half().requires_grad_(), lb.bfloat16().requires_grad_()]
    o, _ = chunk_hgrn(leaves[0], leaves[1], leaves[2], use_gate_in_kernel=True, lower_bound=leaves[3])
    want, _ = chunk_hgrn(leaves[0].detach(), leaves[1].detach().float(), leaves[2].detach().float(), use_gate_in_kernel=True,
                         lower_bound=leaves[3].detach().float())
    assert torch.equal(o, want)
    for leaf, grad in zip(leaves, torch.autograd.grad(o, leaves, do)):
        assert grad.dtype == leaf.dtype and grad.shape == leaf.shape and torch.isfinite(grad).all()
    h, f = x.detach().bfloat16(), g.detach().half()
    assert torch.equal(chunk_hgrn(h, f)[0], chunk_hgrn(h, f.float())[0])


def test_no_tokens(device):
    from fla_amd.ops.hgrn import chunk_hgrn
    h0 = torch.randn(2, 16, device=device, requires_grad=True)
    x = torch.zeros(2, 0, 16, device=device)
    o, ht = chunk_hgrn(x, x, h0, True)
    assert o.shape == x.shape and torch.equal(ht, h0)
    assert torch.equal(torch.autograd.grad(ht.sum(), h0)[0], torch.ones_like(h0))
    o, ht = chunk_hgrn(x, x, output_final_state=True)
    assert not ht.any() and ht.shape == (2, 16)
    x, g = x.clone().requires_grad_(), x.bfloat16().requires_grad_()
    o, _ = chunk_hgrn(x, g)
    o.sum().backward()
    assert o.dtype == x.dtype and x.grad.shape == x.shape and g.grad.shape == x.shape


def test_only_some_gradients_arrive(device):
    x, g, h0, lb, _, do, dht = _inputs(1, 300, 24, BF, BF, True, True, True, None)
    from fla_amd.ops.hgrn import chunk_hgrn
    leaves = [t.to(device).requires_grad_() for t in (x, g, h0, lb)]
    o, ht = chunk_hgrn(leaves[0], leaves[1], leaves[2], True, use_gate_in_kernel=True, lower_bound=leaves[3])
    for out, w, a, b in ((o, do, do, None), (ht, dht, torch.zeros_like(do), dht)):
        want = oracle.backward(x, g, a, b, h0, None, lb, True)
        for k, v in zip(("dx", "dg", "dh0", "dlb"), torch.autograd.grad(out, leaves, w.to(device), retain_graph=True)):
            _check(k, v, want[k], want["e_" + k])


def test_changed_offsets_are_refused_by_the_backward(device):
    from fla_amd.ops.hgrn import chunk_hgrn
    x = torch.randn(1, 64, 16, device=device, requires_grad=True)
    offs = torch.tensor([0, 20, 64], device=device)
    o, _ = chunk_hgrn(x, x, cu_seqlens=offs, use_gate_in_kernel=True)
    offs[1] = 30
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_another_stream_and_two_at_once(device):
    """Two calls on two streams, each with its own workspace."""
    from fla_amd.ops.hgrn import chunk_hgrn
    sets = [[None if t is None else t.to(device) for t in _inputs(1, 3000, 128, BF, BF, True, True, True, None, seed=s)] for s in (1, 2)]
    call = lambda s: chunk_hgrn(s[0], s[1], s[2], True, use_gate_in_kernel=True, lower_bound=s[3])
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = call(sets[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured(device):
    """A cut training step and a decode step as HIP graphs, replayed with eager work between the replays."""
    from fla_amd.ops.hgrn import chunk_hgrn, fused_recurrent_hgrn
    x, g, h0, lb, _, do, dht = [None if t is None else t.to(device) for t in _inputs(1, 900, 64, BF, BF, True, True, True, None)]
    leaves = [t.requires_grad_() for t in (x, g, h0, lb)]

    def train():
        o, ht = chunk_hgrn(leaves[0], leaves[1], leaves[2], True, use_gate_in_kernel=True, lower_bound=leaves[3])
        return [o, ht, *torch.autograd.grad((o, ht), leaves, (do, dht))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    state = h0.detach().clone()
    step_graph = torch.cuda.CUDAGraph()
    xs, gs = x.detach()[:, :1].clone(), g.detach()[:, :1].clone()
    with torch.cuda.graph(step_graph):
        so, _ = fused_recurrent_hgrn(xs, gs, state, True, use_gate_in_kernel=True, lower_bound=lb.detach(), inplace_state=True)
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)))
            xs.copy_(x[:, k:k + 1])
        want = train()
        wo, wht = fused_recurrent_hgrn(xs, gs, state.clone(), True, use_gate_in_kernel=True, lower_bound=lb.detach())
        graph.replay()
        step_graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), k
        assert torch.equal(wo, so) and torch.equal(wht, state), k


def test_long_rows_pass_32_bits(device):
    """A batch whose rows lie further apart than 2^31 bytes from its first to its last: offsets are 64 bits wide."""
    from fla_amd.ops.hgrn import chunk_hgrn
    D, T = 64, 2200
    wide = torch.zeros(1, T, 1 << 20, dtype=BF, device=device)          # 4.6 GB, of which 64 columns are used
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(1, T, D, generator=gen).bfloat16()
    wide[..., :D] = x.to(device)
    with torch.no_grad():
        o, _ = chunk_hgrn(wide[..., :D], wide[..., :D], use_gate_in_kernel=True)
    ho, _, eo, _ = oracle.forward(x, x, gates=True)
    _check("o", o, ho, eo)


def test_packed_batch_captured(device):
    """A packed training step, cut into segments, as a graph: the tables of its offsets are there since an eager step."""
    from fla_amd.ops.hgrn import chunk_hgrn
    ends = [0, 1, 701, 701, 2201, 2264]
    x, g, h0, lb, offs, do, dht = [t.to(device) for t in _inputs(1, ends[-1], 40, HF, FL, True, True, True, ends)]
    leaves = [t.requires_grad_() for t in (x, g, h0, lb)]

    def train():
        o, ht = chunk_hgrn(leaves[0], leaves[1], leaves[2], True, cu_seqlens=offs, use_gate_in_kernel=True, lower_bound=leaves[3])
        return [o.detach(), ht.detach(), *torch.autograd.grad((o, ht), leaves, (do, dht))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)))
        want = train()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), k
